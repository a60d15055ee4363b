// kvq_share_capi.cpp -- the extern "C" entry points of chunk attention and shared
// pages (include/kvq.h, part 8).  Arguments are validated before any HIP call.
#include <limits.h>
#include <math.h>

#include "../../include/kvq.h"
#include "kvq_call.hpp"
#include "kvq_chunk.hpp"
#include "kvq_share.hpp"

namespace {

using kvq::checked_call;

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

bool heads_ok(int num_kv_heads, int head_dim) {
    return num_kv_heads > 0 && head_dim > 0 && head_dim <= KVQ_MAX_HEAD_DIM;
}

// A pool whose slots are numbered in 32 bits.
bool slots_ok(int page_size, int num_pages) {
    return page_size > 0 && num_pages > 0 && static_cast<long long>(page_size) * num_pages <= INT_MAX;
}

// n rows `stride` elements apart lie within an address space.
bool spans(int64_t n, int64_t stride) { return n <= 1 || stride <= (1LL << 46) / n; }

// A table of B rows of max_pages pages, and what a row holds.
bool table_ok(int batch, int most, int max_pages, int page_size) {
    return batch > 0 && batch <= most && max_pages > 0 && page_size > 0 &&
           static_cast<long long>(max_pages) * page_size <= INT_MAX && static_cast<long long>(batch) * max_pages <= INT_MAX;
}

bool chunk_params_ok(const kvq_chunk_attention_params* p) {
    if (!p || !heads_ok(p->num_kv_heads, p->head_dim) || p->num_q_heads <= 0 || p->num_q_heads % p->num_kv_heads != 0)
        return false;
    if (!table_ok(p->batch, KVQ_CHUNK_MAX_BATCH, p->max_pages_per_seq, p->page_size) || p->num_pages <= 0) return false;
    const long long cap = static_cast<long long>(p->max_pages_per_seq) * p->page_size;
    if (p->max_seq_len < 0 || p->max_seq_len > cap || (p->max_seq_len > 0 ? p->max_seq_len : cap) > KVQ_MAX_SEQ_LEN)
        return false;
    if (p->tokens < 0 || static_cast<long long>(p->tokens) * p->num_q_heads > INT_MAX) return false;
    if (p->dtype != KVQ_DTYPE_F32 && p->dtype != KVQ_DTYPE_BF16) return false;
    const int64_t row = static_cast<int64_t>(p->num_q_heads) * p->head_dim;
    if ((p->q_stride != 0 && p->q_stride < row) || (p->out_stride != 0 && p->out_stride < row)) return false;
    if (!spans(p->tokens, p->q_stride) || !spans(p->tokens, p->out_stride)) return false;
    return p->token_offsets && p->lengths && p->block_table && p->q && p->out && p->k_pages && p->v_pages &&
           p->k_scale_pages && p->v_scale_pages;
}

kvq::ChunkArgs chunk_args(const kvq_chunk_attention_params* p) {
    kvq::ChunkArgs a{};
    const int size = p->page_size;
    a.pages = kvq::PageMap{p->block_table, size, p->max_pages_per_seq, p->num_pages,
                           (size & (size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(size)) : -1};
    a.offsets = p->token_offsets;
    a.lengths = p->lengths;
    a.granted = p->granted;
    a.q = p->q;
    a.out = p->out;
    a.k = p->k_pages;
    a.v = p->v_pages;
    a.ks = p->k_scale_pages;
    a.vs = p->v_scale_pages;
    const int64_t row = static_cast<int64_t>(p->num_q_heads) * p->head_dim;
    a.q_stride = p->q_stride ? p->q_stride : row;
    a.out_stride = p->out_stride ? p->out_stride : row;
    a.B = p->batch;
    a.Hq = p->num_q_heads;
    a.Hkv = p->num_kv_heads;
    a.G = p->num_q_heads / p->num_kv_heads;
    a.d = p->head_dim;
    a.T = p->tokens;
    a.max_len = p->max_seq_len > 0 ? p->max_seq_len : p->max_pages_per_seq * p->page_size;
    a.page = kvq::make_fastdiv(static_cast<uint32_t>(size));
    a.bf16 = p->dtype == KVQ_DTYPE_BF16;
    a.causal = p->causal != 0;
    // Rounded once: a relative error of it is one of every score.
    const double scale = p->softmax_scale > 0.0f ? static_cast<double>(p->softmax_scale) : 1.0 / sqrt(static_cast<double>(p->head_dim));
    a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    return a;
}

// Rows of 16-byte pieces, caches of 8-byte ones.
bool chunk_vec_ok(const kvq_chunk_attention_params* p, const kvq::ChunkArgs& a) {
    const int64_t size = a.bf16 ? 2 : 4;
    return ((bits(p->q) | bits(p->out)) & 15u) == 0 && ((bits(p->k_pages) | bits(p->v_pages)) & 7u) == 0 &&
           a.q_stride * size % 16 == 0 && a.out_stride * size % 16 == 0;
}

bool fork_params_ok(const kvq_page_fork_params* p) {
    if (!p || !table_ok(p->batch, KVQ_FORK_MAX_BATCH, p->max_pages_per_seq, p->page_size) ||
        !slots_ok(p->page_size, p->num_pages))
        return false;
    return p->parents && p->lengths && p->block_table && p->shares && p->free_pages && p->free_count && p->new_lengths &&
           p->new_block_table && p->new_shares && p->new_free_count && p->copy_src && p->copy_dst;
}

kvq::ForkArgs fork_args(const kvq_page_fork_params* p) {
    kvq::ForkArgs a{};
    a.parents = p->parents;
    a.keep = p->keep;
    a.lengths = p->lengths;
    a.table = p->block_table;
    a.shares = p->shares;
    a.free_pages = p->free_pages;
    a.free_count = p->free_count;
    a.new_lengths = p->new_lengths;
    a.new_table = p->new_block_table;
    a.new_shares = p->new_shares;
    a.new_free_count = p->new_free_count;
    a.copy_src = p->copy_src;
    a.copy_dst = p->copy_dst;
    a.B = p->batch;
    a.max_pages = p->max_pages_per_seq;
    a.num_pages = p->num_pages;
    a.cap = p->max_pages_per_seq * p->page_size;
    a.page = kvq::make_fastdiv(static_cast<uint32_t>(p->page_size));
    return a;
}

bool compact_params_ok(const kvq_page_compact_params* p) {
    if (!p || !table_ok(p->batch, KVQ_FORK_MAX_BATCH, p->max_pages_per_seq, p->page_size) ||
        !slots_ok(p->page_size, p->num_pages) || p->max_moves <= 0 || (p->shares == nullptr) != (p->new_shares == nullptr))
        return false;
    return p->lengths && p->block_table && p->free_pages && p->free_count && p->new_block_table && p->new_free_pages &&
           p->copy_src && p->copy_dst && p->moved;
}

kvq::CompactArgs compact_args(const kvq_page_compact_params* p) {
    kvq::CompactArgs a{};
    a.lengths = p->lengths;
    a.table = p->block_table;
    a.shares = p->shares;
    a.free_pages = p->free_pages;
    a.free_count = p->free_count;
    a.new_table = p->new_block_table;
    a.new_shares = p->new_shares;
    a.new_free_pages = p->new_free_pages;
    a.copy_src = p->copy_src;
    a.copy_dst = p->copy_dst;
    a.moved = p->moved;
    a.B = p->batch;
    a.max_pages = p->max_pages_per_seq;
    a.num_pages = p->num_pages;
    a.max_moves = p->max_moves;
    a.cap = p->max_pages_per_seq * p->page_size;
    a.page = kvq::make_fastdiv(static_cast<uint32_t>(p->page_size));
    return a;
}

}  // namespace

extern "C" {

size_t kvq_chunk_attention_workspace_size(const kvq_chunk_attention_params* p) {
    if (!chunk_params_ok(p)) return 0;
    const kvq::ChunkArgs a = chunk_args(p);
    return kvq::chunk_plan(a, chunk_vec_ok(p, a)).bytes;
}

hipError_t kvq_chunk_attention_launch(const kvq_chunk_attention_params* p, void* workspace, size_t workspace_bytes,
                                      hipStream_t stream) {
    if (!chunk_params_ok(p)) return hipErrorInvalidValue;
    const kvq::ChunkArgs a = chunk_args(p);
    const kvq::ChunkPlan plan = kvq::chunk_plan(a, chunk_vec_ok(p, a));
    if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes)) return hipErrorInvalidValue;
    return checked_call(stream, [&] { return kvq::launch_chunk(a, plan, workspace, stream); });
}

hipError_t kvq_chunk_attention_plan(const kvq_chunk_attention_params* p, kvq_plan_info* info) {
    if (!info || !chunk_params_ok(p)) return hipErrorInvalidValue;
    const kvq::ChunkArgs a = chunk_args(p);
    const kvq::ChunkPlan plan = kvq::chunk_plan(a, chunk_vec_ok(p, a));
    kvq_plan_info r{};
    r.kernel = plan.mfma ? KVQ_KERNEL_CHUNK_MFMA : KVQ_KERNEL_CHUNK_GENERIC;
    r.heads_per_group = plan.mfma ? a.G : 1;
    const bool split = plan.records > 0;
    r.splits = split ? 0 : 1;
    r.chunk = split ? 0 : a.max_len;
    r.split_plan = split ? KVQ_SPLITS_IN_KERNEL : KVQ_SPLITS_STATIC;
    r.query_block = plan.mfma ? plan.rows : 1;
    r.workspace_bytes = plan.bytes;
    r.tile_tokens = plan.mfma ? kvq::kChunkKeys : 0;
    *info = r;
    return hipSuccess;
}

size_t kvq_page_fork_workspace_size(const kvq_page_fork_params* p) {
    return fork_params_ok(p) ? kvq::fork_workspace(fork_args(p)) : 0;
}

hipError_t kvq_page_fork_launch(const kvq_page_fork_params* p, void* workspace, size_t workspace_bytes,
                                hipStream_t stream) {
    if (!fork_params_ok(p)) return hipErrorInvalidValue;
    kvq::ForkArgs a = fork_args(p);
    if (!workspace || workspace_bytes < kvq::fork_workspace(a)) return hipErrorInvalidValue;
    kvq::fork_place(a, workspace);
    return checked_call(stream, [&] { return kvq::launch_page_fork(a, stream); });
}

hipError_t kvq_page_copy_launch(const kvq_page_copy_params* p, hipStream_t stream) {
    if (!p || p->copies < 0 || p->layers < 1 || p->layers > 65535 || !heads_ok(p->num_kv_heads, p->head_dim) ||
        !slots_ok(p->page_size, p->num_pages) || (p->bounds == nullptr) != (p->bound_scale == nullptr))
        return hipErrorInvalidValue;
    // Pairs of all layers are numbered in 32 bits; a list longer than the pool has mostly nothing to copy.
    const long long units = static_cast<long long>(p->copies) * p->layers;
    if (p->copies >= 1 << 24 || units > INT_MAX || (units >= 1 << 24 && p->copies > p->num_pages)) return hipErrorInvalidValue;
    if (!p->src || !p->dst || !p->k_pages || !p->v_pages || !p->k_scale_pages || !p->v_scale_pages)
        return hipErrorInvalidValue;
    kvq::CopyArgs a{};
    a.src = p->src;
    a.dst = p->dst;
    a.n = p->copies;
    a.layers = p->layers;
    a.num_pages = p->num_pages;
    const size_t rows = static_cast<size_t>(p->num_kv_heads) * p->page_size;
    char* const base[] = {reinterpret_cast<char*>(p->k_pages),       reinterpret_cast<char*>(p->v_pages),
                          reinterpret_cast<char*>(p->k_scale_pages), reinterpret_cast<char*>(p->v_scale_pages),
                          reinterpret_cast<char*>(p->bounds),        reinterpret_cast<char*>(p->bound_scale)};
    const size_t bytes[] = {rows * p->head_dim, rows * p->head_dim, rows * sizeof(float), rows * sizeof(float),
                            2 * static_cast<size_t>(p->num_kv_heads) * p->head_dim, p->num_kv_heads * sizeof(float)};
    for (int i = 0; i < kvq::CopyArgs::kArrays; i++) {
        a.base[i] = base[i];
        a.bytes[i] = bytes[i];
    }
    return checked_call(stream, [&] { return kvq::launch_page_copy(a, stream); });
}

size_t kvq_page_compact_workspace_size(const kvq_page_compact_params* p) {
    return compact_params_ok(p) ? kvq::compact_workspace(compact_args(p)) : 0;
}

hipError_t kvq_page_compact_launch(const kvq_page_compact_params* p, void* workspace, size_t workspace_bytes,
                                   hipStream_t stream) {
    if (!compact_params_ok(p)) return hipErrorInvalidValue;
    kvq::CompactArgs a = compact_args(p);
    if (!workspace || workspace_bytes < kvq::compact_workspace(a)) return hipErrorInvalidValue;
    kvq::compact_place(a, workspace);
    return checked_call(stream, [&] { return kvq::launch_page_compact(a, stream); });
}

}  // extern "C"
