// kvq_pages_capi.cpp -- the extern "C" entry points around a paged cache
// (include/kvq.h, part 7).  Arguments are validated before any HIP call.
#include <limits.h>

#include <algorithm>

#include "../../include/kvq.h"
#include "kvq_call.hpp"
#include "kvq_pages.hpp"

namespace {

using kvq::checked_call;
using kvq::kCounterBytes;

constexpr size_t kAlign = 256;
size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// A pool whose slots are numbered in 32 bits.
bool slots_ok(int page_size, int num_pages) {
    return page_size > 0 && num_pages > 0 && static_cast<long long>(page_size) * num_pages <= INT_MAX;
}

bool heads_ok(int num_kv_heads, int head_dim) {
    return num_kv_heads > 0 && head_dim > 0 && head_dim <= KVQ_MAX_HEAD_DIM;
}

// The tuned bounds kernels address a page's keys with 32-bit offsets.
bool page_fits(int page_size, int head_dim) { return static_cast<long long>(page_size) * head_dim < (1LL << 30); }

// Sequences of a bounds launch and (sequence, kv head)s of a selection lie along
// the grid's x in workgroups of 256 and 512 threads: below 2^32 of them.
constexpr long long kMaxBoundsBatch = (1LL << 24) - 1, kMaxSelectUnits = (1LL << 23) - 1;

// n rows `stride` elements apart lie within an address space.
bool spans(int64_t n, int64_t stride) { return n <= 1 || stride <= (1LL << 46) / n; }

bool dtype_ok(int dtype) { return dtype == KVQ_DTYPE_F32 || dtype == KVQ_DTYPE_BF16; }

kvq::PageMap page_map(const int32_t* table, int size, int max_pages, int num_pages) {
    return kvq::PageMap{table, size, max_pages, num_pages, (size & (size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(size)) : -1};
}

// ---- page map ---------------------------------------------------------------

bool map_params_ok(const kvq_page_map_params* p) {
    if (!p || p->batch <= 0 || p->batch > KVQ_PAGE_MAP_MAX_BATCH || p->max_pages_per_seq <= 0 || p->max_tokens < 0)
        return false;
    if (!slots_ok(p->page_size, p->num_pages)) return false;
    if (static_cast<long long>(p->max_pages_per_seq) * p->page_size > INT_MAX) return false;
    if (static_cast<long long>(p->batch) * p->max_pages_per_seq > INT_MAX) return false;
    return p->new_tokens && p->lengths && p->block_table && p->free_pages && p->free_count && p->new_lengths &&
           p->new_free_count && p->granted && p->token_offsets;
}

kvq::PageMapArgs map_args(const kvq_page_map_params* p) {
    kvq::PageMapArgs a{};
    a.new_tokens = p->new_tokens;
    a.lengths = p->lengths;
    a.table = p->block_table;
    a.free_pages = p->free_pages;
    a.free_count = p->free_count;
    a.new_lengths = p->new_lengths;
    a.new_free_count = p->new_free_count;
    a.granted = p->granted;
    a.offsets = p->token_offsets;
    a.slot_map = p->slot_map;
    a.token_seq = p->token_seq;
    a.token_pos = p->token_pos;
    a.B = p->batch;
    a.max_pages = p->max_pages_per_seq;
    a.num_pages = p->num_pages;
    a.T = p->max_tokens;
    a.cap = p->max_pages_per_seq * p->page_size;
    a.page = kvq::make_fastdiv(static_cast<uint32_t>(p->page_size));
    return a;
}

size_t map_bytes(const kvq::PageMapArgs& a) { return kvq::page_map_groups(a) > 1 ? kAlign : 0; }

// ---- sparse decode ------------------------------------------------------------

struct SparsePlan {
    kvq_paged_decode_params step;  // the attention: one sequence per (sequence, kv head) over `selected`
    kvq::SelectPlan select;
    bool vec_ok;
    size_t step_bytes, keys_at, bytes;
};

// The dense step's longest sequence.
int max_len_of(const kvq_paged_decode_params& p) {
    return p.max_seq_len > 0 ? p.max_seq_len : p.max_pages_per_seq * p.page_size;
}

bool sparse_params_ok(const kvq_sparse_decode_params* p) {
    if (!p) return false;
    kvq_plan_info info;
    if (kvq_paged_decode_plan(&p->decode, &info) != hipSuccess) return false;  // every check of the dense step
    if (p->keep_first < 0 || p->keep_last < 1 || p->max_selected < 1) return false;
    if (static_cast<long long>(p->keep_first) + p->keep_last > p->max_selected) return false;
    if (!p->bounds || !p->bound_scale || !p->selected || !p->selected_lengths) return false;
    const kvq_paged_decode_params& s = p->decode;
    const long long units = static_cast<long long>(s.batch) * s.num_kv_heads;
    if (units > kMaxSelectUnits) return false;
    if (static_cast<long long>(s.num_pages) * s.num_kv_heads > INT_MAX || units * p->max_selected > INT_MAX) return false;
    return static_cast<long long>(p->max_selected) * s.page_size <= INT_MAX;
}

SparsePlan sparse_plan(const kvq_sparse_decode_params* p) {
    SparsePlan r{};
    r.step = p->decode;
    kvq_paged_decode_params& s = r.step;
    const int max_len = max_len_of(s);
    s.batch = p->decode.batch * p->decode.num_kv_heads;
    s.num_q_heads = p->decode.num_q_heads / p->decode.num_kv_heads;
    s.num_kv_heads = 1;
    s.num_pages = p->decode.num_pages * p->decode.num_kv_heads;
    s.max_pages_per_seq = p->max_selected;
    s.max_seq_len = static_cast<int>(std::min<long long>(max_len, static_cast<long long>(p->max_selected) * s.page_size));
    s.block_table = p->selected;
    s.lengths = p->selected_lengths;
    if (s.num_splits == 0) {
        // Sequences longer than the selection attend the same number of tokens,
        // so the split count of a uniform batch, over at least two tiles a wave,
        // beats the plans for ragged ones: 8 heads of 4096 tokens 24.0 us a step
        // with those, 20.3 in 16 splits (21.0 in 8, 21.7 in 32, 41.4 unsplit); 128
        // units of 4096 tokens 47.3 us, 41.2 in 2 splits (55.0 unsplit, 42.5 in 4);
        // 256 units of 2048 tokens, whose ragged plan has a launch of its own, 85.0
        // us, 43.5 unsplit.  It is not the best count of long selections (8192
        // tokens: 192 units 95.8 us unsplit, 88.4 in 4; 96 units 55.9 in 2, 53.2
        // in 8).
        // It is taken where the sequences fit the selection as well, whose lengths
        // may be anything; there the dense step, planned for ragged lengths, is the
        // faster one (G = 4, d = 128, sparse / dense step: 16 sequences of 512 to
        // 8192 tokens 42.8 / 28.5 us, 2048 to 32768 131.6 / 79, 64 of 512 to 8192
        // 129 / 82; all of 8192 48.8 / 52 and 169 / 181).
        // The count goes on as a request, which the planner's rules for small steps
        // leave alone; with them (the uniform plan's kernel too) 3 to 7 heads over
        // 512 tokens take 15.4-18.2 us for 16.6-18.4, but twelve heads over 32
        // tokens of 2048 units 58.8 for 44.7, and the generic kernel over 2112
        // tokens, in 7 splits instead of 8, 288 for 247.
        kvq_paged_decode_params u = s;
        u.lengths = nullptr;
        kvq_plan_info info;
        if (kvq_paged_decode_plan(&u, &info) == hipSuccess) s.num_splits = std::max(1, std::min(info.splits, s.max_seq_len / 256));
    }
    r.step_bytes = kvq_paged_decode_workspace_size(&s);
    r.vec_ok = ((bits(s.k_pages) | bits(p->bounds) | bits(s.q)) & 15u) == 0 && page_fits(s.page_size, s.head_dim);
    r.select = kvq::select_plan(s.batch, s.num_q_heads, s.head_dim, r.vec_ok, (max_len - 1) / s.page_size + 1, p->max_selected);
    // The selection's arrival counters share the workspace's counter prefix with
    // the attention's: the launches are ordered and each leaves them at zero.
    // Ranks never lie in the prefix, which another shape may count in.
    r.keys_at = round_up(std::max(r.step_bytes, kCounterBytes), kAlign);
    r.bytes = r.select.key_bytes ? r.keys_at + r.select.key_bytes : r.step_bytes;
    return r;
}

}  // namespace

extern "C" {

size_t kvq_page_map_workspace_size(const kvq_page_map_params* p) { return map_params_ok(p) ? map_bytes(map_args(p)) : 0; }

hipError_t kvq_page_map_launch(const kvq_page_map_params* p, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
    if (!map_params_ok(p)) return hipErrorInvalidValue;
    kvq::PageMapArgs a = map_args(p);
    const size_t need = map_bytes(a);
    if (need > 0 && (!workspace || workspace_bytes < need)) return hipErrorInvalidValue;
    a.arrivals = need > 0 ? static_cast<int*>(workspace) : nullptr;
    return checked_call(stream, [&] { return kvq::launch_page_map(a, stream); });
}

hipError_t kvq_slot_write_launch(const kvq_slot_write_params* p, hipStream_t stream) {
    if (!p || p->tokens < 0 || !heads_ok(p->num_kv_heads, p->head_dim) || !slots_ok(p->page_size, p->num_pages) ||
        !dtype_ok(p->dtype))
        return hipErrorInvalidValue;
    if (!p->k_new || !p->v_new || !p->slots || !p->k_pages || !p->v_pages || !p->k_scale_pages || !p->v_scale_pages)
        return hipErrorInvalidValue;
    if (static_cast<long long>(p->tokens) * p->num_kv_heads >= (1LL << 31)) return hipErrorInvalidValue;
    const int64_t row = static_cast<int64_t>(p->num_kv_heads) * p->head_dim;
    if ((p->k_stride != 0 && p->k_stride < row) || (p->v_stride != 0 && p->v_stride < row)) return hipErrorInvalidValue;
    if (!spans(p->tokens, p->k_stride) || !spans(p->tokens, p->v_stride)) return hipErrorInvalidValue;
    const bool bf16 = p->dtype == KVQ_DTYPE_BF16;
    kvq::SlotArgs a{};
    a.slots = p->slots;
    a.k = p->k_pages;
    a.v = p->v_pages;
    a.ks = p->k_scale_pages;
    a.vs = p->v_scale_pages;
    a.k_rows = const_cast<void*>(p->k_new);
    a.v_rows = const_cast<void*>(p->v_new);
    a.k_stride = p->k_stride ? p->k_stride : row;
    a.v_stride = p->v_stride ? p->v_stride : row;
    a.head_stride = p->head_dim;
    a.T = p->tokens;
    a.Hkv = p->num_kv_heads;
    a.d = p->head_dim;
    a.slots_in_pool = p->num_pages * p->page_size;
    a.page = kvq::make_fastdiv(static_cast<uint32_t>(p->page_size));
    a.heads = kvq::make_fastdiv(static_cast<uint32_t>(p->num_kv_heads));
    const int64_t size = bf16 ? 2 : 4;
    const bool vec_ok = ((bits(p->k_new) | bits(p->v_new)) & 15u) == 0 && a.k_stride * size % 16 == 0 &&
                        a.v_stride * size % 16 == 0 && ((bits(p->k_pages) | bits(p->v_pages)) & 7u) == 0;
    return checked_call(stream, [&] { return kvq::launch_slot_write(a, bf16, vec_ok, stream); });
}

hipError_t kvq_slot_read_launch(const kvq_slot_read_params* p, hipStream_t stream) {
    if (!p || p->tokens < 0 || !heads_ok(p->num_kv_heads, p->head_dim) || !slots_ok(p->page_size, p->num_pages) ||
        !dtype_ok(p->dtype))
        return hipErrorInvalidValue;
    if (!p->k_out || !p->v_out || !p->slots || !p->k_pages || !p->v_pages || !p->k_scale_pages || !p->v_scale_pages)
        return hipErrorInvalidValue;
    if (static_cast<long long>(p->tokens) * p->num_kv_heads >= (1LL << 31)) return hipErrorInvalidValue;
    // Rows apart: the tokens of a head within a token's heads, or the other way round.
    const int64_t ts = p->token_stride, hs = p->head_stride, d = p->head_dim, T = p->tokens, H = p->num_kv_heads;
    if (ts < 0 || hs < 0 || !spans(T, ts) || !spans(H, hs)) return hipErrorInvalidValue;
    const bool by_token = (H == 1 || hs >= d) && (T <= 1 || ts >= (H > 1 ? (H - 1) * hs : 0) + d);
    const bool by_head = (T <= 1 || ts >= d) && (H == 1 || hs >= (T > 1 ? (T - 1) * ts : 0) + d);
    if (!by_token && !by_head) return hipErrorInvalidValue;
    const bool bf16 = p->dtype == KVQ_DTYPE_BF16;
    kvq::SlotArgs a{};
    a.slots = p->slots;
    a.k = const_cast<int8_t*>(p->k_pages);
    a.v = const_cast<int8_t*>(p->v_pages);
    a.ks = const_cast<float*>(p->k_scale_pages);
    a.vs = const_cast<float*>(p->v_scale_pages);
    a.k_rows = p->k_out;
    a.v_rows = p->v_out;
    a.k_stride = a.v_stride = ts;
    a.head_stride = hs;
    a.T = p->tokens;
    a.Hkv = p->num_kv_heads;
    a.d = p->head_dim;
    a.slots_in_pool = p->num_pages * p->page_size;
    a.page = kvq::make_fastdiv(static_cast<uint32_t>(p->page_size));
    a.heads = kvq::make_fastdiv(static_cast<uint32_t>(p->num_kv_heads));
    const int64_t size = bf16 ? 2 : 4;
    const bool vec_ok = ((bits(p->k_out) | bits(p->v_out)) & 15u) == 0 && (T <= 1 || ts * size % 16 == 0) &&
                        (H == 1 || hs * size % 16 == 0) && ((bits(p->k_pages) | bits(p->v_pages)) & 7u) == 0;
    return checked_call(stream, [&] { return kvq::launch_slot_read(a, bf16, vec_ok, stream); });
}

hipError_t kvq_page_bounds_launch(const kvq_page_bounds_params* p, hipStream_t stream) {
    if (!p || p->batch <= 0 || p->batch > kMaxBoundsBatch || !heads_ok(p->num_kv_heads, p->head_dim) ||
        p->page_size <= 0 || p->num_pages <= 0 || p->max_pages_per_seq <= 0 || p->max_seq_len < 0 || (!p->lengths && p->max_seq_len == 0))
        return hipErrorInvalidValue;
    const long long cap = static_cast<long long>(p->max_pages_per_seq) * p->page_size;
    if (cap > INT_MAX || p->max_seq_len > cap || (p->max_seq_len > 0 ? p->max_seq_len : cap) > KVQ_MAX_SEQ_LEN ||
        static_cast<long long>(p->batch) * p->max_pages_per_seq > INT_MAX ||
        static_cast<long long>(p->max_pages_per_seq) * p->num_kv_heads > INT_MAX)
        return hipErrorInvalidValue;
    if (!p->block_table || !p->k_pages || !p->k_scale_pages || !p->bounds || !p->bound_scale) return hipErrorInvalidValue;
    kvq::BoundsArgs a{};
    a.pages = page_map(p->block_table, p->page_size, p->max_pages_per_seq, p->num_pages);
    a.start = p->start;
    a.lengths = p->lengths;
    a.k = p->k_pages;
    a.ks = p->k_scale_pages;
    a.bounds = p->bounds;
    a.scale = p->bound_scale;
    a.B = p->batch;
    a.Hkv = p->num_kv_heads;
    a.d = p->head_dim;
    a.max_len = p->max_seq_len > 0 ? p->max_seq_len : static_cast<int>(cap);
    a.heads = kvq::make_fastdiv(static_cast<uint32_t>(p->num_kv_heads));
    const bool vec_ok = ((bits(p->k_pages) | bits(p->bounds)) & 15u) == 0 && page_fits(p->page_size, p->head_dim);
    return checked_call(stream, [&] { return kvq::launch_page_bounds(a, vec_ok, stream); });
}

size_t kvq_sparse_decode_workspace_size(const kvq_sparse_decode_params* p) {
    return sparse_params_ok(p) ? sparse_plan(p).bytes : 0;
}

hipError_t kvq_sparse_decode_launch(const kvq_sparse_decode_params* p, void* workspace, size_t workspace_bytes,
                                    hipStream_t stream) {
    if (!sparse_params_ok(p)) return hipErrorInvalidValue;
    const SparsePlan plan = sparse_plan(p);
    if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes)) return hipErrorInvalidValue;
    const kvq_paged_decode_params& s = p->decode;
    char* base = static_cast<char*>(workspace);
    kvq::SelectArgs a{};
    a.b.pages = page_map(s.block_table, s.page_size, s.max_pages_per_seq, s.num_pages);
    a.b.lengths = s.lengths;
    a.b.k = s.k_pages;
    a.b.ks = s.k_scale_pages;
    a.b.bounds = p->bounds;
    a.b.scale = p->bound_scale;
    a.b.B = s.batch;
    a.b.Hkv = s.num_kv_heads;
    a.b.d = s.head_dim;
    a.b.max_len = max_len_of(s);
    a.q = s.q;
    a.G = s.num_q_heads / s.num_kv_heads;
    a.keep_first = p->keep_first;
    a.keep_last = p->keep_last;
    a.max_selected = p->max_selected;
    a.selected = p->selected;
    a.selected_lengths = p->selected_lengths;
    a.splits = plan.select.splits;
    a.counters = plan.select.splits > 1 ? reinterpret_cast<int*>(base) : nullptr;
    a.keys = plan.select.key_bytes ? reinterpret_cast<unsigned*>(base + plan.keys_at) : nullptr;
    a.key_stride = plan.select.key_stride;
    const hipError_t err = checked_call(stream, [&] { return kvq::launch_select(a, plan.select, plan.vec_ok, stream); });
    if (err != hipSuccess) return err;
    return kvq_paged_decode_launch(&plan.step, workspace, plan.step_bytes, stream);
}

hipError_t kvq_sparse_decode_plan(const kvq_sparse_decode_params* p, kvq_plan_info* info) {
    if (!info || !sparse_params_ok(p)) return hipErrorInvalidValue;
    const SparsePlan plan = sparse_plan(p);
    const hipError_t err = kvq_paged_decode_plan(&plan.step, info);
    info->workspace_bytes = plan.bytes;
    return err;
}

}  // extern "C"
