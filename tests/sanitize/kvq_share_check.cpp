// kvq_share_check.cpp -- host-only sweep of the C ABI of chunk attention and shared
// pages (include/kvq.h, part 8) for the sanitizer builds: workspace sizes over
// shapes up to the ends of their ranges, and calls that must be refused before any
// HIP call.  Pointers are stand-ins that are never followed.
#include <limits.h>
#include <stdio.h>

#include "../../include/kvq.h"

namespace {
long checks = 0, failures = 0;
void expect(bool ok, const char* what) {
    checks++;
    if (!ok) {
        failures++;
        fprintf(stderr, "FAILED: %s\n", what);
    }
}
template <class T>
T* at(size_t x) {
    return reinterpret_cast<T*>(x);
}
const int kSizes[] = {-1, 0, 1, 2, 17, 64, 1000, 4096, 4097, 1 << 20, 1 << 28, INT_MAX};

void chunks() {
    for (int B : kSizes)
        for (int T : kSizes)
            for (int H : {0, 1, 8, 1 << 12, 1 << 20})
                for (int G : {1, 5, 128, 129})
                    for (int per : kSizes)
                        for (int d : {1, 20, 64, 72, 128, 192, 256, 264, 4096, 4097})
                            for (int dtype = 0; dtype < 2; dtype++) {
                                kvq_chunk_attention_params p{};
                                p.batch = B, p.num_q_heads = H * G, p.num_kv_heads = H, p.head_dim = d, p.page_size = 16;
                                p.num_pages = 1000, p.max_pages_per_seq = per, p.tokens = T, p.dtype = dtype, p.causal = 1;
                                p.token_offsets = at<int32_t>(4096), p.lengths = at<int32_t>(8192), p.block_table = at<int32_t>(1 << 14);
                                p.q = at<void>(1 << 20), p.out = at<void>(1 << 21);
                                p.k_pages = at<int8_t>(1 << 22), p.v_pages = at<int8_t>(1 << 23);
                                p.k_scale_pages = at<float>(1 << 24), p.v_scale_pages = at<float>(1 << 25);
                                const bool ok = B >= 1 && B <= KVQ_CHUNK_MAX_BATCH && H >= 1 && d >= 1 && d <= KVQ_MAX_HEAD_DIM && per >= 1 &&
                                                16LL * per <= KVQ_MAX_SEQ_LEN && static_cast<long long>(B) * per <= INT_MAX && T >= 0 &&
                                                static_cast<long long>(T) * H * G <= INT_MAX;
                                const size_t n = kvq_chunk_attention_workspace_size(&p);
                                expect(n <= (1u << 18) + 256u * 256u * 258u * 4u, "chunk: a workspace of a bounded size");
                                if (!ok) {
                                    expect(n == 0, "chunk: no workspace for a bad shape");
                                    expect(kvq_chunk_attention_launch(&p, at<void>(4096), 1u << 30, nullptr) == hipErrorInvalidValue, "chunk: refused");
                                } else if (n > 0) {
                                    expect(kvq_chunk_attention_launch(&p, nullptr, n, nullptr) == hipErrorInvalidValue, "chunk: wants its workspace");
                                    expect(kvq_chunk_attention_launch(&p, at<void>(4096), n - 1, nullptr) == hipErrorInvalidValue, "chunk: all of it");
                                }
                            }
}

void pages() {
    for (int B : kSizes)
        for (int size : kSizes)
            for (int num : kSizes)
                for (int per : kSizes) {
                    int32_t* const x = at<int32_t>(1 << 16);
                    const bool ok = B >= 1 && B <= KVQ_FORK_MAX_BATCH && size >= 1 && num >= 1 && per >= 1 && static_cast<long long>(size) * num <= INT_MAX &&
                                    static_cast<long long>(size) * per <= INT_MAX && static_cast<long long>(B) * per <= INT_MAX;
                    kvq_page_fork_params f{B, size, num, per, x, x, x, x, x, x, x, x, x, x, x, x, x};
                    kvq_page_compact_params c{B, size, num, per, 5, x, x, x, x, x, x, x, x, x, x, x};
                    const size_t nf = kvq_page_fork_workspace_size(&f), nc = kvq_page_compact_workspace_size(&c);
                    expect((nf > 0) == ok && (nc > 0) == ok, "pages: workspaces of the shapes that are good");
                    expect(kvq_page_fork_launch(&f, ok ? nullptr : x, size_t(1) << 50, nullptr) == hipErrorInvalidValue, "fork: refused");
                    expect(kvq_page_compact_launch(&c, ok ? nullptr : x, size_t(1) << 50, nullptr) == hipErrorInvalidValue, "compact: refused");
                    if (ok) {
                        expect(kvq_page_fork_launch(&f, x, nf - 1, nullptr) == hipErrorInvalidValue, "fork: all of its workspace");
                        expect(kvq_page_compact_launch(&c, x, nc - 1, nullptr) == hipErrorInvalidValue, "compact: all of its workspace");
                    }
                    for (int d : {0, 64, 4097})
                        for (int layers : {0, 1, 65536}) {
                            kvq_page_copy_params p{1 << 24, layers, 2, d, size, num, x, x, at<int8_t>(64), at<int8_t>(64), at<float>(64), at<float>(64), nullptr, nullptr};
                            expect(kvq_page_copy_launch(&p, nullptr) == hipErrorInvalidValue, "copy: refused");
                        }
                }
}
}  // namespace

int main() {
    chunks();
    pages();
    expect(kvq_chunk_attention_launch(nullptr, nullptr, 0, nullptr) == hipErrorInvalidValue, "null");
    expect(kvq_page_copy_launch(nullptr, nullptr) == hipErrorInvalidValue, "null");
    printf("%ld checks, %ld failures\n", checks, failures);
    return failures ? 1 : 0;
}
