// kvq_pages_check.cpp -- host-only sweep of the C ABI around a paged cache
// (include/kvq.h, part 7) for the sanitizer builds: workspace sizes and plans
// over shapes up to the ends of their ranges, and calls that must be refused
// before any HIP call.  Pointers are stand-ins that are never followed.
#include <limits.h>
#include <stdio.h>

#include <algorithm>

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
const int kSizes[] = {-1, 0, 1, 2, 15, 16, 17, 64, 1000, 4096, 4097, 65536, 1 << 20, 1 << 24, 1 << 30, INT_MAX};

void maps() {
    for (int B : kSizes)
        for (int size : kSizes)
            for (int pages : kSizes)
                for (int per : kSizes)
                    for (int T : {-1, 0, 1, 5000, INT_MAX}) {
                        kvq_page_map_params p{};
                        p.batch = B, p.page_size = size, p.num_pages = pages, p.max_pages_per_seq = per, p.max_tokens = T;
                        p.new_tokens = at<int32_t>(4096), p.lengths = at<int32_t>(8192), p.block_table = at<int32_t>(1 << 14);
                        p.free_pages = at<int32_t>(1 << 15), p.free_count = at<int32_t>(1 << 16), p.new_lengths = at<int32_t>(8192);
                        p.new_free_count = at<int32_t>(1 << 16), p.granted = at<int32_t>(1 << 17), p.token_offsets = at<int32_t>(1 << 18);
                        const bool ok = B >= 1 && B <= KVQ_PAGE_MAP_MAX_BATCH && size >= 1 && pages >= 1 && per >= 1 && T >= 0 &&
                                        static_cast<long long>(size) * pages <= INT_MAX && static_cast<long long>(size) * per <= INT_MAX &&
                                        static_cast<long long>(B) * per <= INT_MAX;
                        for (int arrays = 0; arrays < 2; arrays++) {
                            p.slot_map = arrays ? at<int32_t>(1 << 19) : nullptr;
                            const size_t n = kvq_page_map_workspace_size(&p);
                            if (!ok) {
                                expect(n == 0, "map: no workspace for a bad shape");
                                expect(kvq_page_map_launch(&p, at<void>(4096), 1 << 20, nullptr) == hipErrorInvalidValue, "map: refused");
                            } else if (n > 0) {
                                expect(kvq_page_map_launch(&p, nullptr, n, nullptr) == hipErrorInvalidValue, "map: wants its workspace");
                                expect(kvq_page_map_launch(&p, at<void>(4096), n - 1, nullptr) == hipErrorInvalidValue, "map: all of it");
                            }
                        }
                    }
}

void slots() {
    for (int T : kSizes)
        for (int H : kSizes)
            for (int d : {0, 1, 20, 64, 4096, 4097})
                for (long long stride : {-1LL, 0LL, 64LL, 1LL << 40, LLONG_MAX}) {
                    kvq_slot_write_params w{};
                    w.tokens = T, w.num_kv_heads = H, w.head_dim = d, w.page_size = 16, w.num_pages = 4, w.dtype = KVQ_DTYPE_F32;
                    w.k_new = at<void>(4096), w.v_new = at<void>(8192), w.slots = at<int32_t>(1 << 14), w.k_pages = at<int8_t>(1 << 15);
                    w.v_pages = at<int8_t>(1 << 16), w.k_scale_pages = at<float>(1 << 17);  // no v_scale_pages: never launched
                    w.k_stride = w.v_stride = stride;
                    expect(kvq_slot_write_launch(&w, nullptr) == hipErrorInvalidValue, "write: refused");
                    kvq_slot_read_params r{};
                    r.tokens = T, r.num_kv_heads = H, r.head_dim = d, r.page_size = 16, r.num_pages = 4, r.dtype = KVQ_DTYPE_F32;
                    r.k_out = at<void>(4096), r.v_out = at<void>(8192), r.slots = at<int32_t>(1 << 14), r.k_pages = at<int8_t>(1 << 15);
                    r.v_pages = at<int8_t>(1 << 16), r.k_scale_pages = r.v_scale_pages = at<float>(1 << 17);
                    r.token_stride = stride, r.head_stride = 0;
                    const bool good = H == 1 && T >= 0 && d >= 1 && d <= 4096 && stride >= 0 &&
                                      (T <= 1 || (stride >= d && stride <= (1LL << 46) / T));  // would be launched
                    if (!good) expect(kvq_slot_read_launch(&r, nullptr) == hipErrorInvalidValue, "read: refused");
                }
}

void sparse() {
    for (int B : kSizes)
        for (int H : {0, 1, 8, 1 << 16, INT_MAX})
            for (int G : {1, 4, 16, 300})
                for (int d : {0, 20, 64, 128, 256, 4097})
                    for (int size : {0, 1, 16, 64, 1 << 24})
                        for (int per : kSizes)
                            for (int budget : {0, 1, 2, 64, 1 << 20, INT_MAX}) {
                                if (static_cast<long long>(H) * G > INT_MAX) continue;
                                // Steps of less than 2^40 tokens (times heads): beyond, nothing fits a GPU.
                                if (static_cast<double>(B) * H * G * std::min(static_cast<double>(size) * per, 1073741824.0) > 1.1e12) continue;
                                kvq_sparse_decode_params p{};
                                kvq_paged_decode_params& s = p.decode;
                                s.batch = B, s.num_kv_heads = H, s.num_q_heads = H * G, s.head_dim = d, s.page_size = size;
                                s.num_pages = 1000, s.max_pages_per_seq = per;
                                s.block_table = at<int32_t>(4096), s.lengths = at<int32_t>(8192), s.q = at<float>(1 << 14);
                                s.k_pages = s.v_pages = at<int8_t>(1 << 16), s.k_scale_pages = s.v_scale_pages = at<float>(1 << 17);
                                s.out = at<float>(1 << 18);
                                p.max_selected = budget, p.keep_first = budget > 2, p.keep_last = 1;
                                p.bounds = at<int8_t>(1 << 19), p.bound_scale = at<float>(1 << 20);
                                p.selected = at<int32_t>(1 << 21), p.selected_lengths = at<int32_t>(1 << 22);
                                kvq_plan_info info{}, dense{};
                                const size_t n = kvq_sparse_decode_workspace_size(&p);
                                const hipError_t err = kvq_sparse_decode_plan(&p, &info);
                                if (kvq_paged_decode_plan(&s, &dense) != hipSuccess || budget < 1)
                                    expect(err == hipErrorInvalidValue && n == 0, "sparse: refuses what the dense step refuses");
                                if (err != hipSuccess) {
                                    expect(n == 0, "sparse: no workspace for a bad shape");
                                    expect(kvq_sparse_decode_launch(&p, at<void>(4096), SIZE_MAX, nullptr) == hipErrorInvalidValue, "sparse: refused");
                                } else {
                                    expect(info.workspace_bytes == n, "sparse: the plan's workspace");
                                    if (n > 0) {
                                        expect(kvq_sparse_decode_launch(&p, nullptr, n, nullptr) == hipErrorInvalidValue, "sparse: wants its workspace");
                                        expect(kvq_sparse_decode_launch(&p, at<void>(4096), n - 1, nullptr) == hipErrorInvalidValue, "sparse: all of it");
                                    }
                                }
                            }
}

void bounds() {
    for (int B : kSizes)
        for (int H : kSizes)
            for (int size : kSizes)
                for (int per : kSizes)
                    for (int len : {-1, 0, 1, 1000, 1 << 30, INT_MAX}) {
                        kvq_page_bounds_params p{};
                        p.batch = B, p.num_kv_heads = H, p.head_dim = 64, p.page_size = size, p.num_pages = 9;
                        p.max_pages_per_seq = per, p.max_seq_len = len;
                        p.block_table = at<int32_t>(4096), p.lengths = at<int32_t>(8192), p.k_pages = at<int8_t>(1 << 14);
                        p.k_scale_pages = at<float>(1 << 15), p.bounds = at<int8_t>(1 << 16);  // no bound_scale: never launched
                        expect(kvq_page_bounds_launch(&p, nullptr) == hipErrorInvalidValue, "bounds: refused");
                    }
}
}  // namespace

int main() {
    maps();
    slots();
    sparse();
    bounds();
    printf("%ld checks, %ld failures\n", checks, failures);
    return failures != 0;
}
