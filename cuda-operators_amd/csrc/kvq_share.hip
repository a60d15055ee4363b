// kvq_share.hip -- gfx950 kernels of shared pages: forks, copies and compaction.
#include <limits.h>

#include "kvq_device.hpp"
#include "kvq_share.hpp"

namespace kvq {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;

__device__ __forceinline__ int pages_of(int tokens, const FastDiv& page) {
    return static_cast<int>(fastdiv(static_cast<uint32_t>(tokens) + page.d - 1, page));
}

// Inclusive scan of one value a thread over a workgroup of kThreads, and the
// total; part is the scan's scratch, free again after the next barrier.
__device__ __forceinline__ int group_scan(int v, int& total, int (&part)[kWaves]) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    v = wave_inclusive_scan(v);
    if (lane == kWave - 1) part[wave] = v;
    __syncthreads();
    const int x = wave_inclusive_scan(lane < kWaves ? part[lane] : 0);
    total = __builtin_amdgcn_readlane(x, kWaves - 1);
    const int w = __builtin_amdgcn_readfirstlane(wave);
    if (w > 0) v += __builtin_amdgcn_readlane(x, w - 1);
    __syncthreads();
    return v;
}

// ---------------------------------------------------------------------------
// Forks.
// ---------------------------------------------------------------------------
// With held(p) = shares[p] + 1 + (table entries that name p afterwards, less
// those before), a page that ends at 0 becomes free, and a row that ends inside
// a page of held > 1 takes a copy unless it is the first of holders that all end
// inside it.  Three launches: entries are counted by atomics on the page (sums
// and a max of integers: any order gives the same), one workgroup decides, in
// page and row order by prefix sums, and the rows are written.

struct ForkRow {
    int parent;  // -1: none
    int len, n;  // tokens before, and of the parent to keep
};
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int b) {
    ForkRow r;
    r.parent = a.parents[b];
    if (r.parent < 0 || r.parent >= a.B) r.parent = -1;
    r.len = min(max(a.lengths[b], 0), a.cap);
    r.n = r.parent < 0 ? 0 : r.parent == b ? r.len : min(max(a.lengths[r.parent], 0), a.cap);
    if (a.keep) r.n = min(r.n, max(a.keep[b], 0));
    return r;
}

// Entries of one row: workgroups blockIdx.y of row blockIdx.x.
__global__ __launch_bounds__(256) void fork_count_kernel(const ForkArgs a) {
    const int b = blockIdx.x;
    const ForkRow r = fork_row(a, b);
    const int before = pages_of(r.len, a.page), now = pages_of(r.n, a.page);
    const int32_t* old = a.table + static_cast<size_t>(b) * a.max_pages;
    const int32_t* from = a.table + static_cast<size_t>(max(r.parent, 0)) * a.max_pages;
    auto in_pool = [&](int id) { return id >= 0 && id < a.num_pages; };
    const int step = gridDim.y * 256;
    const bool stays = r.parent == b;
    for (int j = blockIdx.y * 256 + threadIdx.x; j < max(before, now); j += step) {
        if (j < before && !(stays && j < now)) {
            const int id = old[j];
            if (in_pool(id)) atomicSub(a.delta + id, 1);
        }
        if (j < now && !stays) {
            const int id = from[j];
            a.stage[static_cast<size_t>(b) * a.max_pages + j] = id;
            if (in_pool(id)) atomicAdd(a.delta + id, 1);
        }
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        a.want[b] = r.n;
        const int whole = static_cast<int>(fastdiv(static_cast<uint32_t>(r.n), a.page));
        if (whole < now) {  // ends inside a page
            const int id = from[whole];
            if (in_pool(id)) {
                atomicAdd(a.writers + id, 1);
                atomicMax(a.first + id, a.B - b);
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void fork_decide_kernel(const ForkArgs a) {
    __shared__ int s_part[kWaves];
    const int t = threadIdx.x;
    const int F = min(max(*a.free_count, 0), a.num_pages);

    // Pages that have become free.
    int freed = 0;
    const unsigned P = static_cast<unsigned>(a.num_pages);
    for (unsigned p0 = 0; p0 < P; p0 += kThreads) {
        const unsigned p = p0 + t;
        int gone = 0;
        if (p < P) {
            const int delta = a.delta[p];
            gone = delta < 0 && a.shares[p] + 1 + delta <= 0;
        }
        int total;
        const int at = freed + group_scan(gone, total, s_part) - gone;
        if (gone) a.freed[at] = static_cast<int>(p);
        freed += total;
    }
    __syncthreads();
    const long long have = static_cast<long long>(F) + freed;
    auto stack_at = [&](long long i) { return i < F ? a.free_pages[i] : a.freed[i - F]; };

    // Rows that need a page of their own.
    int copies = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
        const int b = b0 + t;
        int need = 0, page = -1, n = 0;
        if (b < a.B) {
            n = a.want[b];
            const int whole = static_cast<int>(fastdiv(static_cast<uint32_t>(n), a.page));
            if (whole * static_cast<int>(a.page.d) < n) {
                const int parent = a.parents[b];
                page = a.table[static_cast<size_t>(parent) * a.max_pages + whole];
                if (page >= 0 && page < a.num_pages) {
                    const int held = a.shares[page] + 1 + a.delta[page];
                    need = held > 1 && !(held <= a.writers[page] && a.first[page] == a.B - b);
                }
            }
        }
        int total;
        const int turn = copies + group_scan(need, total, s_part) - need;
        copies += total;
        if (b < a.B) {
            int dst = -1;
            if (need) {
                if (turn < have) dst = stack_at(have - 1 - turn);
                else n -= n - static_cast<int>(fastdiv(static_cast<uint32_t>(n), a.page) * a.page.d);
            }
            a.copy_src[b] = dst < 0 ? -1 : page;
            a.copy_dst[b] = dst;
            // A row's place in `want` afterwards: its tokens, and whether it has been cut to whole pages.
            a.want[b] = n;
        }
    }
    const long long left = have - min(static_cast<long long>(copies), have);
    __syncthreads();

    // The stack, shares, and the workspace as it was.
    for (unsigned i = t; i < static_cast<unsigned>(freed); i += kThreads) {
        const long long at = static_cast<long long>(F) + i;
        if (at < left && at < a.num_pages) a.free_pages[at] = a.freed[i];
        a.freed[i] = 0;
    }
    for (unsigned p = t; p < P; p += kThreads) {
        const int delta = a.delta[p], writers = a.writers[p];
        int shares = a.shares[p];
        if (delta != 0 || writers != 0) {
            const int held = shares + 1 + delta;
            const int leave = held > 1 ? writers - (held <= writers ? 1 : 0) : 0;
            shares = max(held - leave - 1, 0);
            a.delta[p] = 0;
            a.writers[p] = 0;
            a.first[p] = 0;
        }
        a.new_shares[p] = shares;
    }
    __syncthreads();
    for (int b = t; b < a.B; b += kThreads) {
        const int dst = a.copy_dst[b];
        if (dst >= 0 && dst < a.num_pages) a.new_shares[dst] = 0;
    }
    if (t == 0) *a.new_free_count = static_cast<int>(min(left, static_cast<long long>(a.num_pages)));
}

__global__ __launch_bounds__(256) void fork_write_kernel(const ForkArgs a) {
    const int b = blockIdx.x;
    const int n = a.want[b];
    const int pages = pages_of(n, a.page);
    const int dst = a.copy_dst[b];
    const bool stays = a.parents[b] == b;
    const bool in_place = a.table == a.new_table;
    int32_t* row = a.new_table + static_cast<size_t>(b) * a.max_pages;
    int* stage = a.stage + static_cast<size_t>(b) * a.max_pages;
    const int step = gridDim.y * 256;
    // Staged entries go back to 0, those of a page that was cut off too.
    const int end = min(pages + 1, a.max_pages);
    for (int j = blockIdx.y * 256 + threadIdx.x; j < end; j += step) {
        int id = 0;
        if (!stays) {
            id = stage[j];
            stage[j] = 0;
        } else if (!in_place && j < pages) {
            id = a.table[static_cast<size_t>(b) * a.max_pages + j];
        }
        if (j >= pages) continue;
        if (dst >= 0 && j == pages - 1) row[j] = dst;
        else if (!stays || !in_place) row[j] = id;
    }
}

// want goes back to 0 only when every row's workgroups have read it.
__global__ __launch_bounds__(256) void fork_lengths_kernel(const ForkArgs a) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= a.B) return;
    a.new_lengths[b] = a.want[b];
    a.want[b] = 0;
}

// ---------------------------------------------------------------------------
// Copies.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void page_copy_kernel(const CopyArgs a) {
    const int i = blockIdx.x;
    const int layer = blockIdx.y;
    const int src = a.src[i], dst = a.dst[i];
    if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages) return;
#pragma unroll
    for (int k = 0; k < CopyArgs::kArrays; k++) {
        if (!a.base[k]) continue;
        const char* x = a.base[k] + (static_cast<size_t>(layer) * a.num_pages + src) * a.bytes[k];
        char* y = a.base[k] + (static_cast<size_t>(layer) * a.num_pages + dst) * a.bytes[k];
        for (size_t j = threadIdx.x; j < a.bytes[k]; j += 256) y[j] = x[j];
    }
}

// ---------------------------------------------------------------------------
// Compaction.
// ---------------------------------------------------------------------------
// A page's state: kFree, 0 in use, or where it moves to, + 1.
constexpr int kFree = -1;

__global__ __launch_bounds__(256) void compact_mark_kernel(const CompactArgs a) {
    const unsigned F = static_cast<unsigned>(min(max(*a.free_count, 0), a.num_pages));
    const unsigned me = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
    for (unsigned i = me; i < F; i += step) {
        const int p = a.free_pages[i];
        if (p >= 0 && p < a.num_pages) a.state[p] = kFree;
    }
    for (unsigned i = me; i < static_cast<unsigned>(a.max_moves); i += step) a.copy_src[i] = a.copy_dst[i] = -1;
}

__global__ __launch_bounds__(kThreads) void compact_plan_kernel(const CompactArgs a) {
    __shared__ int s_part[kWaves];
    const unsigned t = threadIdx.x;
    const unsigned P = static_cast<unsigned>(a.num_pages);
    int total, free_total = 0;
    for (unsigned p0 = 0; p0 < P; p0 += kThreads) {
        group_scan(p0 + t < P && a.state[p0 + t] == kFree, total, s_part);
        free_total += total;
    }
    const unsigned used = P - free_total;
    // Free pages before `used`, ascending, then pages in use from there on, descending.
    int holes = 0;
    for (unsigned p0 = 0; p0 < used; p0 += kThreads) {
        const unsigned p = p0 + t;
        const int hole = p < used && a.state[p] == kFree;
        const int at = holes + group_scan(hole, total, s_part) - hole;
        if (hole && at < a.max_moves) {
            a.copy_dst[at] = static_cast<int>(p);
            a.taken[p] = 1;
        }
        holes += total;
    }
    const int moves = min(holes, a.max_moves);
    int highs = 0;
    for (unsigned p0 = 0; p0 < P - used; p0 += kThreads) {
        const unsigned back = p0 + t;
        const int high = back < P - used && a.state[P - 1 - back] != kFree;
        const int at = highs + group_scan(high, total, s_part) - high;
        if (high && at < moves) a.copy_src[at] = static_cast<int>(P - 1 - back);
        highs += total;
    }
    __syncthreads();
    for (unsigned i = t; i < static_cast<unsigned>(moves); i += kThreads) {
        const int src = a.copy_src[i];
        if (src >= 0) a.state[src] = a.copy_dst[i] + 1;
    }
    if (t == 0) *a.moved = moves;
    __syncthreads();
    // The stack afterwards, descending.
    int above = 0;
    for (unsigned p0 = 0; p0 < P; p0 += kThreads) {
        int is_free = 0;
        const unsigned p = P - 1 - (p0 + t);
        if (p0 + t < P) {
            const int s = a.state[p];
            is_free = s > 0 || (s == kFree && !a.taken[p]);
        }
        const int at = above + group_scan(is_free, total, s_part) - is_free;
        if (is_free) a.new_free_pages[at] = static_cast<int>(p);
        above += total;
    }
}

__global__ __launch_bounds__(256) void compact_table_kernel(const CompactArgs a) {
    const int b = blockIdx.x;
    const int pages = pages_of(min(max(a.lengths[b], 0), a.cap), a.page);
    const int32_t* row = a.table + static_cast<size_t>(b) * a.max_pages;
    int32_t* out = a.new_table + static_cast<size_t>(b) * a.max_pages;
    for (int j = blockIdx.y * 256 + threadIdx.x; j < pages; j += gridDim.y * 256) {
        int id = row[j];
        if (id >= 0 && id < a.num_pages) {
            const int s = a.state[id];
            if (s > 0) id = s - 1;
        }
        out[j] = id;
    }
}

__global__ __launch_bounds__(256) void compact_shares_kernel(const CompactArgs a) {
    for (unsigned p = blockIdx.x * 256 + threadIdx.x; p < static_cast<unsigned>(a.num_pages); p += gridDim.x * 256) {
        const int s = a.state[p];
        if (a.shares) {
            if (s > 0) {  // moved: its number goes along, and it is free
                a.new_shares[s - 1] = a.shares[p];
                a.new_shares[p] = 0;
            } else if (!a.taken[p]) {  // (a page moved to gets its number from where it came)
                a.new_shares[p] = s == kFree ? 0 : a.shares[p];
            }
        }
        a.state[p] = 0;
        a.taken[p] = 0;
    }
}

unsigned blocks(long long n, int per, unsigned most) {
    const long long g = (n + per - 1) / per;
    return static_cast<unsigned>(g < 1 ? 1 : g > most ? most : g);
}

}  // namespace

size_t fork_workspace(const ForkArgs& a) {
    return sizeof(int) * (4 * static_cast<size_t>(a.num_pages) + a.B + static_cast<size_t>(a.B) * a.max_pages);
}
void fork_place(ForkArgs& a, void* workspace) {
    a.delta = static_cast<int*>(workspace);
    a.writers = a.delta + a.num_pages;
    a.first = a.writers + a.num_pages;
    a.freed = a.first + a.num_pages;
    a.want = a.freed + a.num_pages;
    a.stage = a.want + a.B;
}

hipError_t launch_page_fork(const ForkArgs& a, hipStream_t stream) {
    const dim3 rows(static_cast<unsigned>(a.B), blocks(a.max_pages, 256, 64));
    hipLaunchKernelGGL(fork_count_kernel, rows, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(fork_decide_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(fork_write_kernel, rows, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(fork_lengths_kernel, dim3(blocks(a.B, 256, 1 << 20)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_page_copy(const CopyArgs& a, hipStream_t stream) {
    if (a.n == 0) return hipSuccess;
    hipLaunchKernelGGL(page_copy_kernel, dim3(static_cast<unsigned>(a.n), static_cast<unsigned>(a.layers)), dim3(256), 0,
                       stream, a);
    return hipGetLastError();
}

size_t compact_workspace(const CompactArgs& a) { return sizeof(int) * 2 * static_cast<size_t>(a.num_pages); }
void compact_place(CompactArgs& a, void* workspace) {
    a.state = static_cast<int*>(workspace);
    a.taken = a.state + a.num_pages;
}

hipError_t launch_page_compact(const CompactArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(compact_mark_kernel, dim3(blocks(max(a.num_pages, a.max_moves), 256, 1024)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(compact_table_kernel, dim3(static_cast<unsigned>(a.B), blocks(a.max_pages, 256, 64)), dim3(256), 0,
                       stream, a);
    hipLaunchKernelGGL(compact_shares_kernel, dim3(blocks(a.num_pages, 256, 1024)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace kvq
