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
// page and row order by prefix sums, and the rows are written.  Bound by latency: 16 rows
// on pages of 64 tokens take 11.5 to 13.7 us a call, 256 of up to 4096 tokens on pages of 16
// 17.7; count, decide and write are 3.6, 4.7 and 2.8 us, and 6.7, 8.8 and 3.0.

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

// Pages that have become free, kPer a thread and pass, so that a pass of 8192
// pages costs two barriers; then the rows, in order.
__global__ __launch_bounds__(kThreads) void fork_decide_kernel(const ForkArgs a) {
    constexpr int kPer = 8;
    __shared__ int s_part[kWaves];
    const unsigned t = threadIdx.x;
    const int F = min(max(*a.free_count, 0), a.num_pages);
    const unsigned P = static_cast<unsigned>(a.num_pages);
    int freed = 0;
    for (unsigned p0 = 0; p0 < P; p0 += kThreads * kPer) {
        int delta[kPer], gone[kPer], mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const unsigned p = p0 + t * kPer + i;
            delta[i] = p < P ? a.delta[p] : 0;
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            gone[i] = delta[i] < 0 && a.shares[p0 + t * kPer + i] + 1 + delta[i] <= 0;
            mine += gone[i];
        }
        int total;
        int at = freed + group_scan(mine, total, s_part) - mine;
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (gone[i]) a.freed[at++] = static_cast<int>(p0 + t * kPer + i);
        freed += total;
    }
    __syncthreads();
    const long long have = static_cast<long long>(F) + freed;
    auto stack_at = [&](long long i) { return i < F ? a.free_pages[i] : a.freed[i - F]; };

    int copies = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
        const int b = b0 + static_cast<int>(t);
        int need = 0, page = -1, n = 0;
        if (b < a.B) {
            n = a.want[b];
            a.want[b] = 0;
            const int whole = static_cast<int>(fastdiv(static_cast<uint32_t>(n), a.page));
            if (whole * static_cast<int>(a.page.d) < n) {
                page = a.table[static_cast<size_t>(a.parents[b]) * a.max_pages + whole];
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
                else n = static_cast<int>(fastdiv(static_cast<uint32_t>(n), a.page) * a.page.d);
            }
            a.copy_src[b] = dst < 0 ? -1 : page;
            a.copy_dst[b] = dst;
            a.new_lengths[b] = n;
        }
    }
    const long long left = have - min(static_cast<long long>(copies), have);
    __syncthreads();
    for (unsigned i = t; i < static_cast<unsigned>(freed); i += kThreads) {
        const long long at = static_cast<long long>(F) + i;
        if (at < left && at < a.num_pages) a.free_pages[at] = a.freed[i];
        a.freed[i] = 0;
    }
    if (t == 0) *a.new_free_count = static_cast<int>(min(left, static_cast<long long>(a.num_pages)));
}

// Rows (workgroups blockIdx.y of row blockIdx.x), then in the rows of the grid
// behind them the pages' shares and the workspace as it was.
__global__ __launch_bounds__(256) void fork_write_kernel(const ForkArgs a) {
    if (blockIdx.x >= static_cast<unsigned>(a.B)) {
        const unsigned groups = (gridDim.x - a.B) * gridDim.y;
        for (unsigned p = ((blockIdx.x - a.B) * gridDim.y + blockIdx.y) * 256 + threadIdx.x; p < static_cast<unsigned>(a.num_pages);
             p += groups * 256) {
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
        return;
    }
    const int b = blockIdx.x;
    const int pages = pages_of(a.new_lengths[b], a.page);
    const int dst = a.copy_dst[b];
    const bool stays = a.parents[b] == b;
    const bool in_place = a.table == a.new_table;
    int32_t* row = a.new_table + static_cast<size_t>(b) * a.max_pages;
    int* stage = a.stage + static_cast<size_t>(b) * a.max_pages;
    // Staged entries go back to 0, that of a page that was cut off too.
    const int end = min(pages + 1, a.max_pages);
    for (int j = blockIdx.y * 256 + threadIdx.x; j < end; j += gridDim.y * 256) {
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

// ---------------------------------------------------------------------------
// Copies.
// ---------------------------------------------------------------------------
// A pair's arrays in one layer are laid end to end in pieces of 16 bytes (or 4, or
// 1, where an array's place or page size is not a multiple); a workgroup takes
// kCopyLoads of a thread's at a time, whose loads go out together.  Bound by HBM: 48
// pairs of pages of 64 tokens in 32 layers of 8 heads, d = 128, 42 of them to copy, from 23
// pages (281 MB read and written): 75 us a call, 65 to 69 the kernel (4.1 TB/s or more); a
// large copy of as much at 5.08 TB/s would take 55.
constexpr int kCopyLoads = 4;
// Pairs of all layers up to which each has workgroups of its own; more go to this many, 16 for
// each that fits the chip.  50,000 pairs of 4.4 KB in 32 layers, none, 1000 or 12,000 of them to
// copy: 32, 59 and 375 us, with a workgroup a pair 518, 560 and 837; but 48 of 135 KB in 32 layers
// 73, with workgroups of their own 67.
constexpr unsigned kCopyGroups = 1 << 15;

template <class T>
__device__ __forceinline__ void copy_page(const CopyArgs& a, unsigned layer, int src, int dst) {
    const size_t first = static_cast<size_t>(layer) * a.num_pages;
    for (size_t p0 = static_cast<size_t>(blockIdx.y) * (256 * kCopyLoads); p0 < a.pieces;
         p0 += static_cast<size_t>(gridDim.y) * (256 * kCopyLoads)) {
        T x[kCopyLoads];
        char* to[kCopyLoads];
#pragma unroll
        for (int u = 0; u < kCopyLoads; u++) {
            size_t p = p0 + u * 256 + threadIdx.x;
            to[u] = nullptr;
            if (p >= a.pieces) continue;
            char* base = a.base[0];
            size_t bytes = a.bytes[0], before = 0;
#pragma unroll
            for (int k = 1; k < CopyArgs::kArrays; k++)
                if (p >= a.begin[k]) base = a.base[k], bytes = a.bytes[k], before = a.begin[k];
            const size_t at = (p - before) * sizeof(T);
            x[u] = *reinterpret_cast<const T*>(base + (first + src) * bytes + at);
            to[u] = base + (first + dst) * bytes + at;
        }
#pragma unroll
        for (int u = 0; u < kCopyLoads; u++)
            if (to[u]) *reinterpret_cast<T*>(to[u]) = x[u];
    }
}

// A workgroup (or some, along y) for each (layer, pair).
template <class T>
__global__ __launch_bounds__(256) void page_copy_kernel(const CopyArgs a) {
    const unsigned unit = blockIdx.x;
    const unsigned layer = fastdiv(unit, a.pairs);
    const int i = static_cast<int>(unit - layer * a.n);
    const int src = a.src[i], dst = a.dst[i];
    if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages) return;
    copy_page<T>(a, layer, src, dst);
}

// Long lists, which may be mostly -1 (a compaction's): workgroups take every so many a pair,
// and read 64 of theirs at once.
template <class T>
__global__ __launch_bounds__(256) void page_copy_list_kernel(const CopyArgs a) {
    const unsigned lane = threadIdx.x & (kWave - 1);
    const unsigned units = static_cast<unsigned>(a.n) * a.layers;
    for (unsigned u0 = blockIdx.x; u0 < units; u0 += gridDim.x * kWave) {
        const unsigned unit = u0 + lane * gridDim.x;
        unsigned layer = 0;
        int src = -1, dst = -1;
        if (unit < units) {
            layer = fastdiv(unit, a.pairs);
            src = a.src[unit - layer * a.n];
            dst = a.dst[unit - layer * a.n];
        }
        unsigned long long live = __builtin_amdgcn_ballot_w64(src >= 0 && src < a.num_pages && dst >= 0 && dst < a.num_pages);
        for (; live; live &= live - 1) {
            const int l = __builtin_ctzll(live);
            copy_page<T>(a, __builtin_amdgcn_readlane(layer, l), __builtin_amdgcn_readlane(src, l), __builtin_amdgcn_readlane(dst, l));
        }
    }
}

// ---------------------------------------------------------------------------
// Compaction.
// ---------------------------------------------------------------------------
// Moves are decided by one workgroup: the i-th free page from below takes the i-th
// page in use from above, as long as it lies lower, and both lists are prefix sums.
// Bound by launches and latency: 16 rows of up to 2048 tokens on pages of 64 take 9.7 to 12.7
// us a call, 256 of up to 4096 on pages of 16 (50,000 pages) 11.7 to 12.4 (32.9
// with all lists written by the one workgroup that scans, and one load at a time), 64 on 261,000
// pages 36.  Above 2^18 pages the one workgroup does all: 264,000 take 523 us, 524,000 1075.
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

// The same with the free pages as bits in LDS, for pools of up to kBitPages: one
// scan each over the words instead of one over the pages.  Both sets of free pages,
// before and after the moves, are left in the workspace with counts for each word, from
// which the launches behind this one write the lists, a page a thread.
constexpr int kBitPages = 1 << 18;  // 32 KB of LDS

__global__ __launch_bounds__(kThreads) void compact_bits_kernel(const CompactArgs a) {
    extern __shared__ unsigned s_bits[];
    __shared__ int s_part[kWaves];
    const int t = threadIdx.x;
    const int P = a.num_pages, words = (P + 31) / 32, per = (words + kThreads - 1) / kThreads;
    const int w0 = min(t * per, words), w1 = min(w0 + per, words);
    for (int w = t; w < words; w += kThreads) s_bits[w] = 0;
    __syncthreads();
    const int F = min(max(*a.free_count, 0), P);
    constexpr int kLoads = 8;  // on their way together
    for (int i = t; i < F; i += kLoads * kThreads) {
        int p[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; j++) p[j] = i + j * kThreads < F ? a.free_pages[i + j * kThreads] : -1;
#pragma unroll
        for (int j = 0; j < kLoads; j++)
            if (p[j] >= 0 && p[j] < P) atomicOr(&s_bits[p[j] >> 5], 1u << (p[j] & 31));
    }
    __syncthreads();
    auto valid = [&](int w) { return w == words - 1 && (P & 31) ? (1u << (P & 31)) - 1 : ~0u; };
    int count = 0, total;
    for (int w = w0; w < w1; w++) {
        a.before[w] = s_bits[w];
        count += __popc(s_bits[w]);
    }
    group_scan(count, total, s_part);
    const int used = P - total;
    auto below = [&](int w) {  // the word's pages before `used`
        const int n = used - 32 * w;
        return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
    };
    int holes = 0, highs = 0;
    for (int w = w0; w < w1; w++) {
        holes += __popc(s_bits[w] & below(w));
        highs += __popc(~s_bits[w] & ~below(w) & valid(w));
    }
    int all_holes, all_highs;
    int hole = group_scan(holes, all_holes, s_part) - holes;
    int high = group_scan(highs, all_highs, s_part);
    high = all_highs - (high - highs);  // pages that could move, from this thread's first word on
    const int moves = min(all_holes, a.max_moves);
    for (int w = w0; w < w1; w++) {
        // The lowest of the free pages are moved to, the highest of those in use moved;
        // in one word each some may stay.
        unsigned x = s_bits[w] & below(w), y = ~s_bits[w] & ~below(w) & valid(w);
        const int nx = static_cast<int>(__popc(x)), ny = static_cast<int>(__popc(y));  // (__popc is unsigned)
        a.hole[w] = hole;
        hole += nx;
        for (int i = min(hole - moves, nx); i > 0; i--) x &= ~(1u << (31 - __clz(x)));
        high -= ny;
        a.high[w] = high;
        for (int i = min(high + ny - moves, ny); i > 0; i--) y &= y - 1;
        s_bits[w] = (s_bits[w] & ~x) | y;
        a.after[w] = s_bits[w];
    }
    if (t == 0) *a.moved = moves;
    // Where the pages go in the stack afterwards, descending.
    count = 0;
    for (int w = w0; w < w1; w++) count += __popc(s_bits[w]);
    int at = group_scan(count, total, s_part) - count;  // free pages before this thread's
    for (int w = w0; w < w1; w++) {
        a.place[w] = total - 1 - at;
        at += __popc(s_bits[w]);
    }
}

// Tables (rows of the grid), shares, the stack, and the lists' ends behind them.  A page is
// moved if it was in use before and is free now, to the page of the same rank among
// those that were free and are in use now.
__device__ __forceinline__ bool has(const unsigned* set, unsigned p) { return (set[p >> 5] >> (p & 31)) & 1; }
__device__ __forceinline__ int move_of(const CompactArgs& a, unsigned p) {  // of a page that moves, from the highest
    const unsigned w = p >> 5;
    return a.high[w] + __popc(~a.before[w] & a.after[w] & ~((2u << (p & 31)) - 1));
}
__global__ __launch_bounds__(256) void compact_bits_apply_kernel(const CompactArgs a) {
    const int moves = *a.moved;
    if (blockIdx.x >= static_cast<unsigned>(a.B)) {
        const unsigned groups = (gridDim.x - a.B) * gridDim.y;
        const unsigned me = ((blockIdx.x - a.B) * gridDim.y + blockIdx.y) * 256 + threadIdx.x;
        for (unsigned i = me + moves; i < static_cast<unsigned>(a.max_moves); i += groups * 256) a.copy_src[i] = a.copy_dst[i] = -1;
        for (unsigned p = me; p < static_cast<unsigned>(a.num_pages); p += groups * 256) {
            const bool was = has(a.before, p), is = has(a.after, p);
            if (is) a.new_free_pages[a.place[p >> 5] - __popc(a.after[p >> 5] & ((1u << (p & 31)) - 1))] = static_cast<int>(p);
            if (!a.shares) continue;
            if (!was && is) {  // moved: its number goes along
                a.new_shares[a.copy_dst[move_of(a, p)]] = a.shares[p];
                a.new_shares[p] = 0;
            } else if (was == is) {  // (a page moved to gets its number from where it came)
                a.new_shares[p] = is ? 0 : a.shares[p];
            }
        }
        return;
    }
    const int b = blockIdx.x;
    const int pages = pages_of(min(max(a.lengths[b], 0), a.cap), a.page);
    const int32_t* row = a.table + static_cast<size_t>(b) * a.max_pages;
    int32_t* out = a.new_table + static_cast<size_t>(b) * a.max_pages;
    for (int j = blockIdx.y * 256 + threadIdx.x; j < pages; j += gridDim.y * 256) {
        int id = row[j];
        if (id >= 0 && id < a.num_pages && !has(a.before, id) && has(a.after, id)) id = a.copy_dst[move_of(a, id)];
        out[j] = id;
    }
}

__global__ __launch_bounds__(256) void compact_bits_moves_kernel(const CompactArgs a) {
    for (unsigned p = blockIdx.x * 256 + threadIdx.x; p < static_cast<unsigned>(a.num_pages); p += gridDim.x * 256) {
        const bool was = has(a.before, p), is = has(a.after, p);
        if (!was && is) a.copy_src[move_of(a, p)] = static_cast<int>(p);
        const unsigned w = p >> 5;
        if (was && !is) a.copy_dst[a.hole[w] + __popc(a.before[w] & ~a.after[w] & ((1u << (p & 31)) - 1))] = static_cast<int>(p);
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
    const unsigned along = blocks(a.max_pages, 256, 64);
    const unsigned pages = blocks(blocks(a.num_pages, 256, 4096), static_cast<int>(along), 4096);
    hipLaunchKernelGGL(fork_count_kernel, dim3(static_cast<unsigned>(a.B), along), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(fork_decide_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(fork_write_kernel, dim3(static_cast<unsigned>(a.B) + pages, along), dim3(256), 0, stream, a);
    return hipGetLastError();
}

namespace {
template <class T>
hipError_t launch_copy(CopyArgs a, hipStream_t stream) {
    a.pieces = 0;
    for (int k = 0; k < CopyArgs::kArrays; k++) {
        a.begin[k] = a.pieces;
        if (a.base[k]) a.pieces += a.bytes[k] / sizeof(T);
    }
    a.pairs = make_fastdiv(static_cast<uint32_t>(a.n));
    const unsigned units = static_cast<unsigned>(a.n) * a.layers;
    if (units <= kCopyGroups) {
        const dim3 grid(units, blocks(static_cast<long long>(a.pieces), 256 * kCopyLoads, 1024));
        hipLaunchKernelGGL((page_copy_kernel<T>), grid, dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((page_copy_list_kernel<T>), dim3(kCopyGroups), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}
}  // namespace

hipError_t launch_page_copy(const CopyArgs& a, hipStream_t stream) {
    if (a.n == 0) return hipSuccess;
    size_t all = 0;
    for (int k = 0; k < CopyArgs::kArrays; k++)
        if (a.base[k]) all |= reinterpret_cast<uintptr_t>(a.base[k]) | a.bytes[k];
    if (all % 16 == 0) return launch_copy<int4>(a, stream);
    if (all % 4 == 0) return launch_copy<int>(a, stream);
    return launch_copy<char>(a, stream);
}

// Bitmaps before and after and three counts a word; or the larger pools' two arrays.
size_t compact_workspace(const CompactArgs& a) {
    const size_t P = static_cast<size_t>(a.num_pages);
    return sizeof(int) * (a.num_pages <= kBitPages ? 5 * ((P + 31) / 32) : 2 * P);
}
void compact_place(CompactArgs& a, void* workspace) {
    a.state = static_cast<int*>(workspace);
    a.taken = a.state + a.num_pages;
    a.before = static_cast<unsigned*>(workspace);
    a.after = a.before + (a.num_pages + 31) / 32;
    a.place = reinterpret_cast<int*>(a.after + (a.num_pages + 31) / 32);
    a.hole = a.place + (a.num_pages + 31) / 32;
    a.high = a.hole + (a.num_pages + 31) / 32;
}

hipError_t launch_page_compact(const CompactArgs& a, hipStream_t stream) {
    const unsigned along = blocks(a.max_pages, 256, 64);
    if (a.num_pages <= kBitPages) {
        const unsigned pages = blocks(blocks(max(a.num_pages, a.max_moves), 256, 4096), static_cast<int>(along), 4096);
        const size_t lds = sizeof(int) * ((a.num_pages + 31) / 32);
        hipLaunchKernelGGL(compact_bits_kernel, dim3(1), dim3(kThreads), lds, stream, a);
        hipLaunchKernelGGL(compact_bits_moves_kernel, dim3(blocks(a.num_pages, 256, 1024)), dim3(256), 0, stream, a);
        hipLaunchKernelGGL(compact_bits_apply_kernel, dim3(static_cast<unsigned>(a.B) + pages, along), dim3(256), 0, stream, a);
        return hipGetLastError();
    }
    // (as the workspace may hold anything)
    const hipError_t err = launch_fill_zero(a.state, compact_workspace(a), stream);
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(compact_mark_kernel, dim3(blocks(max(a.num_pages, a.max_moves), 256, 1024)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(compact_table_kernel, dim3(static_cast<unsigned>(a.B), along), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(compact_shares_kernel, dim3(blocks(a.num_pages, 256, 1024)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace kvq
