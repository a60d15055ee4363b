// kvq_select.hip -- page selection of sparse decode: which pages of each
// (sequence, kv head) a decode step attends.
//
// Score of a page with bounds (high, low, S), for the G query heads of the kv
// head: with integer codes c of the heads' q under one scale,
//   score = RN(RN(max_g sum_i max(c_gi high_i, c_gi low_i)) * S),
// an upper bound of the largest dot product of any of its keys (in units of the
// q scale).  The integer sum is exact and the two roundings are IEEE's, so the
// ranking does not depend on the order of summation.
//
// Ranking: scores become 32-bit keys that order as unsigned integers; the k-th
// largest key is found by narrowing a range of keys with histograms of 2048
// bins (two rounds separate thousands of scores), and one pass in page order
// writes the pages above it, and of those equal to it the first.
#include <limits.h>
#include <math.h>

#include "kvq_bounds.hpp"
#include "kvq_device.hpp"
#include "kvq_pages.hpp"

namespace kvq {
namespace {

constexpr int kSelWaves = 8;
constexpr int kSelThreads = kSelWaves * kWave;
constexpr int kSelBins = 2048;
constexpr int kSelLogBins = 11;

// Order of scores as unsigned integers; NaN above all, -0 as 0.
__device__ __forceinline__ unsigned rank_key(float score) {
    if (score != score) return 0xffffffffu;
    const unsigned u = __float_as_uint(score + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct RankScratch {
    unsigned hist[kSelBins];
    unsigned lo[kSelWaves], hi[kSelWaves];
    int sums[kSelWaves];
    int gt[kSelWaves], eq[kSelWaves];
    int bin, above, count;
};

// The keys above `key`, and the first `ties` of those equal to it.
struct Cut {
    unsigned key;
    int ties;
};

// Cut of the k largest of n keys (0 < k < n), by the whole workgroup; key(i) reads key i.
template <class Key>
__device__ inline Cut rank_cut(const Key& key, int n, int k, RankScratch& s) {
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int wave = t / kWave;
    unsigned lo = 0xffffffffu, hi = 0;
    for (int i = t; i < n; i += kSelThreads) {
        const unsigned x = key(i);
        lo = min(lo, x);
        hi = max(hi, x);
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        lo = min(lo, static_cast<unsigned>(__shfl_xor(static_cast<int>(lo), off)));
        hi = max(hi, static_cast<unsigned>(__shfl_xor(static_cast<int>(hi), off)));
    }
    if (lane == 0) {
        s.lo[wave] = lo;
        s.hi[wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWaves; w++) {
        lo = min(lo, s.lo[w]);
        hi = max(hi, s.hi[w]);
    }
    // The k largest keys of [lo, hi] are wanted; every round leaves a bin of the
    // last one's range, at most a 2048th of it, so three rounds end it.
    for (;;) {
        if (lo == hi) return Cut{lo, k};
        const int shift = max(0, 32 - __clz(static_cast<int>(hi - lo)) - kSelLogBins);
        __syncthreads();
        for (int i = t; i < kSelBins; i += kSelThreads) s.hist[i] = 0;
        __syncthreads();
        for (int i = t; i < n; i += kSelThreads) {
            const unsigned x = key(i);
            if (x >= lo && x <= hi) atomicAdd(&s.hist[(x - lo) >> shift], 1u);
        }
        __syncthreads();
        // Thread t sums bins from the top: [2047 - 4 t - 3, 2047 - 4 t].
        constexpr int kPer = kSelBins / kSelThreads;
        const int top = kSelBins - 1 - t * kPer;
        int sum = 0;
#pragma unroll
        for (int j = 0; j < kPer; j++) sum += static_cast<int>(s.hist[top - j]);
        const int incl_wave = wave_inclusive_scan(sum);
        if (lane == kWave - 1) s.sums[wave] = incl_wave;
        __syncthreads();
        int above = incl_wave - sum;
        for (int w = 0; w < wave; w++) above += s.sums[w];
        if (above < k && k <= above + sum) {
            int j = 0;
            while (j < kPer - 1 && above + static_cast<int>(s.hist[top - j]) < k) above += static_cast<int>(s.hist[top - j++]);
            s.bin = top - j;
            s.above = above;
            s.count = static_cast<int>(s.hist[top - j]);
        }
        __syncthreads();
        lo += static_cast<unsigned>(s.bin) << shift;
        k -= s.above;
        if (k == s.count) return Cut{lo, INT_MAX};  // the whole bin
        if (hi - lo > (1u << shift) - 1u) hi = lo + ((1u << shift) - 1u);
    }
}

// Writes the chosen of n keys in order: emit(place, i).
template <class Key, class Emit>
__device__ inline void rank_emit(const Key& key, int n, const Cut& cut, RankScratch& s, const Emit& emit) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    const int per = ((n + kSelWaves - 1) / kSelWaves + kWave - 1) / kWave * kWave;  // keys a wave
    const int i0 = min(wave * per, n), i1 = min(i0 + per, n);
    int gt = 0, eq = 0;
    for (int i = i0 + lane; i - lane < i1; i += kWave) {
        const unsigned x = i < i1 ? key(i) : 0;
        gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < i1 && x > cut.key));
        eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < i1 && x == cut.key));
    }
    if (lane == 0) {
        s.gt[wave] = gt;
        s.eq[wave] = eq;
    }
    __syncthreads();
    int above = 0, ties = 0;
    for (int w = 0; w < wave; w++) {
        above += s.gt[w];
        ties += s.eq[w];
    }
    int place = above + min(ties, cut.ties);
    const unsigned long long below = (1ull << lane) - 1ull;
    for (int i = i0 + lane; i - lane < i1; i += kWave) {
        const unsigned x = i < i1 ? key(i) : 0;
        const unsigned long long same = __builtin_amdgcn_ballot_w64(i < i1 && x == cut.key);
        const bool take = i < i1 && (x > cut.key || (x == cut.key && ties + __builtin_popcountll(same & below) < cut.ties));
        const unsigned long long taken = __builtin_amdgcn_ballot_w64(take);
        if (take) emit(place + __builtin_popcountll(taken & below), i);
        place += __builtin_popcountll(taken);
        ties += __builtin_popcountll(same);
    }
}

// One (sequence, kv head): its pages, and which of them are scored.
struct Unit {
    int b, h, len, pages;
    int scored;   // pages scored: [keep_first, keep_first + scored); 0: every page is attended
    int wanted;   // of those, how many are attended
    int renewed;  // page entry whose bounds this launch writes, or -1
};
__device__ __forceinline__ Unit unit_of(const SelectArgs& a, int unit) {
    Unit u;
    u.b = unit / a.b.Hkv;
    u.h = unit - u.b * a.b.Hkv;
    u.len = a.b.lengths ? min(max(a.b.lengths[u.b], 0), a.b.max_len) : a.b.max_len;
    const int size = a.b.pages.size;
    u.pages = u.len > 0 ? (u.len - 1) / size + 1 : 0;
    const bool rank = u.pages > a.max_selected;
    u.scored = rank ? u.pages - a.keep_first - a.keep_last : 0;
    u.wanted = rank ? a.max_selected - a.keep_first - a.keep_last : 0;
    u.renewed = u.len > 1 && (u.len - 1) % size == 0 ? u.pages - 2 : -1;
    return u;
}

__device__ __forceinline__ int pool_row(const SelectArgs& a, const Unit& u, int entry) {
    const int id = a.b.pages.table[static_cast<size_t>(u.b) * a.b.pages.max_pages + entry];
    return min(max(id, 0), a.b.pages.num_pages - 1) * a.b.Hkv + u.h;
}

// Everything but the scored pages, and the selection's length.
__device__ inline void write_kept(const SelectArgs& a, const Unit& u, int unit) {
    int32_t* out = a.selected + static_cast<size_t>(unit) * a.max_selected;
    const int size = a.b.pages.size;
    const int n = u.scored > 0 ? a.max_selected : u.pages;
    const int head = u.scored > 0 ? a.keep_first : u.pages;
    for (int i = threadIdx.x; i < a.max_selected; i += kSelThreads) {
        if (i < head) out[i] = pool_row(a, u, i);
        else if (i >= n) out[i] = -1;
        else if (i >= n - a.keep_last) out[i] = pool_row(a, u, u.pages - n + i);
    }
    if (threadIdx.x == 0) a.selected_lengths[unit] = u.len > 0 ? (n - 1) * size + (u.len - 1) % size + 1 : 0;
}

// Any head dim or alignment: a workgroup a unit, a wave a page, keys in global memory.
__global__ __launch_bounds__(kSelThreads) void select_generic(const SelectArgs a) {
    __shared__ RankScratch s;
    __shared__ float s_max[kSelWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    const int unit = blockIdx.x;
    const int d = a.b.d;
    const Unit u = unit_of(a, unit);
    if (u.renewed >= 0 && wave == 0) bounds_generic(a.b, u.b, u.renewed, u.h, a.b.pages.size, lane);
    write_kept(a, u, unit);
    if (u.wanted == 0) return;
    const float* q = a.q + static_cast<size_t>(unit) * a.G * d;
    float amax = 0.0f;
    for (int i = threadIdx.x; i < a.G * d; i += kSelThreads) amax = fmaxf(amax, fabsf(q[i]));
    amax = wave_max(amax);
    if (lane == 0) s_max[wave] = amax;
    __syncthreads();  // and the renewed bounds are written
#pragma unroll
    for (int w = 0; w < kSelWaves; w++) amax = fmaxf(amax, s_max[w]);
    const float qs = quant_scale(amax);
    unsigned* keys = a.keys + static_cast<size_t>(unit) * a.key_stride;
    for (int i = wave; i < u.scored; i += kSelWaves) {
        const size_t row = static_cast<size_t>(pool_row(a, u, a.keep_first + i));
        const int8_t* hi = a.b.bounds + row * 2 * d;
        const int8_t* lo = hi + d;
        int top = INT_MIN;
        for (int g = 0; g < a.G; g++) {
            int sum = 0;
            for (int j = lane; j < d; j += kWave) {
                const int c = quant_one(q[static_cast<size_t>(g) * d + j], qs);
                sum += max(c * hi[j], c * lo[j]);
            }
#pragma unroll
            for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
            top = max(top, sum);
        }
        if (lane == 0) keys[i] = rank_key(static_cast<float>(top) * a.b.scale[row]);
    }
    __syncthreads();
    auto key = [&](int i) { return keys[i]; };
    const Cut cut = rank_cut(key, u.scored, u.wanted, s);
    int32_t* out = a.selected + static_cast<size_t>(unit) * a.max_selected + a.keep_first;
    rank_emit(key, u.scored, cut, s, [&](int place, int i) { out[place] = pool_row(a, u, a.keep_first + i); });
}

}  // namespace

SelectPlan select_plan(int units, int max_pages, int max_selected) {
    SelectPlan p{1, 0, 0};
    if (max_pages <= max_selected) return p;
    p.key_stride = max_pages;
    p.key_bytes = static_cast<size_t>(units) * max_pages * sizeof(unsigned);
    return p;
}

hipError_t launch_select(const SelectArgs& a, bool, hipStream_t stream) {
    hipLaunchKernelGGL(select_generic, dim3(static_cast<unsigned>(a.b.B * a.b.Hkv)), dim3(kSelThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace kvq
