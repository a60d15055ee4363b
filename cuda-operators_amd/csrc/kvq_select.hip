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

#include <algorithm>

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

// The largest and smallest of a wave's unsigned values (the steps of
// wave_inclusive_scan; lanes shifted in from outside a row give 0).
__device__ __forceinline__ unsigned wave_max_u32(unsigned x) {
    int v = static_cast<int>(x);
#define KVQ_STEP(CTRL, ROWS) \
    v = static_cast<int>(max(static_cast<unsigned>(v), static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false))));
    KVQ_STEP(0x111, 0xF)
    KVQ_STEP(0x112, 0xF)
    KVQ_STEP(0x114, 0xF)
    KVQ_STEP(0x118, 0xF)
    KVQ_STEP(0x142, 0xA)
    KVQ_STEP(0x143, 0xC)
#undef KVQ_STEP
    return static_cast<unsigned>(__builtin_amdgcn_readlane(v, kWave - 1));
}
__device__ __forceinline__ unsigned wave_min_u32(unsigned x) { return ~wave_max_u32(~x); }

constexpr int kSelList = kWave;  // keys of one bin that a wave ranks by comparing each with each
struct RankScratch {
    unsigned hist[kSelBins];  // zero whenever rank_cut begins (clear_bins)
    unsigned list[kSelList];
    unsigned lo[kSelWaves], hi[kSelWaves];
    int sums[kSelWaves];
    int gt[kSelWaves], eq[kSelWaves];
    int bin, above, count, listed;
};
__device__ __forceinline__ void clear_bins(RankScratch& s) {
    for (int i = threadIdx.x; i < kSelBins; i += kSelThreads) s.hist[i] = 0;
    if (threadIdx.x == 0) s.listed = 0;
}

// Keys a thread has on their way while it ranks: a step over 2048 pages of 8
// units 21.1 us with one, 20.8 with 2, 20.3 with 4 and 20.9 with 8.
constexpr int kSelAhead = 4;

// The keys above `key`, and the first `ties` of those equal to it.
struct Cut {
    unsigned key;
    int ties;
};

// The workgroup's threads take each of n keys once, several loads of a thread in flight.
template <class Key, class Take>
__device__ __forceinline__ void each_key(const Key& key, int n, const Take& take) {
    for (int first = 0; first < n; first += kSelAhead * kSelThreads) {
        const int i = first + threadIdx.x;
        unsigned x[kSelAhead];
#pragma unroll
        for (int j = 0; j < kSelAhead; j++) x[j] = key(min(i + j * kSelThreads, n - 1));
#pragma unroll
        for (int j = 0; j < kSelAhead; j++) {
            if (first + j * kSelThreads >= n) break;  // for all of them
            if (i + j * kSelThreads < n) take(x[j]);
        }
    }
}

// Cut of the k largest of n keys (0 < k < n), by the whole workgroup; key(i)
// reads key i, lo and hi are the smallest and largest that this thread has seen,
// all threads together having seen all.
template <class Key>
__device__ inline Cut rank_cut(const Key& key, int n, int k, unsigned lo, unsigned hi, RankScratch& s) {
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int wave = t / kWave;
    lo = wave_min_u32(lo);
    hi = wave_max_u32(hi);
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
    // last one's range, at most a 2048th of it, so three rounds end it.  As a
    // rule the first leaves a few keys, which every wave ranks for itself.
    for (;;) {
        if (lo == hi) return Cut{lo, k};
        const int shift = max(0, 32 - __clz(static_cast<int>(hi - lo)) - kSelLogBins);
        each_key(key, n, [&](unsigned x) {
            if (x >= lo && x <= hi) atomicAdd(&s.hist[(x - lo) >> shift], 1u);
        });
        __syncthreads();
        // Thread t sums bins from the top: [2047 - 4 t - 3, 2047 - 4 t].
        constexpr int kPer = kSelBins / kSelThreads;
        const int top = kSelBins - 1 - t * kPer;
        int bins[kPer], sum = 0;
#pragma unroll
        for (int j = 0; j < kPer; j++) sum += bins[j] = static_cast<int>(s.hist[top - j]);
        const int incl_wave = wave_inclusive_scan(sum);
        if (lane == kWave - 1) s.sums[wave] = incl_wave;
        __syncthreads();
        int above = incl_wave - sum;
#pragma unroll
        for (int w = 0; w < kSelWaves; w++) above += w < wave ? s.sums[w] : 0;
        if (above < k && k <= above + sum) {
            bool found = false;
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                if (!found && k <= above + bins[j]) {
                    found = true;
                    s.bin = top - j;
                    s.above = above;
                    s.count = bins[j];
                }
                above += bins[j];
            }
        }
        __syncthreads();
        lo += static_cast<unsigned>(s.bin) << shift;
        k -= s.above;
        const int count = s.count;
        if (k == count) return Cut{lo, INT_MAX};  // the whole bin
        if (hi - lo > (1u << shift) - 1u) hi = lo + ((1u << shift) - 1u);
        if (count <= kSelList) {
            each_key(key, n, [&](unsigned x) {
                if (x >= lo && x <= hi) s.list[atomicAdd(&s.listed, 1)] = x;
            });
            __syncthreads();
            const unsigned mine = lane < count ? s.list[lane] : 0;
            int more = 0, same = 0;  // keys above this lane's, and equal ones
            for (int j = 0; j < count; j++) {
                const unsigned x = static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), j));
                more += x > mine;
                same += x == mine;
            }
            const unsigned long long at = __builtin_amdgcn_ballot_w64(lane < count && more < k && k <= more + same);
            const int l = __builtin_ctzll(at);  // a lane with the k-th key: there is one
            return Cut{static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), l)),
                       k - __builtin_amdgcn_readlane(more, l)};
        }
        for (int i = t; i < kSelBins; i += kSelThreads) s.hist[i] = 0;
        __syncthreads();
    }
}

// Writes the chosen of n keys in order: emit(place, i).
template <class Key, class Emit>
__device__ inline void rank_emit(const Key& key, int n, const Cut& cut, RankScratch& s, const Emit& emit) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int per = ((n + kSelWaves - 1) / kSelWaves + kWave - 1) / kWave * kWave;  // keys a wave
    const int i0 = min(wave * per, n), i1 = min(i0 + per, n);
    int gt = 0, eq = 0;
    unsigned x[kSelAhead];
    auto read = [&](int first) {
#pragma unroll
        for (int j = 0; j < kSelAhead; j++) x[j] = key(min(first + j * kWave + lane, n - 1));
    };
    for (int first = i0; first < i1; first += kSelAhead * kWave) {
        read(first);
#pragma unroll
        for (int j = 0; j < kSelAhead; j++) {
            if (first + j * kWave >= i1) break;
            const bool live = first + j * kWave + lane < i1;
            gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(live && x[j] > cut.key));
            eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(live && x[j] == cut.key));
        }
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
    for (int first = i0; first < i1; first += kSelAhead * kWave) {
        if (i1 - i0 > kSelAhead * kWave) read(first);  // else x still holds them
#pragma unroll
        for (int j = 0; j < kSelAhead; j++) {
            if (first + j * kWave >= i1) break;
            const int i = first + j * kWave + lane;
            const unsigned long long same = __builtin_amdgcn_ballot_w64(i < i1 && x[j] == cut.key);
            const bool take = i < i1 && (x[j] > cut.key || (x[j] == cut.key && ties + __builtin_popcountll(same & below) < cut.ties));
            const unsigned long long taken = __builtin_amdgcn_ballot_w64(take);
            if (take) emit(place + __builtin_popcountll(taken & below), i);
            place += __builtin_popcountll(taken);
            ties += __builtin_popcountll(same);
        }
    }
}

// One (sequence, kv head): its pages, and which of them are scored.
struct Unit {
    int b, h, len, pages;
    int scored;   // pages scored: [keep_first, keep_first + scored); 0: every page is attended
    int wanted;   // of those, how many are attended
    int renewed;  // page entry whose bounds this launch writes, or -1
};
__device__ __forceinline__ int page_entry(const SelectArgs& a, int token) {
    return a.b.pages.shift >= 0 ? token >> a.b.pages.shift : token / a.b.pages.size;
}
__device__ __forceinline__ Unit unit_of(const SelectArgs& a, int unit) {
    Unit u;
    u.b = unit / a.b.Hkv;
    u.h = unit - u.b * a.b.Hkv;
    u.len = a.b.lengths ? min(max(a.b.lengths[u.b], 0), a.b.max_len) : a.b.max_len;
    const int size = a.b.pages.size;
    u.pages = u.len > 0 ? page_entry(a, u.len - 1) + 1 : 0;
    const bool rank = u.pages > a.max_selected;
    u.scored = rank ? u.pages - a.keep_first - a.keep_last : 0;
    u.wanted = rank ? a.max_selected - a.keep_first - a.keep_last : 0;
    u.renewed = u.len > 1 && (u.pages - 1) * size == u.len - 1 ? u.pages - 2 : -1;
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
    if (threadIdx.x == 0) a.selected_lengths[unit] = u.len > 0 ? (n - u.pages) * size + u.len : 0;
}

// Tuned head dims (multiples of 16 up to 256): scores on matrix cores.
//
// max(c high, c low) = max(c, 0) high + min(c, 0) low, so with a page's highs
// and lows as one row of 2 d bytes, which is how they lie in memory, and each
// head's max(c, 0) and min(c, 0) as one column of 2 d bytes, sixteen pages times
// sixteen heads are ND = 2 d / 64 int8 matrix products.  The rows come straight
// from memory into the A operand (16 bytes a lane, four lanes a 64-byte piece),
// the columns from LDS; columns past the last head are left out of the maximum,
// and bytes past 2 d are zero in the columns.  Reading the bounds is all that costs: 16 pages
// a wave at a time, the next 16 on their way, their ids one step further ahead.
//
// A unit's pages go to `splits` workgroups in whole steps of 128; the last one
// to arrive ranks.  One workgroup keeps its keys in LDS; several pass them
// through memory coherently (as split records do, kvq_split.hpp).
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int kSelTile = 16;                      // pages a wave scores at a time
constexpr int kSelStep = kSelTile * kSelWaves;    // pages a workgroup does
constexpr int kSelLdsKeys = 6144;                 // ranks kept in LDS, at most

template <int CTRL>
__device__ __forceinline__ int dpp_max(int x) {
    return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false));
}
// Signed maximum over each 16 lanes.
__device__ __forceinline__ int row16_max(int x) {
    x = dpp_max<kDppQuadXor1>(x);
    x = dpp_max<kDppQuadXor2>(x);
    x = dpp_max<kDppRowHalfMirror>(x);
    return dpp_max<kDppRowMirror>(x);
}

template <int ND>
__global__ __launch_bounds__(kSelThreads) __attribute__((amdgpu_waves_per_eu(4))) void select_kernel(const SelectArgs a, int lds_keys) {
    extern __shared__ __align__(16) unsigned char s_dyn[];  // columns [passes][ND][64] x 16 bytes, lds_keys ranks, their pool rows
    __shared__ RankScratch s;
    __shared__ float s_max[kSelWaves];
    __shared__ int s_last;
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int units = a.b.B * a.b.Hkv;
    const int split = blockIdx.x / units;
    const int unit = blockIdx.x - split * units;
    const int d = a.b.d;
    const int passes = (a.G + 15) / 16;
    unsigned* s_keys = reinterpret_cast<unsigned*>(s_dyn + static_cast<size_t>(passes) * ND * 1024);
    int* s_rows = reinterpret_cast<int*>(s_keys + lds_keys);
    // q is on its way while the length and the page ids are waited for.
    const float4* q = reinterpret_cast<const float4*>(a.q + static_cast<size_t>(unit) * a.G * d);
    const int quads = a.G * d / 4;
    const float4 mine = q[min(t, quads - 1)];
    const Unit u = unit_of(a, unit);

    // This workgroup's pages, and how many workgroups have any.
    const int n = u.wanted > 0 ? u.scored : 0;
    const int steps = (n + kSelStep - 1) / kSelStep;
    const int chunk = (steps + a.splits - 1) / a.splits * kSelStep;
    const int active = n > 0 ? (n + chunk - 1) / chunk : 1;
    if (split >= active) return;
    const int i0 = split * chunk, i1 = min(n, i0 + chunk);

    // The page that has just become whole belongs to the last workgroup, which
    // ranks it if it is ranked.
    if (u.renewed >= 0 && split == active - 1 && wave == 0) {
        constexpr int LPT = bounds_lanes(32 * ND);
        const BoundsWave<LPT, Pages::Passes> w(a.b, kWave / LPT);
        typename BoundsWave<LPT, Pages::Passes>::Piece piece;
        w.fetch(piece, a.b.pages.table[static_cast<size_t>(u.b) * a.b.pages.max_pages + u.renewed], u.h, a.b.pages.size);
        w.finish(piece, true);
    }
    if (n == 0) {
        write_kept(a, u, unit);
        return;
    }

    const int r = lane & 15, c16 = (lane >> 4) * 16;
    auto row_of = [&](int i) { return static_cast<size_t>(pool_row(a, u, a.keep_first + min(i, i1 - 1))); };
    auto load = [&](size_t row, i32x4 (&x)[ND], float& scale) {
        const int8_t* p = a.b.bounds + row * 2 * d;
#pragma unroll
        for (int j = 0; j < ND; j++) x[j] = *reinterpret_cast<const i32x4*>(p + min(j * 64 + c16, 2 * d - 16));
        scale = a.b.scale[row];
    };
    i32x4 next[ND];
    float next_scale = 0.0f;
    int base = i0 + wave * kSelTile;
    const size_t row0 = row_of(base + r);
    size_t next_row = row0;  // of the pages in `next`
    size_t row = row_of(base + kSelStep + r);

    // The heads' codes: four of one head a thread, once into the highs' half of
    // its column (those above zero) and once into the lows' half (those below).
    auto largest = [](const float4& x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); };
    float amax = largest(mine);
    for (int i = t + kSelThreads; i < quads; i += kSelThreads) amax = fmaxf(amax, largest(q[i]));
    amax = __uint_as_float(wave_max_u32(__float_as_uint(amax)));  // not negative, so ordered as its bits; never NaN
    if (lane == 0) s_max[wave] = amax;
    clear_bins(s);
    int* columns = reinterpret_cast<int*>(s_dyn);
    auto word = [&](int g, int off) {  // of byte `off` of head g's column
        return (((g >> 4) * ND + (off >> 6)) * 64 + ((off >> 4) & 3) * 16 + (g & 15)) * 4 + ((off >> 2) & 3);
    };
    if (2 * d < ND * 64)  // what a column has behind its end
        for (int i = t; i < a.G * (ND * 64 - 2 * d) / 4; i += kSelThreads) {
            const int per = (ND * 64 - 2 * d) / 4;
            columns[word(i / per, 2 * d + (i % per) * 4)] = 0;
        }
    __syncthreads();  // and the renewed bounds are written
    // The first pages' ids were on their way until here, their bounds are while
    // the codes are made (fetched before the barrier: 21.7 us a step for 21.1).
    load(row0, next, next_scale);
#pragma unroll
    for (int w = 0; w < kSelWaves; w++) amax = fmaxf(amax, s_max[w]);
    const float qs = quant_scale(amax);
    for (int i = t; i < quads; i += kSelThreads) {
        const float4 x = i == t ? mine : q[i];
        const float y[4] = {x.x, x.y, x.z, x.w};
        int c[4];
        quant_row<4>(y, qs, c);
        const int g = 4 * i / d, off = 4 * i - g * d;
        columns[word(g, off)] = pack4(max(c[0], 0), max(c[1], 0), max(c[2], 0), max(c[3], 0));
        columns[word(g, d + off)] = pack4(min(c[0], 0), min(c[1], 0), min(c[2], 0), min(c[3], 0));
    }
    __syncthreads();
    if (split == 0) write_kept(a, u, unit);

    const bool shared = active > 1 || n > lds_keys;  // keys in memory
    unsigned* keys = shared ? a.keys + static_cast<size_t>(unit) * a.key_stride : nullptr;
    unsigned lo = 0xffffffffu, hi = 0;  // of the keys this thread has seen
    for (; base < i1; base += kSelStep) {
        i32x4 x[ND];
#pragma unroll
        for (int j = 0; j < ND; j++) x[j] = next[j];
        const float scale = next_scale;
        const size_t now = next_row;
        load(row, next, next_scale);
        next_row = row;
        row = row_of(base + 2 * kSelStep + r);
        i32x4 top = {INT_MIN, INT_MIN, INT_MIN, INT_MIN};
        for (int pass = 0; pass < passes; pass++) {
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < ND; j++) {
                const i32x4 y = reinterpret_cast<const i32x4*>(s_dyn)[(pass * ND + j) * 64 + lane];
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[j], y, acc, 0, 0, 0);
            }
            if (pass * 16 + r < a.G) {  // columns past the last head hold anything
#pragma unroll
                for (int i = 0; i < 4; i++) top[i] = max(top[i], acc[i]);
            }
        }
        // Lane 16 g + c holds pages 4 g .. 4 g + 3 of head c; lanes c < 4 write page 4 g + c.
#pragma unroll
        for (int i = 0; i < 4; i++) top[i] = row16_max(top[i]);
        const int best = (r & 2) ? ((r & 1) ? top[3] : top[2]) : ((r & 1) ? top[1] : top[0]);
        const int page = 4 * (lane >> 4) + (r & 3);
        const float sc = __shfl(scale, page);
        if (!shared && lane < kSelTile && base + r < i1) s_rows[base + r] = static_cast<int>(now);
        const int i = base + page;
        if (r < 4 && i < i1) {
            const unsigned key = rank_key(static_cast<float>(best) * sc);
            lo = min(lo, key);
            hi = max(hi, key);
            if (shared) __hip_atomic_store(keys + i, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            else s_keys[i] = key;
        }
    }
    if (active > 1) {
        __builtin_amdgcn_s_waitcnt(0);  // this thread's keys have arrived
        __syncthreads();
        if (t == 0) {
            s_last = __hip_atomic_fetch_add(a.counters + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == active - 1;
            if (s_last) __hip_atomic_store(a.counters + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!s_last) return;
    }
    if (shared && n <= lds_keys) {
        for (int i = t; i < n; i += kSelAhead * kSelThreads) {
            int place[kSelAhead];
            unsigned key[kSelAhead];
#pragma unroll
            for (int j = 0; j < kSelAhead; j++) {
                const int x = min(i + j * kSelThreads, n - 1);
                key[j] = __hip_atomic_load(keys + x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                place[j] = pool_row(a, u, a.keep_first + x);
            }
#pragma unroll
            for (int j = 0; j < kSelAhead; j++) {
                if (i + j * kSelThreads >= n) break;
                s_keys[i + j * kSelThreads] = key[j];
                s_rows[i + j * kSelThreads] = place[j];
                lo = min(lo, key[j]);
                hi = max(hi, key[j]);
            }
        }
    } else if (shared) {
        __builtin_amdgcn_s_waitcnt(0);
        lo = 0, hi = 0xffffffffu;
    }
    __syncthreads();
    int32_t* out = a.selected + static_cast<size_t>(unit) * a.max_selected + a.keep_first;
    auto finish = [&](const auto& key, const auto& place_of) {
        const Cut cut = rank_cut(key, n, u.wanted, lo, hi, s);
        rank_emit(key, n, cut, s, [&](int place, int i) { out[place] = place_of(i); });
    };
    if (n <= lds_keys) finish([&](int i) { return s_keys[i]; }, [&](int i) { return s_rows[i]; });
    else finish([&](int i) { return __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); },
                [&](int i) { return pool_row(a, u, a.keep_first + i); });
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
    clear_bins(s);
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
    const Cut cut = rank_cut(key, u.scored, u.wanted, 0u, 0xffffffffu, s);
    int32_t* out = a.selected + static_cast<size_t>(unit) * a.max_selected + a.keep_first;
    rank_emit(key, u.scored, cut, s, [&](int place, int i) { out[place] = pool_row(a, u, a.keep_first + i); });
}

}  // namespace

// A workgroup's columns fit LDS beside the ranks: up to 32 KB of them.
static bool select_tuned(int G, int d) {
    return d <= 256 && d % 16 == 0 && (G + 15) / 16 * ((2 * d + 63) / 64) <= 32;
}

SelectPlan select_plan(int units, int G, int d, bool vec_ok, int max_pages, int max_selected) {
    SelectPlan p{1, 0, 0, 0};
    if (max_pages <= max_selected) return p;
    if (vec_ok && select_tuned(G, d)) {
        // About two workgroups a CU, each with at least one step of pages; units
        // that fill the CUs alone are not split (whole steps: 2048 pages of 8
        // units 20.4 us in 16 parts, 22.8 in 4, 26.8 in 2; 1024 pages of 128 units
        // 42.6 us in 4 parts, 42.5 in 2, 44.1 in one; of 256 units 45.3 in 2, 43.5
        // in one).
        const long steps = (static_cast<long>(max_pages) + kSelStep - 1) / kSelStep;
        if (units < 256) p.splits = static_cast<int>(std::min(steps, 512L / units));
        p.lds_keys = max_pages <= kSelLdsKeys ? max_pages : 0;
        if (p.splits == 1 && p.lds_keys > 0) return p;
    }
    p.key_stride = max_pages;
    p.key_bytes = static_cast<size_t>(units) * max_pages * sizeof(unsigned);
    return p;
}

hipError_t launch_select(const SelectArgs& a, const SelectPlan& p, bool vec_ok, hipStream_t stream) {
    const unsigned units = static_cast<unsigned>(a.b.B * a.b.Hkv);
    const dim3 block(kSelThreads);
    if (!vec_ok || !select_tuned(a.G, a.b.d)) {
        hipLaunchKernelGGL(select_generic, dim3(units), block, 0, stream, a);
        return hipGetLastError();
    }
    const int nd = (2 * a.b.d + 63) / 64;
    const dim3 grid(units * static_cast<unsigned>(p.splits));
    const size_t lds = static_cast<size_t>((a.G + 15) / 16) * nd * 1024 + static_cast<size_t>(p.lds_keys) * 2 * sizeof(unsigned);
#define KVQ_SELECT_CASE(ND) \
    case ND: hipLaunchKernelGGL(select_kernel<ND>, grid, block, lds, stream, a, p.lds_keys); break;
    switch (nd) {
        KVQ_SELECT_CASE(1)
        KVQ_SELECT_CASE(2)
        KVQ_SELECT_CASE(3)
        KVQ_SELECT_CASE(4)
        KVQ_SELECT_CASE(5)
        KVQ_SELECT_CASE(6)
        KVQ_SELECT_CASE(7)
        KVQ_SELECT_CASE(8)
    }
#undef KVQ_SELECT_CASE
    return hipGetLastError();
}

}  // namespace kvq
