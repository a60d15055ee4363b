// kvq_pages.hip -- gfx950 kernels around a paged cache: page maps, packed cache
// writes and reads, key bounds of pages.
#include <limits.h>
#include <math.h>

#include "kvq_bounds.hpp"
#include "kvq_device.hpp"
#include "kvq_pages.hpp"

namespace kvq {
namespace {

// ---------------------------------------------------------------------------
// Page map: block tables, free pages and slots from request lengths.
// ---------------------------------------------------------------------------
// With old_b and new_b a sequence's lengths and P(x) = ceil(x / page size), it
// needs max(P(new) - P(old), 0) pages or gives up max(P(old) - P(new), 0).  Two
// prefix sums over the batch say everything else: that of the packed rows which
// row is whose, those of the pages which place of the stack
//   S = free_pages[0, F) ++ pages given up, in order (R of them)
// is whose: growing sequences take S[F + R - 1], S[F + R - 2], .. in order, so
// where the prefix sum is beyond F + R the request is refused (sums only grow,
// so the granted ones' sum is their own prefix).  The A pages taken leave
// S[0, F + R - A); of these the places from F on are written back.  Places read
// to hand out, [F + R - A, F) and pages given up, are never written, so the
// workgroups need no order among them; only lengths and the free count, which
// may be updated in place, are written by the last workgroup to arrive.
// Bound by latency: every workgroup loads the lengths and scans them (so a call
// is one launch), then takes its share of the rows and pages, each a search in
// LDS, a dependent load of a page id and a store.
constexpr int kMapThreads = 1024;
constexpr int kMapWaves = kMapThreads / kWave;

__device__ __forceinline__ int pages_of(int tokens, const FastDiv& page) {
    return static_cast<int>(fastdiv(static_cast<uint32_t>(tokens) + page.d - 1, page));
}

// For each x the last i in [0, n) with v[i] <= x, for ascending v with v[0] <= x;
// the K searches' loads go out together.
template <int K>
__device__ __forceinline__ void last_not_above(const int* v, int n, const int (&x)[K], int (&at)[K]) {
#pragma unroll
    for (int k = 0; k < K; k++) at[k] = 0;
    for (int step = 1 << (31 - __clz(n)); step > 0; step >>= 1) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int i = at[k] + step;
            if (i < n && v[min(i, n - 1)] <= x[k]) at[k] = i;
        }
    }
}
__device__ __forceinline__ int last_not_above(const int* v, int n, int x) {
    const int xs[1] = {x};
    int at[1];
    last_not_above<1>(v, n, xs, at);
    return at[0];
}

// Inclusive scans of K values a thread over the workgroup, and their totals;
// part: this scan's own scratch.
template <int K>
__device__ __forceinline__ void group_inclusive_scan(int (&v)[K], int (&total)[K], int (&part)[K][kMapWaves]) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
#pragma unroll
    for (int k = 0; k < K; k++) {
        v[k] = wave_inclusive_scan(v[k]);
        if (lane == kWave - 1) part[k][wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int x = wave_inclusive_scan(lane < kMapWaves ? part[k][lane] : 0);
        total[k] = __builtin_amdgcn_readlane(x, kMapWaves - 1);
        const int w = __builtin_amdgcn_readfirstlane(wave);
        if (w > 0) v[k] += __builtin_amdgcn_readlane(x, w - 1);
    }
}

// PER sequences a thread: thread t has sequences [t * PER, (t + 1) * PER).
template <int PER>
__global__ __launch_bounds__(kMapThreads) void page_map_kernel(const PageMapArgs a) {
    // Exclusive prefix sums of rows (saturated at a.T), pages needed and pages
    // given up, each with its total behind it; and the lengths, bit 31 set where
    // a request is refused.
    extern __shared__ int s_map[];
    __shared__ int s_rows[2][kMapWaves], s_pages[2][kMapWaves], s_taken[kMapWaves];
    __shared__ int s_last;
    const int B = a.B;
    int* s_off = s_map;
    int* s_need = s_off + B + 1;
    int* s_gives = s_need + B + 1;
    int* s_old = s_gives + B + 1;
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int b0 = t * PER;

    int n[PER], old[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int b = b0 + k;
        n[k] = b < B ? a.new_tokens[b] : 0;
        old[k] = b < B ? min(max(a.lengths[b], 0), a.cap) : 0;
    }
    const int F = min(max(*a.free_count, 0), a.num_pages);

    // Rows: sums of up to 4096 requests below 2^31, as sums of their halves.
    int half[2] = {0, 0}, sum[2];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        half[0] += max(n[k], 0) & 0xffff;
        half[1] += max(n[k], 0) >> 16;
    }
    int scan[2] = {half[0], half[1]};
    group_inclusive_scan(scan, sum, s_rows);
    long long at = static_cast<long long>(scan[0] - half[0]) + (static_cast<long long>(scan[1] - half[1]) << 16);
    const long long all = static_cast<long long>(sum[0]) + (static_cast<long long>(sum[1]) << 16);

    // Pages.  Totals stay below 2^31: B * max_pages does.
    int want[PER], p0[PER], moves[PER];  // moves: pages needed, or those given up as a negative number
    int pages[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int b = b0 + k;
        if (b < B) s_off[b] = static_cast<int>(min(at, static_cast<long long>(a.T)));
        at += max(n[k], 0);
        want[k] = n[k] < 0 ? max(old[k] + n[k], 0) : n[k] <= a.cap - old[k] && at <= a.T ? old[k] + n[k] : old[k];
        p0[k] = pages_of(old[k], a.page);
        moves[k] = pages_of(want[k], a.page) - p0[k];
        pages[0] += max(moves[k], 0);
        pages[1] += max(-moves[k], 0);
    }
    int pscan[2] = {pages[0], pages[1]}, ptotal[2];
    group_inclusive_scan(pscan, ptotal, s_pages);
    const int R = ptotal[1];
    const long long have = static_cast<long long>(F) + R;
    int need = pscan[0] - pages[0], gives = pscan[1] - pages[1], taken = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int b = b0 + k;
        const int incl = need + max(moves[k], 0);
        const bool enough = incl <= have;
        const bool refused = n[k] > 0 && (want[k] == old[k] || (moves[k] > 0 && !enough));
        if (b < B) {
            s_need[b] = need;
            s_gives[b] = gives;
            s_old[b] = old[k] | (refused ? INT_MIN : 0);
        }
        if (refused) want[k] = old[k];
        if (enough) taken = max(taken, incl);
        need = incl;
        gives += max(-moves[k], 0);
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) taken = max(taken, __shfl_xor(taken, off));
    if (lane == 0) s_taken[t / kWave] = taken;
    if (t == 0) {
        s_off[B] = static_cast<int>(min(all, static_cast<long long>(a.T)));
        s_need[B] = ptotal[0];
        s_gives[B] = R;
    }
    __syncthreads();
    int A = 0;  // pages taken
#pragma unroll
    for (int w = 0; w < kMapWaves; w++) A = max(A, s_taken[w]);
    const long long left = have - A;  // entries of the stack afterwards

    auto given_up = [&](int g, int c) {  // the g-th page given up, by sequence c
        const int end = pages_of(s_old[c], a.page);  // a shrinking sequence is not refused
        return a.table[static_cast<size_t>(c) * a.max_pages + end - (s_gives[c + 1] - s_gives[c]) + (g - s_gives[c])];
    };
    auto stack_at = [&](long long i) {
        if (i < F) return a.free_pages[i];
        const int g = static_cast<int>(i - F);
        return given_up(g, last_not_above(s_gives, B, g));
    };

    // Each job begins at another third of the threads, so that small ones run at
    // the same time in different waves instead of one load after the other.
    const int step = gridDim.x * kMapThreads;
    const int me = blockIdx.x * kMapThreads + t;
    const int third = step / 3 / kWave * kWave;
    for (long long i = me; i < A; i += step) {
        const int page = static_cast<int>(i);
        const int b = last_not_above(s_need, B, page);
        a.table[static_cast<size_t>(b) * a.max_pages + pages_of(s_old[b], a.page) + (page - s_need[b])] = stack_at(have - 1 - i);
    }
    const long long back = min(left, static_cast<long long>(a.num_pages)) - F;  // pages given up that stay on the stack
    constexpr int kBack = 4;  // loads in flight
    for (long long i = me < third ? me - third + step : me - third; i < back; i += static_cast<long long>(kBack) * step) {
        int g[kBack], c[kBack], id[kBack];
#pragma unroll
        for (int k = 0; k < kBack; k++) g[k] = static_cast<int>(min(i + static_cast<long long>(k) * step, back - 1));
        last_not_above<kBack>(s_gives, B, g, c);
#pragma unroll
        for (int k = 0; k < kBack; k++) id[k] = given_up(g[k], c[k]);
#pragma unroll
        for (int k = 0; k < kBack; k++)
            if (i + static_cast<long long>(k) * step < back) a.free_pages[F + i + static_cast<long long>(k) * step] = id[k];
    }

    // Packed rows.  A new page's id is taken from the stack again rather than
    // from the table, which another wave may not have written yet.
    if (a.slot_map || a.token_seq || a.token_pos) {
        for (long long i = me < 2 * third ? me - 2 * third + step : me - 2 * third; i < a.T; i += step) {
            int slot = -1, seq = -1, pos = -1;
            const int row = static_cast<int>(i);
            if (row < s_off[B]) {
                seq = last_not_above(s_off, B, row);
                const int held = s_old[seq];
                const unsigned at_pos = static_cast<unsigned>(held & INT_MAX) + static_cast<unsigned>(row - s_off[seq]);
                pos = static_cast<int>(min(at_pos, static_cast<unsigned>(INT_MAX)));
                if (held >= 0) {
                    const int pi = static_cast<int>(fastdiv(static_cast<uint32_t>(pos), a.page));
                    const int first = pages_of(held, a.page);
                    const int id = pi < first ? a.table[static_cast<size_t>(seq) * a.max_pages + pi]
                                              : stack_at(have - 1 - (s_need[seq] + pi - first));
                    const int size = static_cast<int>(a.page.d);
                    if (id >= 0 && id < a.num_pages) slot = id * size + (pos - pi * size);
                }
            }
            if (a.slot_map) a.slot_map[i] = slot;
            if (a.token_seq) a.token_seq[i] = seq;
            if (a.token_pos) a.token_pos[i] = pos;
        }
    }

    // The last workgroup writes what the others read.
    if (a.arrivals) {
        __syncthreads();
        if (t == 0) {
            s_last = __hip_atomic_fetch_add(a.arrivals, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                     static_cast<int>(gridDim.x) - 1;
            if (s_last) __hip_atomic_store(a.arrivals, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!s_last) return;
    }
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int b = b0 + k;
        if (b >= B) break;
        a.new_lengths[b] = want[k];
        a.granted[b] = want[k] - old[k];
        a.offsets[b] = s_off[b];
    }
    if (t == 0) {
        a.offsets[B] = s_off[B];
        *a.new_free_count = static_cast<int>(min(left, static_cast<long long>(a.num_pages)));
    }
}

// ---------------------------------------------------------------------------
// Packed rows into and out of their slots.
// ---------------------------------------------------------------------------
constexpr int kSlotWaves = 4;
// Workgroups along a grid's x: a dimension of 2^32 threads or more is not
// launched, which short rows reach (fp32 of up to 32 elements, four threads a
// row, at 2^30 rows).  Further workgroups lie along y.
constexpr unsigned kSlotGroups = 1u << 20;

// Pool row of token t's row for kv head h; -1: the slot lies outside the pool.
__device__ __forceinline__ long long slot_row(const SlotArgs& a, int t, int h) {
    const int s = a.slots[t];
    if (s < 0 || s >= a.slots_in_pool) return -1;
    const int page = static_cast<int>(fastdiv(static_cast<uint32_t>(s), a.page));
    const int size = static_cast<int>(a.page.d);
    return (static_cast<long long>(page) * a.Hkv + h) * size + (s - page * size);
}

template <bool BF16>
__device__ __forceinline__ float row_elem(const void* x, int64_t i) {
    if constexpr (BF16) return __uint_as_float(static_cast<unsigned>(static_cast<const uint16_t*>(x)[i]) << 16);
    else return static_cast<const float*>(x)[i];
}

// Tuned rows: LPR lanes a row with 16 bytes of it each (fp32: 4 elements, bf16:
// 8), U loads in flight a lane.  A wave takes U * RPW consecutive tokens of one
// kv head: in the pool these are as a rule consecutive rows of a page, so its
// codes and scales go out (or come in) in whole cache lines, while neighbouring
// waves take the other heads of the same tokens, whose packed rows lie beside.
// The packed side streams past the caches.  Bound by the mixed stream of reads
// and writes (a large copy moves 4.8 TB/s): writes of 24,560 tokens, 8 heads, d =
// 128 and bf16 34 us out of a fused projection (4.5 TB/s; U = 1 35 us, 4 39 us, 8
// 42 us; without streaming loads 46 us at U = 4), 30 us packed, fp32 47 us packed
// (5.3 TB/s); reads of 98,304 tokens as bf16 113 us (5.4 TB/s; U = 2 134 us, 4
// 120 us; without streaming stores 2 us more).  A small read is bound by its
// chain of loads, and shorter waves are done sooner: 4099 tokens as fp32 7.4 us
// at U = 2, 8.4 at 8.
// PAD: a row of d < D elements, whole 16-byte pieces; the lanes past its last
// piece read that piece again and store nothing.
template <int D, bool BF16, int LOADS>
struct SlotGeom {
    static constexpr int EPL = BF16 ? 8 : 4;  // elements a lane
    static constexpr int LPR = D / EPL;       // lanes a row
    static constexpr int RPW = kWave / LPR;   // rows a wave load
    static constexpr int U = LOADS;
    static constexpr int TB = RPW * U;        // tokens a wave
    static_assert(LPR >= 1 && LPR <= kWave && kWave % LPR == 0, "row geometry");
};

// The wave's unit (token block, head) and plane (blockIdx.y's last bit: K or V):
// false past the last unit.  Units number at most T * Hkv, below 2^31.
__device__ __forceinline__ bool slot_unit(const SlotArgs& a, int tb, int& t0, int& h) {
    const unsigned group = (blockIdx.y >> 1) * kSlotGroups + blockIdx.x;
    const unsigned unit = group * kSlotWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned blk = fastdiv(unit, a.heads);
    h = static_cast<int>(unit - blk * a.Hkv);
    const long long first = static_cast<long long>(blk) * tb;
    t0 = static_cast<int>(first);
    return first < a.T;
}

constexpr int kWriteLoads = 2, kReadLoads = 8, kSmallReadLoads = 2;

template <int D, bool BF16, bool PAD>
__global__ __launch_bounds__(kSlotWaves* kWave) void slot_write_kernel(const SlotArgs a) {
    using Geo = SlotGeom<D, BF16, kWriteLoads>;
    constexpr int EPL = Geo::EPL, LPR = Geo::LPR, RPW = Geo::RPW, U = Geo::U;
    int t0, h;
    if (!slot_unit(a, Geo::TB, t0, h)) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int d = PAD ? a.d : D;
    const int ls = PAD ? min(lane % LPR, d / EPL - 1) : lane % LPR;  // 16-byte piece of the row
    const bool owner = !PAD || ls == lane % LPR;
    const int kv = blockIdx.y & 1;
    const int64_t stride = kv ? a.v_stride : a.k_stride;
    const char* x = static_cast<const char*>(kv ? a.v_rows : a.k_rows) +
                    (static_cast<int64_t>(h) * a.head_stride + ls * EPL) * (BF16 ? 2 : 4);
    int8_t* qo = kv ? a.v : a.k;
    float* so = kv ? a.vs : a.ks;
    int4 raw[U];
    long long orow[U];
#pragma unroll
    for (int u = 0; u < U; u++) {  // a token past the end reads the last one again and is dropped
        const int tc = min(t0 + u * RPW + lane / LPR, a.T - 1);
        const v4i_t w = __builtin_nontemporal_load(reinterpret_cast<const v4i_t*>(x + tc * stride * (BF16 ? 2 : 4)));
        raw[u] = make_int4(w.x, w.y, w.z, w.w);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int t = t0 + u * RPW + lane / LPR;
        orow[u] = slot_row(a, min(t, a.T - 1), h);
        if (t >= a.T) orow[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float e[EPL];
        const int w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        float am = 0.0f;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            if constexpr (BF16) e[i] = __uint_as_float((i & 1) ? (static_cast<unsigned>(w[i >> 1]) & 0xffff0000u)
                                                             : (static_cast<unsigned>(w[i >> 1]) << 16));
            else e[i] = __int_as_float(w[i]);
            am = fmaxf(am, fabsf(e[i]));
        }
        const float scale = quant_scale(lanes_max<LPR>(am));
        if (orow[u] < 0 || !owner) continue;
        int qv[EPL];
        quant_row<EPL>(e, scale, qv);
        int8_t* o = qo + orow[u] * d + ls * EPL;
        if constexpr (BF16)
            *reinterpret_cast<int2*>(o) = make_int2(pack4(qv[0], qv[1], qv[2], qv[3]), pack4(qv[4], qv[5], qv[6], qv[7]));
        else *reinterpret_cast<int*>(o) = pack4(qv[0], qv[1], qv[2], qv[3]);
        if (ls == 0) so[orow[u]] = scale;
    }
}

template <int D, bool BF16, bool PAD, int LOADS>
__global__ __launch_bounds__(kSlotWaves* kWave) void slot_read_kernel(const SlotArgs a) {
    using Geo = SlotGeom<D, BF16, LOADS>;
    constexpr int EPL = Geo::EPL, LPR = Geo::LPR, RPW = Geo::RPW, U = Geo::U;
    int t0, h;
    if (!slot_unit(a, Geo::TB, t0, h)) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int d = PAD ? a.d : D;
    const int ls = PAD ? min(lane % LPR, d / EPL - 1) : lane % LPR;
    const bool owner = !PAD || ls == lane % LPR;
    const int kv = blockIdx.y & 1;
    const int64_t stride = kv ? a.v_stride : a.k_stride;
    char* x = static_cast<char*>(kv ? a.v_rows : a.k_rows) +
              (static_cast<int64_t>(h) * a.head_stride + ls * EPL) * (BF16 ? 2 : 4);
    const int8_t* qi = kv ? a.v : a.k;
    const float* si = kv ? a.vs : a.ks;
    long long irow[U];
    int2 raw[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; u++) irow[u] = slot_row(a, min(t0 + u * RPW + lane / LPR, a.T - 1), h);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long r = max(irow[u], 0LL);  // a row that is nowhere reads the pool's first and gives zeros
        const int8_t* p = qi + r * d + ls * EPL;
        if constexpr (BF16) raw[u] = *reinterpret_cast<const int2*>(p);
        else raw[u] = make_int2(*reinterpret_cast<const int*>(p), 0);
        scale[u] = si[r];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int t = t0 + u * RPW + lane / LPR;
        if (t >= a.T || !owner) continue;
        float y[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) y[i] = irow[u] < 0 ? 0.0f : sbyte(i < 4 ? raw[u].x : raw[u].y, i & 3) * scale[u];
        v4i_t out;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (BF16) out[i] = static_cast<int>(bf16_of(y[2 * i]) | (static_cast<unsigned>(bf16_of(y[2 * i + 1])) << 16));
            else out[i] = __float_as_int(y[i]);
        }
        __builtin_nontemporal_store(out, reinterpret_cast<v4i_t*>(x + t * stride * (BF16 ? 2 : 4)));
    }
}

// Any head dim, stride or alignment: a wave a row, an element a load.
template <bool BF16>
__global__ __launch_bounds__(kSlotWaves* kWave) void slot_write_generic(const SlotArgs a) {
    const int lane = threadIdx.x & (kWave - 1);
    const int kv = blockIdx.y;
    const void* x = kv ? a.v_rows : a.k_rows;
    const int64_t stride = kv ? a.v_stride : a.k_stride;
    int8_t* qo = kv ? a.v : a.k;
    float* so = kv ? a.vs : a.ks;
    const unsigned rows = static_cast<unsigned>(a.T) * a.Hkv;
    const unsigned step = gridDim.x * kSlotWaves;
    for (unsigned r = blockIdx.x * kSlotWaves + threadIdx.x / kWave; r < rows; r += step) {
        const int t = static_cast<int>(fastdiv(r, a.heads));
        const int h = static_cast<int>(r - static_cast<unsigned>(t) * a.Hkv);
        const long long orow = slot_row(a, t, h);
        if (orow < 0) continue;
        const int64_t x0 = t * stride + h * a.head_stride;
        float am = 0.0f;
        for (int i = lane; i < a.d; i += kWave) am = fmaxf(am, fabsf(row_elem<BF16>(x, x0 + i)));
        const float scale = quant_scale(wave_max(am));
        for (int i = lane; i < a.d; i += kWave)
            qo[orow * a.d + i] = static_cast<int8_t>(quant_one(row_elem<BF16>(x, x0 + i), scale));
        if (lane == 0) so[orow] = scale;
    }
}

template <bool BF16>
__global__ __launch_bounds__(kSlotWaves* kWave) void slot_read_generic(const SlotArgs a) {
    const int lane = threadIdx.x & (kWave - 1);
    const int kv = blockIdx.y;
    void* x = kv ? a.v_rows : a.k_rows;
    const int64_t stride = kv ? a.v_stride : a.k_stride;
    const int8_t* qi = kv ? a.v : a.k;
    const float* si = kv ? a.vs : a.ks;
    const unsigned rows = static_cast<unsigned>(a.T) * a.Hkv;
    const unsigned step = gridDim.x * kSlotWaves;
    for (unsigned r = blockIdx.x * kSlotWaves + threadIdx.x / kWave; r < rows; r += step) {
        const int t = static_cast<int>(fastdiv(r, a.heads));
        const int h = static_cast<int>(r - static_cast<unsigned>(t) * a.Hkv);
        const long long irow = slot_row(a, t, h);
        const float scale = irow < 0 ? 0.0f : si[irow];
        const int64_t x0 = t * stride + h * a.head_stride;
        for (int i = lane; i < a.d; i += kWave) {
            const float y = irow < 0 ? 0.0f : static_cast<float>(qi[irow * a.d + i]) * scale;
            if constexpr (BF16) static_cast<uint16_t*>(x)[x0 + i] = bf16_of(y);
            else static_cast<float*>(x)[x0 + i] = y;
        }
    }
}

// ---------------------------------------------------------------------------
// Key bounds of pages.
// ---------------------------------------------------------------------------
constexpr int kBoundsWaves = 4;

// Pages that sequence b asks for: [p0, p0 + n), and its length.
struct PageRange {
    int len, p0, n;
};
__device__ __forceinline__ PageRange bounds_range(const BoundsArgs& a, int b) {
    PageRange r;
    r.len = a.lengths ? min(max(a.lengths[b], 0), a.max_len) : a.max_len;
    const int first = a.start ? max(a.start[b], 0) : 0;
    r.p0 = first / a.pages.size;
    r.n = first < r.len ? (r.len - 1) / a.pages.size + 1 - r.p0 : 0;
    return r;
}

// Tuned head dims: a wave takes 64 / (LPT * groups) (page, kv head) units at a
// time, the heads of a page one after the other as they lie in the pool; the
// next units' page ids are on their way.
template <int LPT, Pages MODE>
__global__ __launch_bounds__(kBoundsWaves* kWave) void page_bounds_kernel(const BoundsArgs a, int groups) {
    using Wave = BoundsWave<LPT, MODE>;
    const int b = blockIdx.x;
    const PageRange r = bounds_range(a, b);
    const int units = r.n * a.Hkv;
    const int per = MODE == Pages::Several ? kWave / (LPT * groups) : 1;
    const int mine = MODE == Pages::Several ? (threadIdx.x & (kWave - 1)) / (LPT * groups) : 0;
    const int step = gridDim.y * kBoundsWaves * per;
    int u0 = (blockIdx.y * kBoundsWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) * per;
    if (u0 >= units) return;
    const Wave w(a, groups);
    const int32_t* table = a.pages.table + static_cast<size_t>(b) * a.pages.max_pages;
    struct Where {
        int pi, h, id;
    };
    auto find = [&](long long u) {  // this lane's unit of those from u on; one past the last is the last
        const unsigned x = static_cast<unsigned>(min(u + mine, static_cast<long long>(units) - 1));
        Where o;
        o.pi = static_cast<int>(fastdiv(x, a.heads));
        o.h = static_cast<int>(x) - o.pi * a.Hkv;
        o.pi += r.p0;
        o.id = table[o.pi];
        return o;
    };
    auto fetch = [&](typename Wave::Piece& p, const Where& o) { w.fetch(p, o.id, o.h, min(a.pages.size, r.len - o.pi * a.pages.size)); };
    typename Wave::Piece piece;
    Where at = find(u0);
    for (;;) {
        fetch(piece, at);
        const bool more = units - u0 > step;
        if (more) at = find(static_cast<long long>(u0) + step);
        w.finish(piece, mine < units - u0);
        if (!more) break;
        u0 += step;
    }
}

// Any head dim, page size or alignment: a wave a (page, kv head), workgroups
// blockIdx.y of sequence blockIdx.x striding over its pages.
__global__ __launch_bounds__(kBoundsWaves* kWave) void page_bounds_generic(const BoundsArgs a) {
    const int lane = threadIdx.x & (kWave - 1);
    const int b = blockIdx.x;
    const PageRange r = bounds_range(a, b);
    const long long units = static_cast<long long>(r.n) * a.Hkv;
    for (long long u = static_cast<long long>(blockIdx.y) * kBoundsWaves + threadIdx.x / kWave; u < units;
         u += static_cast<long long>(gridDim.y) * kBoundsWaves) {
        const int pi = r.p0 + static_cast<int>(u / a.Hkv);
        const int h = static_cast<int>(u % a.Hkv);
        bounds_generic(a, b, pi, h, min(a.pages.size, r.len - pi * a.pages.size), lane);
    }
}

}  // namespace

// Each workgroup scans the whole batch, so more of them only share out what comes
// after, of which the releases of a decode step are not known here: one for each
// 32 rows, up to 128 (steps of 1000 sequences 7.6 us, with one for each 256 rows
// 9.6, each 2048 16.4; of 256 sequences 7.8 / 8.1 / 8.1; of 64 6.4 / 6.2 / 6.2;
// 131008 rows of 64 prompts 6.0 in 128, 6.4 in 64, 7.9 in 32 workgroups).
// Without arrays of rows the pages are what there is to do.
constexpr int kMapRows = 32, kMapGroups = 128;
int page_map_groups(const PageMapArgs& a) {
    const long long work = a.slot_map || a.token_seq || a.token_pos
                               ? a.T
                               : min(static_cast<long long>(a.T / static_cast<int>(a.page.d)) + a.B, static_cast<long long>(a.num_pages));
    return static_cast<int>(max(1LL, min(static_cast<long long>(kMapGroups), (work + kMapRows - 1) / kMapRows)));
}

hipError_t launch_page_map(const PageMapArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(page_map_groups(a))), block(kMapThreads);
    const size_t lds = sizeof(int) * (4 * static_cast<size_t>(a.B) + 3);
    if (a.B <= kMapThreads) hipLaunchKernelGGL(page_map_kernel<1>, grid, block, lds, stream, a);
    else hipLaunchKernelGGL(page_map_kernel<4>, grid, block, lds, stream, a);
    return hipGetLastError();
}

namespace {
dim3 slot_grid(unsigned rows, unsigned rows_per_group) {
    const unsigned groups = (rows + rows_per_group - 1) / rows_per_group;
    return dim3(groups < kSlotGroups ? groups : kSlotGroups, 2);
}
}  // namespace

namespace {
template <bool BF16>
hipError_t launch_slots(const SlotArgs& a, bool write, bool vec_ok, hipStream_t stream) {
    if (a.T == 0) return hipSuccess;
    const dim3 block(kSlotWaves * kWave);
    // Rows of whole 16-byte pieces up to 256 elements; others, and misaligned
    // ones, go to the generic kernels.
    if (vec_ok && a.d <= 256 && a.d % (BF16 ? 8 : 4) == 0) {
        auto units = [&](int tb) { return (static_cast<long long>(a.T) + tb - 1) / tb * a.Hkv; };  // waves of K or of V
        auto grid = [&](int tb) {
            const unsigned groups = static_cast<unsigned>((units(tb) + kSlotWaves - 1) / kSlotWaves);
            return dim3(groups < kSlotGroups ? groups : kSlotGroups, 2 * ((groups + kSlotGroups - 1) / kSlotGroups));
        };
#define KVQ_SLOT_LAUNCH(KERNEL, LOADS) \
    hipLaunchKernelGGL(KERNEL, grid(SlotGeom<DD, BF16, LOADS>::TB), block, 0, stream, a)
#define KVQ_SLOT_CASE(DIM)                                                                                             \
    if (a.d <= DIM) {                                                                                                  \
        constexpr int DD = DIM;                                                                                        \
        const bool few = units(SlotGeom<DD, BF16, kReadLoads>::TB) < 4096;                                             \
        if (write && a.d == DD) KVQ_SLOT_LAUNCH((slot_write_kernel<DD, BF16, false>), kWriteLoads);                    \
        else if (write) KVQ_SLOT_LAUNCH((slot_write_kernel<DD, BF16, true>), kWriteLoads);                             \
        else if (few && a.d == DD) KVQ_SLOT_LAUNCH((slot_read_kernel<DD, BF16, false, kSmallReadLoads>), kSmallReadLoads); \
        else if (few) KVQ_SLOT_LAUNCH((slot_read_kernel<DD, BF16, true, kSmallReadLoads>), kSmallReadLoads);           \
        else if (a.d == DD) KVQ_SLOT_LAUNCH((slot_read_kernel<DD, BF16, false, kReadLoads>), kReadLoads);              \
        else KVQ_SLOT_LAUNCH((slot_read_kernel<DD, BF16, true, kReadLoads>), kReadLoads);                              \
        return hipGetLastError();                                                                                      \
    }
        KVQ_SLOT_CASE(32)
        KVQ_SLOT_CASE(64)
        KVQ_SLOT_CASE(128)
        KVQ_SLOT_CASE(256)
#undef KVQ_SLOT_CASE
#undef KVQ_SLOT_LAUNCH
    }
    const dim3 grid = slot_grid(static_cast<unsigned>(a.T) * a.Hkv, kSlotWaves);
    if (write) hipLaunchKernelGGL((slot_write_generic<BF16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((slot_read_generic<BF16>), grid, block, 0, stream, a);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_slot_write(const SlotArgs& a, bool bf16, bool vec_ok, hipStream_t stream) {
    return bf16 ? launch_slots<true>(a, true, vec_ok, stream) : launch_slots<false>(a, true, vec_ok, stream);
}
hipError_t launch_slot_read(const SlotArgs& a, bool bf16, bool vec_ok, hipStream_t stream) {
    return bf16 ? launch_slots<true>(a, false, vec_ok, stream) : launch_slots<false>(a, false, vec_ok, stream);
}

namespace {
template <int LPT>
void launch_bounds_pages(const BoundsArgs& a, int groups, dim3 grid, dim3 block, hipStream_t stream) {
    if (groups < kWave / LPT) hipLaunchKernelGGL((page_bounds_kernel<LPT, Pages::Several>), grid, block, 0, stream, a, groups);
    else if (a.pages.size <= 16 * groups) hipLaunchKernelGGL((page_bounds_kernel<LPT, Pages::One>), grid, block, 0, stream, a, groups);
    else hipLaunchKernelGGL((page_bounds_kernel<LPT, Pages::Passes>), grid, block, 0, stream, a, groups);
}
}  // namespace

hipError_t launch_page_bounds(const BoundsArgs& a, bool vec_ok, hipStream_t stream) {
    const bool tuned = vec_ok && a.d <= 256 && a.d % 16 == 0;
    const int lanes = bounds_lanes(a.d);
    const int groups = bounds_groups(a.pages.size, lanes);
    // A sequence's workgroups stride over its pages: about 4096 in all at most
    // (generic: 8192), more than the three rounds that fit the CUs at a time, so
    // that ragged batches fill them (16 prompts of up to 8192 tokens: 23.8 us
    // with 1024, 21.0 with 4096, 20.7 with 16384).
    const long long units = (static_cast<long long>(a.max_len - 1) / a.pages.size + 1) * a.Hkv;
    const int per = tuned ? kBoundsWaves * (kWave / (lanes * groups)) : kBoundsWaves;
    const long long most = tuned ? 4096 : 8192;
    const unsigned ny = static_cast<unsigned>(min((units + per - 1) / per, max(1LL, most / a.B)));
    const dim3 grid(static_cast<unsigned>(a.B), ny), block(kBoundsWaves * kWave);
    if (!tuned) hipLaunchKernelGGL(page_bounds_generic, grid, block, 0, stream, a);
    else if (lanes == 4) launch_bounds_pages<4>(a, groups, grid, block, stream);
    else if (lanes == 8) launch_bounds_pages<8>(a, groups, grid, block, stream);
    else if (lanes == 16) launch_bounds_pages<16>(a, groups, grid, block, stream);
    else launch_bounds_pages<32>(a, groups, grid, block, stream);
    return hipGetLastError();
}

}  // namespace kvq
