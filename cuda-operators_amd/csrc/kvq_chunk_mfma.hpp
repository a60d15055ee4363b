// kvq_chunk_mfma.hpp -- chunk attention on gfx950's f16 matrix cores.
#pragma once

#include <limits.h>
#include <math.h>

#include "kvq_chunk.hpp"
#include "kvq_device.hpp"

namespace kvq {
namespace {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kChunkWaves = 4;
constexpr int kChunkThreads = kChunkWaves * kWave;
constexpr int kChunkCoherent = 16;  // buffer cache policy sc1: device-coherent
constexpr float kWeightTop = 15.0f;   // log2 of the largest f16 weight that is let grow,
constexpr float kWeightReset = 12.0f; // and of what a row's weights are set to when they pass it
constexpr float kKsMax = 0x1p80f;     // |k scale|s above overflow as scores of q scaled to 2^15
constexpr float kVsMax = 0x1p40f, kVsMin = 0x1p-40f;  // |v scale|s outside take fp32 weights, as does a
template <int LIMBS>                                  // tile set whose scales differ by more than this
constexpr float kVsRatio = LIMBS == 1 ? 0x1p18f : 0x1p14f;

// Eight int8 as f16: each byte, made unsigned, under the exponent of 1024, so
// kCodeBias + code; then f of each pair.
constexpr float kCodeBias = 1152.0f;
template <class F>
__device__ __forceinline__ h16x8 codes_to_f16(int2 w, F&& f) {
    const unsigned x = static_cast<unsigned>(w.x) ^ 0x80808080u, y = static_cast<unsigned>(w.y) ^ 0x80808080u;
    auto pair = [&](unsigned z, unsigned sel) { return f(__builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, z, sel))); };
    const h16x2 a = pair(x, 0x04010400u), b = pair(x, 0x04030402u), c = pair(y, 0x04010400u), e = pair(y, 0x04030402u);
    return h16x8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

// x times lane I's y of the 16-lane row.
template <int I>
__device__ __forceinline__ float times_lane(float x, float y) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x150 + I, 0xF, 0xF, true)) * x;
}
template <int I = 0>
__device__ __forceinline__ void times_lanes(f32x16& x, float y) {
    if constexpr (I < 16) {
        x[I] = times_lane<I>(x[I], y);
        times_lanes<I + 1>(x, y);
    }
}

// What a workgroup computes: query tile `tile` of sequence b and one kv head,
// over key blocks [k0, k1) of the tile's, as split `split` of nsplit.
struct ChunkItem {
    int b, tile, split, nsplit;
    int unit;  // split tiles' counter
    int rec;   // first of the tile's records
};

// Sequence b's query tiles and key blocks.
__device__ __forceinline__ void chunk_counts(const ChunkArgs& a, const ChunkSeq& s, int& tiles, int& blocks) {
    tiles = (s.n + a.tile_tokens - 1) / a.tile_tokens;
    blocks = (s.len + kChunkKeys - 1) / kChunkKeys;
}

// The plan, derived by every workgroup from the lengths.  Where the tiles alone
// are a.slots workgroups or more, each is one item.  Otherwise keys are split into
// chunks of the fewest blocks (in steps) with which the items are at most a.slots;
// all tiles of a sequence have the same number of splits.
struct ChunkPlanLds {
    int part[kChunkWaves], best[kChunkWaves];
    int tiles[kChunkThreads], blocks[kChunkThreads];
    int found[6];
};
__device__ inline bool chunk_locate(const ChunkArgs& a, ChunkPlanLds& s, int r, ChunkItem& w) {
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1), wave = t / kWave;
    const int per = (a.B + kChunkThreads - 1) / kChunkThreads;
    const int b0 = t * per;
    auto counts = [&](int b, int& tiles, int& blocks) {
        tiles = blocks = 0;
        if (b < a.B) chunk_counts(a, chunk_seq(a, b), tiles, blocks);
    };
    auto sum = [&](int v, int& total) {  // exclusive scan
        const int incl = wave_inclusive_scan(v);
        if (lane == kWave - 1) s.part[wave] = incl;
        __syncthreads();
        int before = 0;
        total = 0;
#pragma unroll
        for (int i = 0; i < kChunkWaves; i++) {
            if (i < wave) before += s.part[i];
            total += s.part[i];
        }
        __syncthreads();
        return before + incl - v;
    };
    int mine = 0, first_tiles = 0, first_blocks = 0;
    for (int i = 0; i < per; i++) {
        int tiles, blocks;
        counts(b0 + i, tiles, blocks);
        if (i == 0) first_tiles = tiles, first_blocks = blocks;
        mine += tiles;
    }
    int all;
    int before = sum(mine, all);
    int chunk = 0;  // 0: nothing is split
    if (a.max_splits > 1 && static_cast<long long>(all) * a.Hkv < a.slots && all <= a.max_tiles && per == 1) {
        // Candidates: chunks of i + 1 steps; the smallest one that fits.
        s.tiles[t] = first_tiles;
        s.blocks[t] = first_blocks;
        __syncthreads();
        const int top = (a.max_len + kChunkKeys - 1) / kChunkKeys;
        const int least = max(1, (top + a.max_splits - 1) / a.max_splits);
        const int step = (top - least) / (kChunkThreads - 1) + 1;
        const int c = least + t * step;
        int items = 0;
        for (int b = 0; b < a.B; b++) items += s.tiles[b] * max(1, (s.blocks[b] + c - 1) / c);
        const unsigned long long fits = __builtin_amdgcn_ballot_w64(static_cast<long long>(items) * a.Hkv <= a.slots);
        if (lane == 0) s.best[wave] = fits ? __builtin_ctzll(fits) + wave * kWave : INT_MAX;
        __syncthreads();
        int best = INT_MAX;
#pragma unroll
        for (int i = 0; i < kChunkWaves; i++) best = min(best, s.best[i]);
        chunk = best == INT_MAX ? top : least + best * step;
        mine = first_tiles * max(1, (first_blocks + chunk - 1) / chunk);
        before = sum(mine, all);
    }
    if (r >= all) return false;
    if (r >= before && r < before + mine) {
        int at = before;
        for (int i = 0; i < per; i++) {
            int tiles = first_tiles, blocks = first_blocks;
            if (i > 0) counts(b0 + i, tiles, blocks);
            const int nsplit = chunk > 0 ? max(1, (blocks + chunk - 1) / chunk) : 1;
            if (r < at + tiles * nsplit) {
                const int local = r - at;
                const int tile = local / nsplit;
                s.found[0] = b0 + i;
                s.found[1] = tiles - 1 - tile;  // the longest first
                s.found[2] = local - tile * nsplit;
                s.found[3] = nsplit;
                s.found[4] = at + tile * nsplit;
                break;
            }
            at += tiles * nsplit;
        }
    }
    __syncthreads();
    w.b = __builtin_amdgcn_readfirstlane(s.found[0]);
    w.tile = __builtin_amdgcn_readfirstlane(s.found[1]);
    w.split = __builtin_amdgcn_readfirstlane(s.found[2]);
    w.nsplit = __builtin_amdgcn_readfirstlane(s.found[3]);
    w.rec = __builtin_amdgcn_readfirstlane(s.found[4]);
    return true;
}

// LDS exchange within a wave.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One row by one wave in fp32, over keys [k0, k1): for values that f16 weights do
// not hold.  scratch: 2 D + 64 floats and 64 row numbers.
template <int D>
__device__ __forceinline__ void chunk_row_f32(const ChunkArgs& a, int b, int kvh, int64_t q_at, int k0, int k1, float* scratch,
                                              float& m, float& l) {
    float* s_q = scratch;
    float* s_acc = s_q + D;
    float* s_w = s_acc + D;
    size_t* s_row = reinterpret_cast<size_t*>(s_w + kWave);
    const int lane = threadIdx.x & (kWave - 1);
    for (int i = lane; i < D; i += kWave) {
        s_q[i] = i < a.d ? chunk_load(a, q_at + i) : 0.0f;
        s_acc[i] = 0.0f;
    }
    m = -INFINITY;
    l = 0.0f;
    for (int t0 = k0; t0 < k1; t0 += kWave) {
        wave_sync();
        float x = -INFINITY;
        size_t row = 0;
        const bool in = t0 + lane < k1;
        if (in) {
            row = cache_row(a.pages, a.Hkv, 0, b, kvh, t0 + lane);
            float dot = 0.0f;
            for (int i = 0; i < a.d; i++) dot = fmaf(s_q[i], static_cast<float>(a.k[row * a.d + i]), dot);
            x = dot * a.ks[row] * a.scale_log2;
        }
        const float mn = fmaxf(m, wave_max(x));
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float alpha = fast_exp2(m - ms);
        const float p = fast_exp2(x - ms);
        m = mn;
        l = l * alpha + (in ? p : 0.0f);
        s_w[lane] = in ? p * a.vs[row] : 0.0f;
        s_row[lane] = row;
        wave_sync();
        const int n = min(kWave, k1 - t0);
        for (int i = lane; i < a.d; i += kWave) {
            float acc = s_acc[i] * alpha;
            for (int k = 0; k < n; k++) acc = fmaf(s_w[k], static_cast<float>(a.v[s_row[k] * a.d + i]), acc);
            s_acc[i] = acc;
        }
    }
    l = wave_sum(l);
    wave_sync();
}

template <int D, int LIMBS>
__global__ __launch_bounds__(kChunkThreads) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void chunk_mfma(
    const ChunkArgs a) {
    constexpr int KS = D + 8, VS = D + 16;     // LDS row strides in f16
    constexpr int NS = D / 16;                 // QK contraction steps
    constexpr int NB = D / 32;                 // output blocks
    constexpr int PPR = D / 8;                 // 8-code pieces of a row
    constexpr int NP = kChunkKeys * PPR / kChunkThreads;  // a thread's, of K and of V
    static_assert(D % 32 == 0 && kChunkKeys * PPR % kChunkThreads == 0, "whole pieces");
    struct alignas(16) Buf {
        _Float16 k[kChunkKeys * KS];
        _Float16 v[kChunkKeys * VS];
    };
    // A tile's scales, in the slot of its number: kept four, as rows and scales
    // are fetched up to three tiles ahead.
    struct Scales {
        long long row[kChunkKeys];  // pool rows
        float ks[kChunkKeys];
        float vs[kChunkKeys];       // LIMBS == 1: two f16 of vs / 2^lv
        float lv, unit;             // |vs| <= 2^lv; 2^-lv
    };
    __shared__ __align__(16) Buf s_buf[2];
    __shared__ __align__(16) Scales s_scale[4];
    __shared__ ChunkPlanLds s_plan;
    __shared__ int s_flag;

    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int c32 = lane & 31, h = lane >> 5, c16 = lane & 15;
    const int r = static_cast<int>(fastdiv(blockIdx.x, a.heads));
    const int kvh = static_cast<int>(blockIdx.x) - r * a.Hkv;
    ChunkItem w;
    if (!chunk_locate(a, s_plan, r, w)) return;
    const ChunkSeq s = chunk_seq(a, w.b);
    const int i0 = w.tile * a.tile_tokens;                       // the tile's new tokens
    const int tokens = min(a.tile_tokens, s.n - i0);
    const int kend = chunk_keys(a, s, i0 + tokens - 1);          // keys that any of them attends
    const int nblocks = (kend + kChunkKeys - 1) / kChunkKeys;
    const int share = (nblocks + w.nsplit - 1) / w.nsplit;
    const int k0 = min(w.split * share, nblocks) * kChunkKeys;
    const int k1 = min(min((w.split + 1) * share, nblocks) * kChunkKeys, kend);
    const int tiles = k1 > k0 ? (k1 - k0 + kChunkKeys - 1) / kChunkKeys : 0;

    // This lane's query row: (token, head) = divmod(row, G).
    const int row = wave * 32 + c32;
    const int tok = static_cast<int>(fastdiv(row, a.group));
    const int head = kvh * a.G + row - tok * a.G;
    const bool live = tok < tokens;
    const int keys = live ? chunk_keys(a, s, i0 + tok) : 0;
    const int64_t q_at = static_cast<int64_t>(s.row0 + i0 + tok) * a.q_stride + static_cast<int64_t>(head) * a.d;
    const int wave_rows = min(max(tokens * a.G - wave * 32, 0), 32);  // live rows of this wave
    // Keys that every live row of the wave attends, and that any does.
    const int first_tok = static_cast<int>(fastdiv(wave * 32, a.group));
    const int last_tok = static_cast<int>(fastdiv(wave * 32 + max(wave_rows, 1) - 1, a.group));
    const int keys_all = __builtin_amdgcn_readfirstlane(wave_rows > 0 ? chunk_keys(a, s, i0 + first_tok) : 0);
    const int keys_any = __builtin_amdgcn_readfirstlane(wave_rows > 0 ? chunk_keys(a, s, i0 + last_tok) : 0);

    // Pool row of key t0 + (t % 64) (past the end: the last key's again).
    const int32_t* table = a.pages.table + static_cast<size_t>(w.b) * a.pages.max_pages;
    auto page_of = [&](int tile) { return static_cast<int>(fastdiv(min(k0 + tile * kChunkKeys + lane, max(k1 - 1, 0)), a.page)); };
    auto pool_row = [&](int tile, int id) {
        const int key = min(k0 + tile * kChunkKeys + lane, max(k1 - 1, 0));
        const int page = static_cast<int>(fastdiv(key, a.page));
        id = min(max(id, 0), a.pages.num_pages - 1);
        return (static_cast<long long>(id) * a.Hkv + kvh) * a.pages.size + (key - page * a.pages.size);
    };

    int2 kraw[NP], vraw[NP];
    float ksr = 0.0f, vsr = 0.0f;
    float vmax = 0.0f, vmin = INFINITY, kmax = 0.0f;
    bool vbad = false;
    auto load_tile = [&](int tile) {
        const long long* rows = s_scale[tile & 3].row;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int piece = i * kChunkThreads + t;
            const int kr = piece / PPR, c = (piece - kr * PPR) * 8;
            const long long at = rows[kr] * a.d + c;
            const bool in = c < a.d;
            kraw[i] = in ? *reinterpret_cast<const int2*>(a.k + at) : make_int2(0, 0);
            vraw[i] = in ? *reinterpret_cast<const int2*>(a.v + at) : make_int2(0, 0);
        }
    };
    // Codes become f16 here, once a workgroup.  bf16: K keeps its bias (taken off
    // in the accumulators' start), V is scaled by vs / 2^lv, rounded to f16; fp32:
    // codes are exact.
    auto store_tile = [&](int tile) {
        Buf& buf = s_buf[tile & 1];
        const h16x2 bias = {static_cast<_Float16>(kCodeBias), static_cast<_Float16>(kCodeBias)};
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int piece = i * kChunkThreads + t;
            const int kr = piece / PPR, c = (piece - kr * PPR) * 8;
            *reinterpret_cast<h16x8*>(buf.k + kr * KS + c) =
                codes_to_f16(kraw[i], [&](h16x2 x) { return LIMBS == 1 ? x : x - bias; });
            const h16x2 f = LIMBS == 1 ? __builtin_bit_cast(h16x2, s_scale[tile & 3].vs[kr]) : bias;
            *reinterpret_cast<h16x8*>(buf.v + kr * VS + c) =
                codes_to_f16(vraw[i], [&](h16x2 x) { return LIMBS == 1 ? (x - bias) * f : x - bias; });
        }
    };
    // Wave 0 looks after rows and scales, a key a lane.
    auto load_scales = [&](int tile, long long at) {
        s_scale[tile & 3].row[lane] = at;
        ksr = a.ks[at];
        vsr = a.vs[at];
        if (k0 + tile * kChunkKeys + lane >= k1) ksr = vsr = 0.0f;
    };
    auto store_scales = [&](int tile) {
        Scales& x = s_scale[tile & 3];
        const float v = fabsf(vsr);
        kmax = fmaxf(kmax, fabsf(ksr));
        vbad |= !(v < INFINITY);
        vmax = fmaxf(vmax, v);
        if (v > 0.0f) vmin = fminf(vmin, v);
        const int e = min(max(__builtin_amdgcn_frexp_expf(lanes_max<kWave>(v)), -60), 60);
        x.ks[lane] = ksr;
        const _Float16 h = static_cast<_Float16>(ldexpf(vsr, -e));
        x.vs[lane] = LIMBS == 1 ? __builtin_bit_cast(float, h16x2{h, h}) : vsr;
        if (lane == 0) {
            x.lv = static_cast<float>(e);
            x.unit = ldexpf(1.0f, -e);
        }
    };
    int next_id = 0;
    if (tiles > 0 && wave == 0) {
        const int id0 = table[page_of(0)], id1 = table[page_of(1)], id2 = table[page_of(2)];
        next_id = table[page_of(3)];
        load_scales(0, pool_row(0, id0));
        store_scales(0);
        load_scales(1, pool_row(1, id1));
        store_scales(1);
        load_scales(2, pool_row(2, id2));
    }

    // q^T operands: lane has dims 16 s + 8 h + [0, 8) of its row, scaled to 2^15.
    h16x8 q[LIMBS][NS];
    float c_row;
    float start = 0.0f;  // of a score's sum: minus the codes' bias times the sum of q
    {
        float x[NS][8];
        float top = 0.0f;
        bool bad = false;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const int dim = 16 * n + 8 * h;
            const bool in = live && dim < a.d;
            if (LIMBS == 1) {
                uint4 raw = make_uint4(0, 0, 0, 0);
                if (in) raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + q_at + dim);
                const unsigned u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[n][2 * j] = __uint_as_float(u[j] << 16);
                    x[n][2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                }
            } else {
                float4 y = make_float4(0, 0, 0, 0), z = y;
                if (in) {
                    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + q_at + dim);
                    y = p[0];
                    z = p[1];
                }
                x[n][0] = y.x, x[n][1] = y.y, x[n][2] = y.z, x[n][3] = y.w;
                x[n][4] = z.x, x[n][5] = z.y, x[n][6] = z.z, x[n][7] = z.w;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                top = fmaxf(top, fabsf(x[n][j]));
                bad |= !(fabsf(x[n][j]) < INFINITY);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        bad |= __shfl_xor(static_cast<int>(bad), 32) != 0;
        const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
        c_row = fmaxf(ldexpf(a.scale_log2, e), 0x1p-126f);
        if (bad) c_row = NAN;
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = bad ? 0.0f : ldexpf(x[n][j], -e);
                q[0][n][j] = static_cast<_Float16>(y);
                if (LIMBS == 1) start -= static_cast<float>(q[0][n][j]);
                if (LIMBS == 2) q[LIMBS - 1][n][j] = static_cast<_Float16>(y - static_cast<float>(q[0][n][j]));
            }
    }

    f32x16 sum0;
    if (LIMBS == 1) start = (start + __shfl_xor(start, 32)) * kCodeBias;
#pragma unroll
    for (int i = 0; i < 16; i++) sum0[i] = start;
    f32x16 o[NB];
#pragma unroll
    for (int c = 0; c < NB; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[c][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // Keys of this lane's score registers: block 32 kb, register i: 32 kb + 8 (i / 4) + 4 h + i % 4.
    const int scale_at = 8 * (c16 >> 2) + 4 * h + (c16 & 3);
    auto compute = [&](int tile) {
        const Buf& buf = s_buf[tile & 1];
        const Scales& sc = s_scale[tile & 3];
        const int t0 = k0 + tile * kChunkKeys;
        f32x16 p[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            f32x16 acc = sum0, low;
#pragma unroll
            for (int i = 0; i < 16; i++) low[i] = 0.0f;
            const _Float16* kp = buf.k + (32 * kb + c32) * KS + 8 * h;
#pragma unroll
            for (int n = 0; n < NS; n++) {
                const h16x8 x = *reinterpret_cast<const h16x8*>(kp + 16 * n);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[0][n], acc, 0, 0, 0);
                if (LIMBS == 2) low = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[LIMBS - 1][n], low, 0, 0, 0);
            }
            if (LIMBS == 2) acc += low;
            times_lanes(acc, sc.ks[32 * kb + scale_at]);
            p[kb] = acc;
        }
        if (t0 + kChunkKeys > keys_all) {
            asm volatile("");  // a branch, not selects: most tiles need no mask (95 of 575 VALU slots of a tile)
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (t0 + 32 * kb + 8 * (i / 4) + 4 * h + i % 4 >= keys) p[kb][i] = -INFINITY;
        }
        float top = p[0][0];
#pragma unroll
        for (int i = 1; i < 32; i++) top = fmaxf(top, p[i / 16][i % 16]);
        const float u = fmaf(top, c_row, sc.lv);
        if (__builtin_amdgcn_ballot_w64(u > m + kWeightTop) != 0) {
            const float un = fmaxf(u, __shfl_xor(u, 32)) - kWeightReset;
            const float mn = un > m ? un : m;
            const float alpha = mn == -INFINITY ? 1.0f : fast_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int c = 0; c < NB; c++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[c][i] *= alpha;
        }
        const float ms = (m == -INFINITY ? 0.0f : m) - (LIMBS == 1 ? sc.lv : 0.0f);
        h16x8 wt[LIMBS][4];
        // Summed by itself, so l rounds once a tile (2000 keys in fp32: error 2.0e-6 with a sum key by key).
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                p[kb][i] = fast_exp2(fmaf(p[kb][i], c_row, -ms));
                part[i % 4] += p[kb][i];
            }
            if (LIMBS == 2) times_lanes(p[kb], sc.vs[32 * kb + scale_at]);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (LIMBS == 2) {
                    // One value for both limbs: contracted into one of them, the product would be
                    // rounded once there and twice here, 2^-10 apart in one weight of some thousand.
                    float x = p[kb][i];
                    asm("" : "+v"(x));
                    p[kb][i] = x;
                }
                const _Float16 hi = static_cast<_Float16>(p[kb][i]);
                wt[0][2 * kb + i / 8][i % 8] = hi;
                if (LIMBS == 2) wt[LIMBS - 1][2 * kb + i / 8][i % 8] = static_cast<_Float16>(p[kb][i] - static_cast<float>(hi));
            }
        }
        l = fmaf((part[0] + part[1]) + (part[2] + part[3]), LIMBS == 1 ? sc.unit : 1.0f, l);
        // Keys 16 n + 8 j + 4 h + [0, 4), j = 0, 1, are the lane's 8 slots of step n.
        const _Float16* vp = buf.v + (4 * h + (c16 >> 2)) * VS + 16 * ((lane >> 4) & 1) + 4 * (c16 & 3);
#pragma unroll
        for (int n = 0; n < 4; n++) {
#pragma unroll
            for (int c = 0; c < NB; c++) {
                const _Float16* x = vp + 16 * n * VS + 32 * c;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(const_cast<_Float16*>(x)));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(const_cast<_Float16*>(x + 8 * VS)));
                const h16x8 v = __builtin_bit_cast(h16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, wt[0][n], o[c], 0, 0, 0);
                if (LIMBS == 2) o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, wt[LIMBS - 1][n], o[c], 0, 0, 0);
            }
        }
    };

    __syncthreads();
    if (tiles > 0) {
        load_tile(0);
        store_tile(0);
        if (tiles > 1) load_tile(1);
    }
    __syncthreads();
    // Iteration i: tile i + 1 becomes f16 in the buffer that was last read before
    // the last barrier, codes of tile i + 2 are on their way, scales of tile i + 2
    // are stored, and rows and scales of tile i + 3 fetched; the slot of those held
    // tile i - 1's.
    for (int i = 0; i < tiles; i++) {
        if (i + 1 < tiles) store_tile(i + 1);
        if (i + 2 < tiles) load_tile(i + 2);
        if (wave == 0 && i + 2 < tiles) {
            store_scales(i + 2);
            if (i + 3 < tiles) load_scales(i + 3, pool_row(i + 3, next_id));
            next_id = table[page_of(i + 4)];
        }
        if (k0 + i * kChunkKeys < keys_any) compute(i);
        __syncthreads();
    }

    // Scales that f16 weights, or q scaled to 2^15, do not cover.
    if (wave == 0) {
        const float top = wave_max(vmax), low = -wave_max(-vmin);
        const bool bad = __builtin_amdgcn_ballot_w64(vbad || kmax > kKsMax) != 0 ||
                         (top > 0.0f && (top > kVsMax || low < kVsMin || top > low * kVsRatio<LIMBS>));
        if (lane == 0) s_flag = bad;
    }
    __syncthreads();
    l += __shfl_xor(l, 32);
    const bool exact = s_flag != 0;
    const bool whole = w.nsplit == 1;
    const size_t item = static_cast<size_t>(w.rec + w.split) * a.Hkv + kvh;
    const buf_rsrc acc_rs = make_rsrc(a.part_acc + (whole ? 0 : item * kChunkRows * D), kChunkRows * D * 4u);
    const buf_rsrc ml_rs = make_rsrc(a.part_ml + (whole ? 0 : item * kChunkRows * 2), kChunkRows * 8u);
    const int64_t o_at = static_cast<int64_t>(s.row0 + i0 + tok) * a.out_stride + static_cast<int64_t>(head) * a.d;
    auto put4 = [&](int64_t at, float x, float y, float z, float u) {
        if (LIMBS == 1) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
                make_uint2(bf16_of(x) | static_cast<unsigned>(bf16_of(y)) << 16, bf16_of(z) | static_cast<unsigned>(bf16_of(u)) << 16);
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x, y, z, u);
        }
    };
    if (!exact) {
        if (live) {
            const float inv = keys > 0 ? 1.0f / l : 0.0f;
#pragma unroll
            for (int c = 0; c < NB; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int dim = 32 * c + 8 * j + 4 * h;
                    if (whole) {
                        if (dim >= a.d) continue;
                        if (keys > 0) put4(o_at + dim, o[c][4 * j] * inv, o[c][4 * j + 1] * inv, o[c][4 * j + 2] * inv, o[c][4 * j + 3] * inv);
                        else put4(o_at + dim, 0.0f, 0.0f, 0.0f, 0.0f);
                    } else {
                        const v4i_t x = {__float_as_int(o[c][4 * j]), __float_as_int(o[c][4 * j + 1]),
                                         __float_as_int(o[c][4 * j + 2]), __float_as_int(o[c][4 * j + 3])};
                        __builtin_amdgcn_raw_buffer_store_b128(x, acc_rs, (row * D + dim) * 4, 0, kChunkCoherent);
                    }
                }
            if (!whole && h == 0) {
                typedef int v2i_t __attribute__((ext_vector_type(2)));
                __builtin_amdgcn_raw_buffer_store_b64(v2i_t{__float_as_int(m), __float_as_int(l)}, ml_rs, row * 8, 0, kChunkCoherent);
            }
        }
    } else {
        float* const scratch = reinterpret_cast<float*>(s_buf) + wave * (2 * D + kWave + 2 * kWave);
        const float* s_acc = scratch + D;
        for (int j = 0; j < wave_rows; j++) {
            const int jt = static_cast<int>(fastdiv(wave * 32 + j, a.group));
            const int jh = kvh * a.G + wave * 32 + j - jt * a.G;
            const int jkeys = chunk_keys(a, s, i0 + jt);
            float jm, jl;
            chunk_row_f32<D>(a, w.b, kvh, static_cast<int64_t>(s.row0 + i0 + jt) * a.q_stride + static_cast<int64_t>(jh) * a.d, k0,
                             min(k1, jkeys), scratch, jm, jl);
            const int64_t at = static_cast<int64_t>(s.row0 + i0 + jt) * a.out_stride + static_cast<int64_t>(jh) * a.d;
            for (int i = lane; i < D; i += kWave) {
                if (whole) {
                    if (i < a.d) chunk_store(a, at + i, jkeys > 0 ? s_acc[i] / jl : 0.0f);
                } else {
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(s_acc[i]), acc_rs, ((wave * 32 + j) * D + i) * 4, 0, kChunkCoherent);
                }
            }
            if (!whole && lane < 2)
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(lane ? jl : jm), ml_rs, (wave * 32 + j) * 8 + lane * 4, 0, kChunkCoherent);
            wave_sync();
        }
    }
    if (whole) return;

    // The last of the tile's workgroups joins the records.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t == 0) {
        int* const counter = a.counters + static_cast<size_t>(w.rec) * a.Hkv + kvh;
        const int prev = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_flag = prev == w.nsplit - 1;
        if (prev == w.nsplit - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s_flag == 0) return;
    const size_t rec0 = static_cast<size_t>(w.rec) * a.Hkv + kvh;
    constexpr int LPR = D / 4;                   // lanes a row
    constexpr int RPP = kChunkThreads / LPR;     // rows a pass
    const int live_rows = tokens * a.G;
    for (int jr = t / LPR; jr < live_rows; jr += RPP) {
        if (t / LPR >= RPP) break;
        const int dim = 4 * (t % LPR);
        float M = -INFINITY;
        for (int i = 0; i < w.nsplit; i++) {
            const float* ml = a.part_ml + ((rec0 + static_cast<size_t>(i) * a.Hkv) * kChunkRows + jr) * 2;
            M = fmaxf(M, __hip_atomic_load(ml, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        }
        const float Ms = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, A[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < w.nsplit; i++) {
            const size_t rec = rec0 + static_cast<size_t>(i) * a.Hkv;
            const float* ml = a.part_ml + (rec * kChunkRows + jr) * 2;
            const float mi = __hip_atomic_load(ml, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const float li = __hip_atomic_load(ml + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const buf_rsrc rs = make_rsrc(a.part_acc + rec * kChunkRows * D, kChunkRows * D * 4u);
            const v4i_t x = __builtin_amdgcn_raw_buffer_load_b128(rs, (jr * D + dim) * 4, 0, kChunkCoherent);
            if (mi == -INFINITY && li == 0.0f) continue;  // no key of this split
            const float f = fast_exp2(mi - Ms);
            L = fmaf(li, f, L);
#pragma unroll
            for (int j = 0; j < 4; j++) A[j] = fmaf(__int_as_float(x[j]), f, A[j]);
        }
        const int jt = static_cast<int>(fastdiv(jr, a.group));
        const int jh = kvh * a.G + jr - jt * a.G;
        const bool any = chunk_keys(a, s, i0 + jt) > 0;
        const float inv = any ? 1.0f / L : 0.0f;
        const int64_t at = static_cast<int64_t>(s.row0 + i0 + jt) * a.out_stride + static_cast<int64_t>(jh) * a.d + dim;
        if (dim < a.d) {
            if (any) put4(at, A[0] * inv, A[1] * inv, A[2] * inv, A[3] * inv);
            else put4(at, 0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
}

}  // namespace
}  // namespace kvq
