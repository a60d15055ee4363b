// kvq_chunk_mfma.hpp -- chunk attention on gfx950's f16 matrix cores.
//
// A query row (one head of one new token) over the keys j that it sees, of int8
// codes k_j, v_j with scales ks_j, vs_j, one of each a key and kv head:
//   s_j = ks_j (q . k_j) scale log2(e),  p_j = 2^(s_j - m),
//   out = sum p_j vs_j v_j / sum p_j,
// in one pass with a running m and sum.  int8 codes are exact in f16, so both
// products run on the f16 matrix cores (32x32x16): S^T = K q^T, O^T = V^T P^T, whose
// results both have a row of q per lane, so m, the sum and the rescaling of O
// need no exchange.  ks multiplies S, a key per register, by a DPP broadcast; vs goes
// into V's f16 tile (bf16, unless a tile's are too far apart for f16), or into p.  fp32
// takes q and p as two f16 limbs.
//
// Rows of a kv head's G query heads and of neighbouring tokens share a tile, so
// codes are read once per waves * 32 rows.  What bounds it then, at 2048 new tokens of
// 32 query heads over 8 kv heads, d = 128, behind 30,720 others (1065 GFLOP; 1234 to 1256 us on
// three GPUs, 848 to 863 TFLOP/s; a bf16 8192^3 library product runs 1208 to 1246): matrix
// cores are busy 38 % of the cycles, and the vector ALU's share (softmax, codes to f16: 312 M
// wave instructions) takes about as long, so the two have to overlap:
// * Four waves of 32 rows, one a SIMD, one after the other in program order: 1398 us, when
//   eight took 1197.
// * Eight waves in two phases, each SIMD's pair in opposite ones, a barrier after
//   each phase.  The matrix phase by itself takes 556 us, softmax 390, the two without
//   conversion and loads 882.
// * Tiles of 64 keys: V, K and the rows' state fit two waves a SIMD (256 registers).
// * Operands are read kAhead MFMAs early (4 and 8 for bf16: within 2 %).  Priorities
//   (s_setprio) gain nothing; reading scales before the matrix phase 1269 against 1211 us.
// Tiles of up to 32 rows take the narrow path, which is bound by bytes: 64 single
// tokens over 512 to 8192 keys 160 us (3.7 TB/s; by the wide path 403), one over
// 131,072 keys 62 us (4.5 TB/s; a copy moves 5.08 to 5.14).
#pragma once

#include <limits.h>
#include <math.h>

#include <type_traits>

#include "kvq_chunk.hpp"
#include "kvq_device.hpp"

namespace kvq {
namespace {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Waves of a workgroup, 32 query rows each.  Eight run in two phases a tile, which
// takes two waves a SIMD; where the state needs a SIMD's registers, four run.
// (64 sequences over 512 to 8192 keys, four with up to 511 new tokens, the others
// with one, bf16, d = 128: eight 446 us, four 798.)
constexpr int chunk_waves(int D, int limbs) { return D <= (limbs == 1 ? 128 : 96) ? 8 : 4; }
constexpr int kChunkCoherent = 16;  // buffer cache policy sc1: device-coherent
constexpr float kWeightTop = 15.0f;   // log2 of the largest f16 weight that is let grow,
constexpr float kWeightReset = 12.0f; // and of what a row's weights are set to when they pass it
constexpr float kKsMax = 0x1p80f;     // |k scale|s above overflow as scores of q scaled to 2^15
// |vs|s that are computed in fp32 throughout (chunk_row_f32); within them ratios do not
// matter.  Above: the weights of other tokens would leave fp32.  Below, 2^-10 (fp32: 2^-6)
// under the lowest exponent that m counts, f16 weights would lose bits.
constexpr float kVsMax = 0x1p60f;
template <int LIMBS>
constexpr float kVsMin = LIMBS == 1 ? 0x1p-90f : 0x1p-86f;
constexpr int kVsHigh = 60, kVsLow = -80;
// A row's m is set so that weights times |vs| are at most 2^15 and some of them 2^12, by
// s + (an exponent of vs): a tile's largest, unless some token's scale is 2^kSpreadBits below
// it.  Then each token counts its own, as a weight that m overrates has fewer bits: from
// 2^12 / 2^13 on they are enough for one f16 (off by 2^-25), from 2^12 / 2^6 for two.  In bf16's V
// tiles vs / 2^e is normal in f16 then, with e within +-kVfRange: 2^e in a weight's sum is
// within fp32 beside kVsHigh.
template <int LIMBS>
constexpr int kSpreadBits = LIMBS == 1 ? 12 : 5;
constexpr int kVfRange = 48;

// Dims that lane half h contracts in step n: steps 2 j and 2 j + 1 take the halves
// of one 16-byte piece, so that a row's codes can come straight from memory.
__device__ __forceinline__ constexpr int chunk_dim_of(int n, int h) { return 32 * (n >> 1) + 16 * h + 8 * (n & 1); }

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

// The largest of x[i] c + (lane i's y) and u.
template <int I = 0>
__device__ __forceinline__ float max_with_lanes(const f32x16& x, float c, float y, float u) {
    if constexpr (I < 16) {
        const float lane = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x150 + I, 0xF, 0xF, true));
        return max_with_lanes<I + 1>(x, c, y, fmaxf(u, fmaf(x[I], c, lane)));
    }
    return u;
}

// What a workgroup computes: query tile `tile` of sequence b and one kv head,
// over key blocks [k0, k1) of the tile's, as split `split` of nsplit.
struct ChunkItem {
    int b, tile, split, nsplit;
    int rec;   // first of the tile's records
    ChunkSeq seq;
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
// One workgroup a CU fits (LDS), so the slots are the 256 CUs: with 512, 512 tokens
// over 8192 keys take 168 us against 125.  A split is at least two blocks: with 4 and 8,
// five tokens over 1001 keys take 18.2 and 20.2 us against 17.2.
struct ChunkPlanLds {
    int part[8], best[8];
    int tiles[512], blocks[512];
    int found[8];
};
template <int W>
__device__ inline bool chunk_locate(const ChunkArgs& a, ChunkPlanLds& s, int r, ChunkItem& w) {
    constexpr int kChunkWaves = W, kChunkThreads = W * kWave;
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
    ChunkSeq first{};
    if (b0 < a.B) {
        first = chunk_seq(a, b0);
        chunk_counts(a, first, first_tiles, first_blocks);
        mine = first_tiles;
    }
    for (int i = 1; i < per; i++) {
        int tiles, blocks;
        counts(b0 + i, tiles, blocks);
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
                const ChunkSeq q = i > 0 ? chunk_seq(a, b0 + i) : first;
                s.found[5] = q.row0;
                s.found[6] = q.n;
                s.found[7] = q.len;
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
    w.seq.row0 = __builtin_amdgcn_readfirstlane(s.found[5]);
    w.seq.n = __builtin_amdgcn_readfirstlane(s.found[6]);
    w.seq.len = __builtin_amdgcn_readfirstlane(s.found[7]);
    return true;
}

// The root of what sums are multiplied by when their reference moves from m to mn: applied
// twice, as V scales of 2^-80 and 2^60 put more than fp32's range between two references,
// and l, which they are not in, has to come through.
__device__ __forceinline__ float half_step(float m, float mn) { return fast_exp2(0.5f * (m - mn)); }

// e with |vs| < 2^e, within [kVsLow, kVsHigh].  A token of value zero has the lowest there is:
// its score shall not raise m, under which the weights of others would lose bits.
__device__ __forceinline__ int scale_exponent(float v) {
    return v > 0.0f ? min(max(__builtin_amdgcn_frexp_expf(v), kVsLow), kVsHigh) : kVsLow;
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
__global__ __launch_bounds__(chunk_waves(D, LIMBS) * kWave) __attribute__((amdgpu_waves_per_eu(chunk_waves(D, LIMBS) / 4))) void
chunk_mfma(const ChunkArgs a) {
    constexpr int W = chunk_waves(D, LIMBS);
    constexpr bool kPhased = W == 8;
    constexpr int kChunkThreads = W * kWave;
    constexpr int kChunkRows = 32 * W;
    constexpr int KS = D + 8, VS = D + 16;     // LDS row strides in f16
    constexpr int NS = D / 16;                 // QK contraction steps
    constexpr int NB = D / 32;                 // output blocks
    constexpr int PPR = D / 8;                 // 8-code pieces of a row
    constexpr int NP = kChunkKeys * PPR / 256;  // a thread's: of K and of V, or (phased) of one of them
    static_assert(D % 32 == 0 && kChunkKeys * PPR % 256 == 0, "whole pieces");
    // A tile's scales, in the slot of its number.
    struct Scales {
        long long at[kChunkKeys];   // byte offsets of the pool rows
        float ks[kChunkKeys];
        float vs[kChunkKeys];
        unsigned vf[LIMBS == 1 ? kChunkKeys : 1];  // V's factor in the f16 tile, twice
        // x: |vs| <= 2^x; w: the tile's scales are far apart; y: log2 of the factor that the f16
        // tile's V lacks, z: its inverse (0 and 1 where vs goes into the weights)
        float4 v;
    };
    constexpr int kKTile = kChunkKeys * KS, kVTile = kChunkKeys * VS;
    __shared__ __align__(16) _Float16 s_buf[2 * (kKTile + kVTile)];
    auto s_k = [&](int tile) { return s_buf + (tile & 1) * kKTile; };
    auto s_v = [&](int tile) { return s_buf + 2 * kKTile + (tile & 1) * kVTile; };
    constexpr int kSlots = kPhased ? 8 : 4;
    __shared__ __align__(16) Scales s_scale[kSlots];
    static_assert(sizeof(ChunkPlanLds) <= sizeof(s_buf), "the plan's scratch lies where tiles come later");
    ChunkPlanLds& s_plan = *reinterpret_cast<ChunkPlanLds*>(s_buf);
    __shared__ int s_flag;

    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int c32 = lane & 31, h = lane >> 5, c16 = lane & 15;
    const int r = static_cast<int>(fastdiv(blockIdx.x, a.heads));
    const int kvh = static_cast<int>(blockIdx.x) - r * a.Hkv;
    ChunkItem w;
    if (!chunk_locate<W>(a, s_plan, r, w)) return;
    const ChunkSeq s = w.seq;
    const int i0 = w.tile * a.tile_tokens;                       // the tile's new tokens
    const int tokens = min(a.tile_tokens, s.n - i0);
    const int kend = chunk_keys(a, s, i0 + tokens - 1);          // keys that any of them attends
    const int nblocks = (kend + kChunkKeys - 1) / kChunkKeys;
    const int share = (nblocks + w.nsplit - 1) / w.nsplit;
    const int k0 = min(w.split * share, nblocks) * kChunkKeys;
    const int k1 = min(min((w.split + 1) * share, nblocks) * kChunkKeys, kend);
    const int tiles = k1 > k0 ? (k1 - k0 + kChunkKeys - 1) / kChunkKeys : 0;

    // Tiles of up to 32 rows are computed by all waves, each with the same rows and
    // keys of its own.
    const bool narrow = tokens * a.G <= 32;
    // This lane's query row: (token, head) = divmod(row, G).
    const int row = (narrow ? 0 : wave * 32) + c32;
    const int tok = static_cast<int>(fastdiv(row, a.group));
    const int head = kvh * a.G + row - tok * a.G;
    bool live = tok < tokens;
    const int keys = live ? chunk_keys(a, s, i0 + tok) : 0;
    const int64_t q_at = static_cast<int64_t>(s.row0 + i0 + tok) * a.q_stride + static_cast<int64_t>(head) * a.d;
    int wave_rows = min(max(tokens * a.G - (narrow ? 0 : wave * 32), 0), 32);  // live rows of this wave
    // Keys that every live row of the wave attends.
    const int first_tok = narrow ? 0 : static_cast<int>(fastdiv(wave * 32, a.group));
    const int keys_all = __builtin_amdgcn_readfirstlane(wave_rows > 0 ? chunk_keys(a, s, i0 + first_tok) : 0);

    // Pool row of key t0 + (t % 64) (past the end: the last key's again).
    const int32_t* table = a.pages.table + static_cast<size_t>(w.b) * a.pages.max_pages;
    auto page_of = [&](int tile) { return static_cast<int>(fastdiv(min(k0 + tile * kChunkKeys + lane, max(k1 - 1, 0)), a.page)); };
    auto pool_row = [&](int tile, int id) {
        const int key = min(k0 + tile * kChunkKeys + lane, max(k1 - 1, 0));
        const int page = static_cast<int>(fastdiv(key, a.page));
        id = min(max(id, 0), a.pages.num_pages - 1);
        return (static_cast<long long>(id) * a.Hkv + kvh) * a.pages.size + (key - page * a.pages.size);
    };

    // Phased: the first four waves fetch and convert K, the others V.
    const bool is_v = kPhased && wave >= 4;
    const int t256 = t & 255;
    int2 kraw[NP], vraw[kPhased ? 1 : NP];
    float ksr = 0.0f, vsr = 0.0f;
    float vmax = 0.0f, vmin = INFINITY, kmax = 0.0f;
    bool vbad = false;
    // Places of a tile's codes, read ahead of the loads that need them.
    long long at[NP];
    auto read_places = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NP; i++) at[i] = s_scale[tile & (kSlots - 1)].at[(i * 256 + t256) / PPR];
    };
    auto load_codes = [&](const int8_t* src, int2* raw) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int c = (i * 256 + t256) % PPR * 8;
            raw[i] = c < a.d ? *reinterpret_cast<const int2*>(src + at[i] + c) : make_int2(0, 0);
        }
    };
    // Codes become f16 here, once a workgroup: K exactly; V too for fp32, for bf16
    // times vs / 2^lv, rounded to f16.
    const h16x2 bias = {static_cast<_Float16>(kCodeBias), static_cast<_Float16>(kCodeBias)};
    auto store_k = [&](const int2* raw, int tile) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int piece = i * 256 + t256;
            const int kr = piece / PPR, c = (piece - kr * PPR) * 8;
            *reinterpret_cast<h16x8*>(s_k(tile) + kr * KS + c) =
                codes_to_f16(raw[i], [&](h16x2 x) { return x - bias; });
        }
    };
    auto store_v = [&](const int2* raw, int tile) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int piece = i * 256 + t256;
            const int kr = piece / PPR, c = (piece - kr * PPR) * 8;
            const h16x2 f = LIMBS == 1 ? __builtin_bit_cast(h16x2, s_scale[tile & (kSlots - 1)].vf[LIMBS == 1 ? kr : 0]) : bias;
            *reinterpret_cast<h16x8*>(s_v(tile) + kr * VS + c) =
                codes_to_f16(raw[i], [&](h16x2 x) { return LIMBS == 1 ? (x - bias) * f : x - bias; });
        }
    };
    auto load_tile = [&]() {
        if constexpr (kPhased) {
            load_codes(is_v ? a.v : a.k, kraw);
        } else {
            load_codes(a.k, kraw);
            load_codes(a.v, vraw);
        }
    };
    auto store_tile = [&](int tile) {
        if constexpr (kPhased) {
            if (is_v) store_v(kraw, tile);
            else store_k(kraw, tile);
        } else {
            store_k(kraw, tile);
            store_v(vraw, tile);
        }
    };
    // Wave 0 looks after rows and scales, a key a lane.
    auto load_scales = [&](int tile, long long row) {
        s_scale[tile & (kSlots - 1)].at[lane] = row * a.d;
        ksr = a.ks[row];
        vsr = a.vs[row];
        if (k0 + tile * kChunkKeys + lane >= k1) ksr = vsr = 0.0f;
    };
    auto store_scales = [&](int tile) {
        Scales& x = s_scale[tile & (kSlots - 1)];
        const float v = fabsf(vsr);
        kmax = fmaxf(kmax, fabsf(ksr));
        vbad |= !(v < INFINITY);
        vmax = fmaxf(vmax, v);
        if (v > 0.0f) vmin = fminf(vmin, v);
        // (bits of a float >= 0 order as integers; their top ones are the exponent)
        const int top = __builtin_amdgcn_readlane(wave_inclusive_max_nonneg(__float_as_int(v)), kWave - 1);
        const int e = (top >> 23) - 126;
        const bool in = k0 + tile * kChunkKeys + lane < k1;
        const bool spread = __builtin_amdgcn_ballot_w64(in && __float_as_int(v) < top - (kSpreadBits<LIMBS> << 23)) != 0 || e < -kVfRange || e > kVfRange;
        const float unit = spread ? 1.0f : __int_as_float((127 - e) << 23);  // 2^-e
        x.ks[lane] = ksr;
        x.vs[lane] = vsr;
        if (LIMBS == 1) {
            const _Float16 h = static_cast<_Float16>(spread ? 1.0f : vsr * unit);
            x.vf[LIMBS == 1 ? lane : 0] = __builtin_bit_cast(unsigned, h16x2{h, h});
        }
        const float lv = static_cast<float>(min(max(e, kVsLow), kVsHigh));
        if (lane == 0) x.v = make_float4(lv, spread ? 0.0f : lv, unit, spread ? 1.0f : 0.0f);
    };
    int far_id = 0;
    if (tiles > 0 && wave == 0 && !narrow) {
        const int id0 = table[page_of(0)], id1 = table[page_of(1)], id2 = table[page_of(2)];
        far_id = table[page_of(3)];
        load_scales(0, pool_row(0, id0));
        store_scales(0);
        load_scales(1, pool_row(1, id1));
        store_scales(1);
        load_scales(2, pool_row(2, id2));
    }

    // Narrow tiles: a block's codes and scales.
    constexpr int NK = D / 32;    // 16-byte pieces of K, and of V, a lane,
    constexpr int LPV = D / 16;   // lanes a row of V
    struct Block {
        int4 k[NK], v[NK];
        float ks, vs;
    };
    const int blocks = (k1 - k0 + 31) / 32;
    auto key_of = [&](int blk, int r) { return min(k0 + blk * 32 + r, max(k1 - 1, 0)); };
    auto id_of = [&](int blk) { return table[fastdiv(key_of(blk, c32), a.page)]; };
    auto piece = [&](const int8_t* src, long long at, int c) {  // codes c .. c + 15 of a row, zeros past its end
        int4 x = make_int4(0, 0, 0, 0);
        if (c + 16 <= a.d) {
            x = *reinterpret_cast<const int4*>(src + at + c);
        } else if (c < a.d) {
            const int2 y = *reinterpret_cast<const int2*>(src + at + c);
            x.x = y.x, x.y = y.y;
        }
        return x;
    };
    auto load = [&](Block& x, int blk, int id) __attribute__((always_inline)) {
        const int key = key_of(blk, c32);
        const int page = static_cast<int>(fastdiv(key, a.page));
        id = min(max(id, 0), a.pages.num_pages - 1);
        const long long mine = (static_cast<long long>(id) * a.Hkv + kvh) * a.pages.size + (key - page * a.pages.size);
#pragma unroll
        for (int j = 0; j < NK; j++) x.k[j] = piece(a.k, mine * a.d, 32 * j + 16 * h);
#pragma unroll
        for (int j = 0; j < NK; j++) {
            const int n = j * kWave + lane;
            x.v[j] = piece(a.v, __shfl(mine, n / LPV) * a.d, n % LPV * 16);
        }
        const bool in = k0 + blk * 32 + c32 < k1;
        x.ks = in ? a.ks[mine] : 0.0f;
        x.vs = in ? a.vs[mine] : 0.0f;
    };

    // q^T operands: lane has dims chunk_dim_of(n, h) + [0, 8) of its row, scaled to 2^15.
    h16x8 q[LIMBS][NS];
    float c_row;
    {
        float x[NS][8];
        float top = 0.0f;
        bool bad = false;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const int dim = chunk_dim_of(n, h);
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
                if (LIMBS == 2) q[LIMBS - 1][n][j] = static_cast<_Float16>(y - static_cast<float>(q[0][n][j]));
            }
    }

    f32x16 o[NB];
#pragma unroll
    for (int c = 0; c < NB; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[c][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // Keys of this lane's score registers: block 32 kb, register i: 32 kb + 8 (i / 4) + 4 h + i % 4.
    const int scale_at = 8 * (c16 >> 2) + 4 * h + (c16 & 3);
    f32x16 p[2];        // scores, then weights, of a tile
    h16x8 wt[LIMBS][4]; // weights as the operands of PV
    // PV of tile `pv` (O^T += V^T P^T) and QK of tile `qk` (S^T = K q^T), as one
    // sequence of A operands that are read kAhead of their MFMA: 8 keys of V (16 n +
    // 8 j + 4 h + [0, 4), j = 0, 1, are the lane's slots of step n) by two transposing
    // reads, 8 dims of K by one.
    auto matrix = [&](auto do_pv, auto do_qk, int pv, int qk) {
        constexpr int kPv = decltype(do_pv)::value ? 4 * NB : 0, kQk = decltype(do_qk)::value ? 2 * NS : 0;
        constexpr int kAll = kPv + kQk, kAhead = LIMBS == 1 ? 5 : 4;
        const _Float16* kp = s_k(qk) + c32 * KS;
        const _Float16* vp = s_v(pv) + (4 * h + (c16 >> 2)) * VS + 16 * ((lane >> 4) & 1) + 4 * (c16 & 3);
        auto read = [&](int n) {
            if (n < kPv) {
                const _Float16* x = vp + 16 * (n / NB) * VS + 32 * (n % NB);
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(const_cast<_Float16*>(x)));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(const_cast<_Float16*>(x + 8 * VS)));
                return __builtin_bit_cast(h16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
            n -= kPv;
            return *reinterpret_cast<const h16x8*>(kp + 32 * (n & 1) * KS + chunk_dim_of(n >> 1, h));
        };
        h16x8 x[kAll];
        f32x16 low[2];
#pragma unroll
        for (int n = 0; n < kAhead && n < kAll; n++) x[n] = read(n);
#pragma unroll
        for (int n = 0; n < kAll; n++) {
            if (n + kAhead < kAll) x[n + kAhead] = read(n + kAhead);
            __builtin_amdgcn_sched_barrier(0);
            if (n < kPv) {
                const int c = n % NB, step = n / NB;
                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[n], wt[0][step], o[c], 0, 0, 0);
                if (LIMBS == 2) o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[n], wt[LIMBS - 1][step], o[c], 0, 0, 0);
            } else {
                const int kb = (n - kPv) & 1, step = (n - kPv) >> 1;
                if (step == 0) {
#pragma unroll
                    for (int i = 0; i < 16; i++) p[kb][i] = low[kb][i] = 0.0f;
                }
                p[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[n], q[0][step], p[kb], 0, 0, 0);
                if (LIMBS == 2) low[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[n], q[LIMBS - 1][step], low[kb], 0, 0, 0);
                if (LIMBS == 2 && step == NS - 1) p[kb] += low[kb];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    auto softmax = [&](int tile) {
        const Scales& sc = s_scale[tile & (kSlots - 1)];
        const int t0 = k0 + tile * kChunkKeys;
#pragma unroll
        for (int kb = 0; kb < 2; kb++) times_lanes(p[kb], sc.ks[32 * kb + scale_at]);
        if (t0 + kChunkKeys > keys_all) {
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (t0 + 32 * kb + 8 * (i / 4) + 4 * h + i % 4 >= keys) p[kb][i] = -INFINITY;
        }
        float top = p[0][0];
#pragma unroll
        for (int i = 1; i < 32; i++) top = fmaxf(top, p[i / 16][i % 16]);
        const float4 sv = sc.v;
        const bool spread = __builtin_amdgcn_readfirstlane(__float_as_int(sv.w)) != 0;
        // m is a reference that weights pass by up to 2^kWeightTop: it moves, with the
        // state, only when some row's could pass by more.
        float u = fmaf(top, c_row, sv.x);
        if (__builtin_amdgcn_ballot_w64(u > m + kWeightTop) != 0) {
            if (spread) {
                u = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
                    u = max_with_lanes(p[kb], c_row, static_cast<float>(scale_exponent(fabsf(sc.vs[32 * kb + scale_at]))), u);
            }
            const float un = fmaxf(u, __shfl_xor(u, 32)) - kWeightReset;
            const float mn = un > m ? un : m;
            const float half = mn == -INFINITY ? 1.0f : half_step(m, mn);
            const float alpha = half * half;
            m = mn;
            l = l * half * half;
#pragma unroll
            for (int c = 0; c < NB; c++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[c][i] *= alpha;
        }
        const float ms = (m == -INFINITY ? 0.0f : m) - (LIMBS == 1 ? sv.y : 0.0f);
        auto weights = [&](auto vs_in_weights) __attribute__((always_inline)) {
            // Summed by themselves, so l rounds once a tile (2000 keys in fp32: error 2.0e-6 with a sum key by key).
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    p[kb][i] = fast_exp2(fmaf(p[kb][i], c_row, -ms));
                    part[i % 4] += p[kb][i];
                }
                if (decltype(vs_in_weights)::value) times_lanes(p[kb], sc.vs[32 * kb + scale_at]);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float y = p[kb][i];
                    // One value for both limbs: contracted into one of them, the product would be
                    // rounded once there and twice here, 2^-10 apart in one weight of some thousand.
                    if (LIMBS == 2) asm("" : "+v"(y));
                    const _Float16 hi = static_cast<_Float16>(y);
                    wt[0][2 * kb + i / 8][i % 8] = hi;
                    if (LIMBS == 2) wt[LIMBS - 1][2 * kb + i / 8][i % 8] = static_cast<_Float16>(y - static_cast<float>(hi));
                }
            }
            l = fmaf((part[0] + part[1]) + (part[2] + part[3]), LIMBS == 1 ? sv.z : 1.0f, l);
        };
        if (LIMBS == 2 || spread) weights(yes);
        else weights(no);
    };
    // Rows and scales ahead of tile i's: scales of tile i + 2 are stored, rows and
    // scales of tile i + 3 fetched into the slot of tile i - 1.
    auto ahead = [&](int i) {
        if (wave == 0 && i + 2 < tiles) {
            store_scales(i + 2);
            if (i + 3 < tiles) load_scales(i + 3, pool_row(i + 3, far_id));
            far_id = table[page_of(i + 4)];
        }
    };

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
    // Four sums of this lane's row, dims 32 (g / 4) + 8 (g % 4) + 4 h: the output, or a
    // record of a split.
    auto store_group = [&](int g, float4 x, float l_row) __attribute__((always_inline)) {
        const int dim = 32 * (g >> 2) + 8 * (g & 3) + 4 * h;
        if (!live) return;
        if (whole) {
            if (dim >= a.d) return;
            const float inv = 1.0f / l_row;
            if (keys > 0) put4(o_at + dim, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            else put4(o_at + dim, 0.0f, 0.0f, 0.0f, 0.0f);
        } else {
            const v4i_t y = {__float_as_int(x.x), __float_as_int(x.y), __float_as_int(x.z), __float_as_int(x.w)};
            __builtin_amdgcn_raw_buffer_store_b128(y, acc_rs, (row * D + dim) * 4, 0, kChunkCoherent);
        }
    };
    auto store_state = [&](float m_row, float l_row) __attribute__((always_inline)) {
        typedef int v2i_t __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(v2i_t{__float_as_int(m_row), __float_as_int(l_row)}, ml_rs, row * 8, 0, kChunkCoherent);
    };

    // Whether the scales that this wave knows of are not finite, or beyond what m and q scaled
    // to 2^15 cover.
    auto out_of_range = [&]() {
        const float top = wave_max(vmax), low = -wave_max(-vmin);
        return __builtin_amdgcn_ballot_w64(vbad || kmax > kKsMax) != 0 ||
               top > kVsMax || low < kVsMin<LIMBS>;
    };
    if (narrow) {
        // Each wave takes every W-th block of 32 keys, with nothing to wait for but its
        // own loads: K codes come as A operands straight from memory, V codes through a
        // part of LDS of the wave's own, read transposed.  The waves' states are joined
        // at the end.
        constexpr int VS8 = D + 16;   // LDS row stride of V codes
        static_assert(W * 32 * VS8 <= sizeof(s_buf) && W / 2 * 32 * D * 4 <= sizeof(s_buf), "LDS");
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
        int8_t* const vl = reinterpret_cast<int8_t*>(s_buf) + wave * 32 * VS8;
        const int scale_key = 8 * (c16 >> 2) + 4 * h + (c16 & 3);
        auto compute = [&](const Block& x, int blk) __attribute__((always_inline)) {
            wave_sync();
#pragma unroll
            for (int j = 0; j < NK; j++) {
                const int n = j * kWave + lane;
                *reinterpret_cast<int4*>(vl + n / LPV * VS8 + n % LPV * 16) = x.v[j];
            }
            const h16x2 bias = {static_cast<_Float16>(kCodeBias), static_cast<_Float16>(kCodeBias)};
            auto exact = [&](int2 w) { return codes_to_f16(w, [&](h16x2 y) { return y - bias; }); };
            f32x16 p, low;
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] = low[i] = 0.0f;
#pragma unroll
            for (int n = 0; n < NS; n++) {
                const int4 w = x.k[n / 2];
                const h16x8 y = exact(n & 1 ? make_int2(w.z, w.w) : make_int2(w.x, w.y));
                p = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, q[0][n], p, 0, 0, 0);
                if (LIMBS == 2) low = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, q[LIMBS - 1][n], low, 0, 0, 0);
            }
            if (LIMBS == 2) p += low;
            kmax = fmaxf(kmax, fabsf(x.ks));
            const float v = fabsf(x.vs);
            vbad |= !(v < INFINITY);
            vmax = fmaxf(vmax, v);
            if (v > 0.0f) vmin = fminf(vmin, v);
            const int vtop = __builtin_amdgcn_readlane(wave_inclusive_max_nonneg(__float_as_int(v)), kWave - 1);
            const int e = min(max((vtop >> 23) - 126, kVsLow), kVsHigh);
            times_lanes(p, __shfl(x.ks, scale_key));
            const int t0 = k0 + blk * 32;
            if (t0 + 32 > keys_all) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (t0 + 8 * (i / 4) + 4 * h + i % 4 >= keys) p[i] = -INFINITY;
            }
            float top = p[0];
#pragma unroll
            for (int i = 1; i < 16; i++) top = fmaxf(top, p[i]);
            float u = fmaf(top, c_row, static_cast<float>(e));
            if (__builtin_amdgcn_ballot_w64(u > m + kWeightTop) != 0) {
                // (tokens' scales too far apart)
                if (__builtin_amdgcn_ballot_w64(k0 + blk * 32 + c32 < k1 && __float_as_int(v) < vtop - (kSpreadBits<LIMBS> << 23)) != 0 || e == kVsLow)
                    u = max_with_lanes(p, c_row, __shfl(static_cast<float>(scale_exponent(v)), scale_key), -INFINITY);
                const float un = fmaxf(u, __shfl_xor(u, 32)) - kWeightReset;
                const float mn = un > m ? un : m;
                const float half = mn == -INFINITY ? 1.0f : half_step(m, mn);
                const float alpha = half * half;
                m = mn;
                l = l * half * half;
#pragma unroll
                for (int c = 0; c < NB; c++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[c][i] *= alpha;
            }
            const float ms = m == -INFINITY ? 0.0f : m;
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 16; i++) {
                p[i] = fast_exp2(fmaf(p[i], c_row, -ms));
                part[i % 4] += p[i];
            }
            l += (part[0] + part[1]) + (part[2] + part[3]);
            times_lanes(p, __shfl(x.vs, scale_key));
            h16x8 w[LIMBS][2];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float y = p[i];
                if (LIMBS == 2) asm("" : "+v"(y));  // one value for both limbs, as in softmax()
                const _Float16 hi = static_cast<_Float16>(y);
                w[0][i / 8][i % 8] = hi;
                if (LIMBS == 2) w[LIMBS - 1][i / 8][i % 8] = static_cast<_Float16>(y - static_cast<float>(hi));
            }
            wave_sync();
            // Lanes 2 r and 2 r + 1 of each 16 address row r of eight; lane i gets column i.
            const int r8 = c16 >> 1;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < NB; c++) {
                    const int8_t* src = vl + (16 * n + 8 * (r8 >> 2) + 4 * h + (r8 & 3)) * VS8 + 32 * c + 16 * ((lane >> 4) & 1) + 8 * (c16 & 1);
                    const i32x2 b = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(const_cast<int8_t*>(src)));
                    const h16x8 y = exact(make_int2(b[0], b[1]));
                    o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, w[0][n], o[c], 0, 0, 0);
                    if (LIMBS == 2) o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, w[LIMBS - 1][n], o[c], 0, 0, 0);
                }
        };
        __syncthreads();
        if (wave < blocks) {
            Block cur;
            load(cur, wave, id_of(wave));
            int next_id = id_of(wave + W);
            for (int b = wave; b < blocks; b += W) {
                Block next;
                load(next, b + W, next_id);  // (past the end: the last key's again)
                next_id = id_of(b + 2 * W);
                compute(cur, b);
                cur = next;
            }
        }
        // The waves' states: every wave finds the common reference, then the upper half
        // of the waves hands its sums to the lower one, and so on.
        __shared__ float s_ml[W][32][2];
        l += __shfl_xor(l, 32);
        if (h == 0) s_ml[wave][c32][0] = m, s_ml[wave][c32][1] = l;
        const bool odd = __builtin_amdgcn_ballot_w64(vbad || kmax > kKsMax) != 0;
        const float vtop = wave_max(vmax), vlow = -wave_max(-vmin);
        __shared__ float s_range[W][3];
        if (lane == 0) s_range[wave][0] = vtop, s_range[wave][1] = vlow, s_range[wave][2] = odd ? 1.0f : 0.0f;
        __syncthreads();
        // One wave's ranges for all.
        vmax = 0.0f, vmin = INFINITY, vbad = false;
#pragma unroll
        for (int i = 0; i < W; i++) {
            vmax = fmaxf(vmax, s_range[i][0]);
            vmin = fminf(vmin, s_range[i][1]);
            vbad |= s_range[i][2] != 0.0f;
        }
        // (rows that are computed again are not stored here)
        const bool stored = !out_of_range();
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) M = fmaxf(M, s_ml[i][c32][0]);
        const float Ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int i = 0; i < W; i++) {
            const float half = half_step(s_ml[i][c32][0], Ms);
            L = fmaf(s_ml[i][c32][1] * half, half, L);
        }
        const float own = half_step(m, Ms);
        const float f = own * own;
#pragma unroll
        for (int c = 0; c < NB; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[c][i] *= f;
        // Sums go through LDS in groups of 64 lanes' four values; wave g % W adds up
        // group g of all waves, and stores it.
        constexpr int kGroups = 4 * NB;
        constexpr int kRound = kGroups % 16 == 0 && W * 16 * 1024 <= sizeof(s_buf) ? 16 : kGroups % 8 == 0 && W * 8 * 1024 <= sizeof(s_buf) ? 8 : 4;
        static_assert(kGroups % kRound == 0 && W * kRound * 1024 <= sizeof(s_buf), "LDS");
        float4* const s_o = reinterpret_cast<float4*>(s_buf);
#pragma unroll
        for (int g0 = 0; g0 < kGroups; g0 += kRound) {
            __syncthreads();
#pragma unroll
            for (int g = g0; g < g0 + kRound; g++)
                s_o[(wave * kRound + g - g0) * kWave + lane] =
                    make_float4(o[g / 4][4 * (g % 4)], o[g / 4][4 * (g % 4) + 1], o[g / 4][4 * (g % 4) + 2], o[g / 4][4 * (g % 4) + 3]);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < (kRound + W - 1) / W; n++) {
                const int g = g0 + n * W + wave;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (n * W + wave < kRound) {
#pragma unroll
                    for (int i = 0; i < W; i++) {
                        const float4 y = s_o[(i * kRound + n * W + wave) * kWave + lane];
                        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                    }
                    if (stored) store_group(g, x, L);
                }
            }
        }
        if (stored && !whole && live && h == 0 && wave == 0) store_state(M, L);
        __syncthreads();
    } else {
        __syncthreads();
        if (tiles > 0) {
            read_places(0);
            load_tile();
            read_places(1);
            store_tile(0);
            if (tiles > 1) load_tile();
        }
        __syncthreads();
        if constexpr (kPhased) {
            // Two phases a tile, a barrier after each: matrix cores (PV of tile i - 1, QK
            // of tile i), then vector ALU (softmax of tile i, codes of tile i + 1).  The
            // V waves are one phase behind the K waves, so a SIMD's two waves, one of
            // each, use different units.  K waves are in phases 2 i and 2 i + 1, V waves
            // in 2 i + 1 and 2 i + 2.
            // * K of tile i + 1 is stored in phase 2 i + 1: its buffer's last readers (QK
            //   of i - 1) were V waves in phase 2 i - 1, its first is a K wave in 2 i + 2.
            // * V of tile i + 1 is stored in phase 2 i + 2: last read (PV of i - 1) by V
            //   waves in phase 2 i + 1, first by K waves in 2 i + 4.
            // * Wave 0 writes places of tile i + 3 and scales of tile i + 2 in phase 2 i, where
            //   V waves may still read those of tile i - 1: there are eight slots.
            // Every wave passes 2 tiles + 1 barriers.
            if (is_v) __syncthreads();
            auto stage = [&](int i) {
                if (i + 1 < tiles) {
                    store_tile(i + 1);
                    if (i + 2 < tiles) load_tile();
                }
                __syncthreads();
            };
            if (wave_rows > 0 && tiles > 0) {
                read_places(2);
                matrix(no, yes, 0, 0);
                ahead(0);
                __syncthreads();
                softmax(0);
                stage(0);
                for (int i = 1; i < tiles; i++) {
                    read_places(i + 2);
                    matrix(yes, yes, i - 1, i);
                    ahead(i);
                    __syncthreads();
                    softmax(i);
                    stage(i);
                }
                matrix(yes, no, tiles - 1, 0);
            } else {
                for (int i = 0; i < tiles; i++) {
                    read_places(i + 2);
                    ahead(i);
                    __syncthreads();
                    stage(i);
                }
            }
            if (!is_v) __syncthreads();
        } else {
            // Tile i + 1 becomes f16 in the buffer that was last read before the last
            // barrier; codes of tile i + 2 are on their way.
            for (int i = 0; i < tiles; i++) {
                if (i + 1 < tiles) {
                    read_places(i + 2);
                    store_tile(i + 1);
                    if (i + 2 < tiles) load_tile();
                }
                ahead(i);
                if (wave_rows > 0) {
                    matrix(no, yes, 0, i);
                    softmax(i);
                    matrix(yes, no, i, 0);
                }
                __syncthreads();
            }
        }
        __syncthreads();
    }

    // Then all its rows are computed in fp32, one after the other (one V scale of 1e-30 before 512
    // tokens over 8192 keys: 41 ms, not 0.12).
    if (wave == 0) {
        const bool bad = out_of_range();
        if (lane == 0) s_flag = bad;
    }
    __syncthreads();
    const bool exact = s_flag != 0;
    if (!exact) {
        if (live && !narrow) {
            l += __shfl_xor(l, 32);
#pragma unroll
            for (int g = 0; g < 4 * NB; g++)
                store_group(g, make_float4(o[g / 4][4 * (g % 4)], o[g / 4][4 * (g % 4) + 1], o[g / 4][4 * (g % 4) + 2], o[g / 4][4 * (g % 4) + 3]), l);
            if (!whole && h == 0) store_state(m, l);
        }
    } else {
        if (narrow && wave > 0) wave_rows = 0;
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
    // Records of eight splits are on their way together.
    constexpr int kDeep = 8;
    const unsigned step_acc = a.Hkv * kChunkRows * D * 4u, step_ml = a.Hkv * kChunkRows * 8u;
    const unsigned span = static_cast<unsigned>(w.nsplit - 1);
    const buf_rsrc accs = make_rsrc(a.part_acc + rec0 * kChunkRows * D, span * step_acc + kChunkRows * D * 4u);
    const buf_rsrc mls = make_rsrc(a.part_ml + rec0 * kChunkRows * 2, span * step_ml + kChunkRows * 8u);
    for (int jr = t / LPR; jr < live_rows; jr += RPP) {
        if (t / LPR >= RPP) break;
        const int dim = 4 * (t % LPR);
        float M = -INFINITY, L = 0.0f, A[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = 0; i0 < w.nsplit; i0 += kDeep) {
            typedef int v2i_t __attribute__((ext_vector_type(2)));
            v2i_t ml[kDeep];
            v4i_t acc[kDeep];
#pragma unroll
            for (int i = 0; i < kDeep; i++) {  // (past the last split: the last one's again, left out below)
                const int at = min(i0 + i, w.nsplit - 1);
                ml[i] = __builtin_bit_cast(v2i_t, __builtin_amdgcn_raw_buffer_load_b64(mls, jr * 8 + at * step_ml, 0, kChunkCoherent));
                acc[i] = __builtin_amdgcn_raw_buffer_load_b128(accs, (jr * D + dim) * 4 + at * step_acc, 0, kChunkCoherent);
            }
            float top = M;
#pragma unroll
            for (int i = 0; i < kDeep; i++) top = fmaxf(top, __int_as_float(ml[i].x));
            const float Ms = top == -INFINITY ? 0.0f : top;
            const float moved = half_step(M, Ms);
            const float alpha = moved * moved;
            M = top;
            L = L * moved * moved;
#pragma unroll
            for (int j = 0; j < 4; j++) A[j] *= alpha;
#pragma unroll
            for (int i = 0; i < kDeep; i++) {
                const float mi = __int_as_float(ml[i].x), li = __int_as_float(ml[i].y);
                if (i0 + i >= w.nsplit || (mi == -INFINITY && li == 0.0f)) continue;  // (or no key of this split)
                const float half = half_step(mi, Ms);
                const float f = half * half;
                L = fmaf(li * half, half, L);
#pragma unroll
                for (int j = 0; j < 4; j++) A[j] = fmaf(__int_as_float(acc[i][j]), f, A[j]);
            }
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
