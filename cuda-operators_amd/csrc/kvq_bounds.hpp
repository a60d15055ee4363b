// kvq_bounds.hpp -- key bounds of one page, shared by the bounds kernel and the
// page selection (which renews those of a page that has just become whole).
//
// With s_t the scales and k_t the codes of the page's tokens, S = max |s_t| and
// r_t = RN(s_t / S): per dim, high = ceil(max_t RN(k_t r_t)), low =
// floor(min_t RN(k_t r_t)).  |k_t| <= 128 and |r_t| <= 1, so both fit int8 once
// clamped to 127 (a code of -128, which no quantiser here writes, would give -128:
// clamped to -127 it may lie above the true bound by one step).
#pragma once

#include <math.h>

#include "kvq_device.hpp"
#include "kvq_pages.hpp"

namespace kvq {

__device__ __forceinline__ int bound_code(float x) { return static_cast<int>(fminf(fmaxf(x, -127.0f), 127.0f)); }

// Ratio s / S of a scale; S finite.
__device__ __forceinline__ float bound_ratio(float s, float S) { return S > 0.0f ? s / S : 0.0f; }

// Page entry pi of sequence b, kv head h, its first `tokens` >= 1 tokens: one
// wave, an element a load.
__device__ inline void bounds_generic(const BoundsArgs& a, int b, int pi, int h, int tokens, int lane) {
    const int id = a.pages.table[static_cast<size_t>(b) * a.pages.max_pages + pi];
    const size_t unit = static_cast<size_t>(min(max(id, 0), a.pages.num_pages - 1)) * a.Hkv + h;
    const int8_t* k = a.k + unit * a.pages.size * a.d;
    const float* s = a.ks + unit * a.pages.size;
    float S = 0.0f;
    for (int t = lane; t < tokens; t += kWave) S = max_or_nan(S, fabsf(s[t]));
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) S = max_or_nan(S, __shfl_xor(S, off));
    const bool fine = S < INFINITY;  // neither infinite nor NaN
    int8_t* o = a.bounds + unit * 2 * a.d;
    for (int i = lane; i < a.d; i += kWave) {
        float hi = -INFINITY, lo = INFINITY;
        for (int t = 0; t < tokens && fine; t++) {
            const float x = static_cast<float>(k[static_cast<size_t>(t) * a.d + i]) * bound_ratio(s[t], S);
            hi = fmaxf(hi, x);
            lo = fminf(lo, x);
        }
        o[i] = static_cast<int8_t>(fine ? bound_code(ceilf(hi)) : 127);
        o[a.d + i] = static_cast<int8_t>(fine ? bound_code(floorf(lo)) : -127);
    }
    if (lane == 0) a.scale[unit] = fine ? S : INFINITY;
}

// Tuned: LPT lanes a token with 8 bytes of its row each (LPT: d / 8 rounded up to
// a power of two; the lanes past the row's end read its last piece again), groups
// of LPT lanes a page (a power of two up to 64 / LPT), so a wave holds
// 64 / (LPT * groups) pages.  Group g of a page takes tokens g, g + groups, ..,
// 16 loads at a time (one pass over pages of up to 16 * groups tokens); a token past the page's last one repeats that one, which
// changes no maximum.  The ratios are divided once a token (lane j of a group
// that of token j) and handed round.  What bounds it is the chain of loads (the
// page's id, its scales, its keys) of waves that each read a few KB: 8 bytes a
// lane leave 16 results instead of 32 in its registers, so that twice as many
// waves are there to wait.
enum class Pages {
    Several,  // several pages a wave, each in one pass
    One,      // a page a wave, in one pass
    Passes,   // a page a wave, in any number of passes
};
template <int LPT, Pages MODE>
struct BoundsWave {
    static constexpr int NT = 16;                            // tokens a group takes in a pass
    static constexpr int NS = NT / LPT > 1 ? NT / LPT : 1;  // scales a lane holds of them
    typedef int v2i_t __attribute__((ext_vector_type(2)));

    // The first pass of one (page, kv head), on its way.
    struct Piece {
        v2i_t raw[NT];
        float sc[NS];
        size_t unit;  // page id * Hkv + kv head
        int tokens;
    };

    const BoundsArgs& a;
    const int groups, ds, g, off, passes;

    __device__ __forceinline__ BoundsWave(const BoundsArgs& args, int groups)
        : a(args),
          groups(groups),
          ds((threadIdx.x & (kWave - 1)) % LPT),
          g((threadIdx.x & (kWave - 1)) / LPT % groups),
          off(min(ds * 8, args.d - 8)),
          passes(MODE == Pages::Passes ? (args.pages.size + groups * NT - 1) / (groups * NT) : 1) {}

    __device__ __forceinline__ void scales(const Piece& p, int pass, float (&x)[NS]) const {
#pragma unroll
        for (int j = 0; j < NS; j++)
            x[j] = a.ks[p.unit * a.pages.size + min((pass * NT + (ds + j * LPT) % NT) * groups + g, p.tokens - 1)];
    }
    __device__ __forceinline__ void rows(const Piece& p, int pass, v2i_t (&x)[NT]) const {
        const int8_t* k = a.k + p.unit * a.pages.size * a.d;
        const int step = groups * a.d, last = (p.tokens - 1) * a.d + off;  // below 2^30 (the launcher sees to it)
        const int first = g * a.d + off + pass * NT * step;
#pragma unroll
        for (int u = 0; u < NT; u++)
            x[u] = __builtin_nontemporal_load(reinterpret_cast<const v2i_t*>(k + static_cast<unsigned>(min(first + u * step, last))));
    }
    // id: the page's entry of the block table; tokens: those of it that count, >= 1.
    __device__ __forceinline__ void fetch(Piece& p, int id, int h, int tokens) const {
        if constexpr (MODE != Pages::Several) id = __builtin_amdgcn_readfirstlane(id);
        p.unit = static_cast<size_t>(min(max(id, 0), a.pages.num_pages - 1)) * a.Hkv + h;
        p.tokens = tokens;
        scales(p, 0, p.sc);
        rows(p, 0, p.raw);
    }

    // live: this lane's page exists (others run along on another page and store nothing).
    __device__ __forceinline__ void finish(Piece& p, bool live) const {
        const int lane = threadIdx.x & (kWave - 1);
        float S = 0.0f;
#pragma unroll
        for (int j = 0; j < NS; j++) S = max_or_nan(S, fabsf(p.sc[j]));
        for (int pass = 1; pass < passes; pass++) {
            float x[NS];
            scales(p, pass, x);
#pragma unroll
            for (int j = 0; j < NS; j++) S = max_or_nan(S, fabsf(x[j]));
        }
        for (int o = 1; o < LPT * groups; o <<= 1) S = max_or_nan(S, __shfl_xor(S, o));
        const bool fine = S < INFINITY;

        float hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; i++) hi[i] = -INFINITY, lo[i] = INFINITY;
        for (int pass = 0; pass < passes; pass++) {
            if (pass > 0) {
                scales(p, pass, p.sc);
                rows(p, pass, p.raw);
            }
            float r[NS];
#pragma unroll
            for (int j = 0; j < NS; j++) r[j] = bound_ratio(p.sc[j], S);
            // Keeps the conversions here: moved up into the blocks that load raw,
            // they would hold every token's 8 products at once (230 registers).
            if constexpr (MODE == Pages::Passes) {
#pragma unroll
                for (int u = 0; u < NT; u++) asm volatile("" : "+v"(p.raw[u]));
            }
            // RN(k r) = fma(k + 128, r, -128 r), where -128 r is exact: unsigned
            // bytes and fused products run at 0.7 of the time of signed ones
            // (v_cvt_f32_ubyte and v_fma 7.2 cycles an element with its maximum,
            // v_cvt_f32_i32 with a byte select and v_mul 10.3).
#pragma unroll
            for (int u = 0; u < NT; u += 2) {
                const float r0 = __shfl(r[u / LPT], (lane & ~(LPT - 1)) + u % LPT);
                const float r1 = __shfl(r[(u + 1) / LPT], (lane & ~(LPT - 1)) + (u + 1) % LPT);
                const float c0 = -128.0f * r0, c1 = -128.0f * r1;
                const v2i_t flip = {static_cast<int>(0x80808080u), static_cast<int>(0x80808080u)};
                const v2i_t w0 = p.raw[u] ^ flip, w1 = p.raw[u + 1] ^ flip;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x0 = __builtin_fmaf(static_cast<float>(static_cast<uint8_t>(static_cast<unsigned>(w0[i / 4]) >> (8 * (i & 3)))), r0, c0);
                    const float x1 = __builtin_fmaf(static_cast<float>(static_cast<uint8_t>(static_cast<unsigned>(w1[i / 4]) >> (8 * (i & 3)))), r1, c1);
                    hi[i] = fmaxf(fmaxf(x0, x1), hi[i]);
                    lo[i] = fminf(fminf(x0, x1), lo[i]);
                }
                __builtin_amdgcn_sched_barrier(0);  // a pair of tokens at a time, for the same reason
            }
        }
        // (high, -low) as two 16-bit codes, so one packed maximum joins the groups' both.
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        s16x2 m[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            m[i] = s16x2{static_cast<short>(bound_code(ceilf(hi[i]))), static_cast<short>(-bound_code(floorf(lo[i])))};
        for (int o = LPT; o < LPT * groups; o <<= 1) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int x = __shfl_xor(__builtin_bit_cast(int, m[i]), o);
                m[i] = __builtin_elementwise_max(m[i], __builtin_bit_cast(s16x2, x));
            }
        }
        if (!live || g != 0) return;
        if (!fine) {
#pragma unroll
            for (int i = 0; i < 8; i++) m[i] = s16x2{127, 127};
        }
        if (ds * 8 < a.d) {
            int8_t* o = a.bounds + p.unit * 2 * a.d + off;
            *reinterpret_cast<int2*>(o) = make_int2(pack4(m[0].x, m[1].x, m[2].x, m[3].x), pack4(m[4].x, m[5].x, m[6].x, m[7].x));
            *reinterpret_cast<int2*>(o + a.d) =
                make_int2(pack4(-m[0].y, -m[1].y, -m[2].y, -m[3].y), pack4(-m[4].y, -m[5].y, -m[6].y, -m[7].y));
        }
        if (ds == 0) a.scale[p.unit] = fine ? S : INFINITY;
    }
};

// Lanes a token takes, and groups a page that leave a group 16 tokens or fewer where it can.
constexpr int bounds_lanes(int d) { return d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32; }
__host__ __device__ inline int bounds_groups(int page_size, int lanes) {
    int g = 1;
    while (g < kWave / lanes && g * 16 < page_size) g *= 2;
    return g;
}

}  // namespace kvq
