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
// 16 loads at a time; a token past the page's last one repeats that one, which
// changes no maximum.  The ratios are divided once a token (lane j of a group
// that of token j) and handed round.  What bounds it is the chain of loads (the
// page's id, its scales, its keys) of waves that each read a few KB: 8 bytes a
// lane leave 16 results instead of 32 in its registers, so that twice as many
// waves are there to wait.
// live: this lane's page exists (others run along on another page and store nothing).
template <int LPT>
__device__ inline void bounds_wave(const BoundsArgs& a, int groups, bool live, int b, int pi, int h, int tokens) {
    constexpr int NT = 16;                            // tokens a group takes at a time
    constexpr int NS = NT / LPT > 1 ? NT / LPT : 1;  // scales a lane holds of them
    typedef int v2i_t __attribute__((ext_vector_type(2)));
    const int lane = threadIdx.x & (kWave - 1);
    const int ds = lane % LPT;
    const int g = lane / LPT % groups;
    const int d = a.d;
    const int off = min(ds * 8, d - 8);
    const int id = a.pages.table[static_cast<size_t>(b) * a.pages.max_pages + pi];
    const size_t unit = static_cast<size_t>(min(max(id, 0), a.pages.num_pages - 1)) * a.Hkv + h;
    const int8_t* k = a.k + unit * a.pages.size * d + off;
    const float* s = a.ks + unit * a.pages.size;
    const int passes = (a.pages.size + groups * NT - 1) / (groups * NT);  // the same in every lane

    auto scales = [&](int pass, float (&x)[NS]) {
#pragma unroll
        for (int j = 0; j < NS; j++) x[j] = s[min((pass * NT + (ds + j * LPT) % NT) * groups + g, tokens - 1)];
    };
    v2i_t raw[NT];
    auto load = [&](int pass) {
#pragma unroll
        for (int u = 0; u < NT; u++) {
            const int t = min((pass * NT + u) * groups + g, tokens - 1);
            raw[u] = __builtin_nontemporal_load(reinterpret_cast<const v2i_t*>(k + static_cast<size_t>(t) * d));
        }
    };
    float sc[NS];
    scales(0, sc);
    load(0);  // on its way while the scales are reduced
    float S = 0.0f;
    for (int pass = 0; pass < passes; pass++) {
        if (pass > 0) scales(pass, sc);
#pragma unroll
        for (int j = 0; j < NS; j++) S = max_or_nan(S, fabsf(sc[j]));
    }
    for (int o = 1; o < LPT * groups; o <<= 1) S = max_or_nan(S, __shfl_xor(S, o));
    const bool fine = S < INFINITY;

    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; i++) hi[i] = -INFINITY, lo[i] = INFINITY;
    if (passes > 1) scales(0, sc);
    for (int pass = 0; pass < passes; pass++) {
        if (pass > 0) {
            scales(pass, sc);
            load(pass);
        }
        float r[NS];
#pragma unroll
        for (int j = 0; j < NS; j++) r[j] = bound_ratio(sc[j], S);
        // Keeps the conversions here: moved up into the two blocks that load raw,
        // they would hold every token's 8 products at once (230 registers).
#pragma unroll
        for (int u = 0; u < NT; u++) asm volatile("" : "+v"(raw[u]));
#pragma unroll
        for (int u = 0; u < NT; u += 2) {
            const float r0 = __shfl(r[u / LPT], (lane & ~(LPT - 1)) + u % LPT);
            const float r1 = __shfl(r[(u + 1) / LPT], (lane & ~(LPT - 1)) + (u + 1) % LPT);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x0 = sbyte(raw[u][i / 4], i & 3) * r0;
                const float x1 = sbyte(raw[u + 1][i / 4], i & 3) * r1;
                hi[i] = fmaxf(fmaxf(x0, x1), hi[i]);
                lo[i] = fminf(fminf(x0, x1), lo[i]);
            }
        }
    }
    // (high, -low) as two 16-bit codes, so one packed maximum joins the groups' both.
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 m[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        m[i] = fine ? s16x2{static_cast<short>(bound_code(ceilf(hi[i]))), static_cast<short>(-bound_code(floorf(lo[i])))}
                    : s16x2{127, 127};
    for (int o = LPT; o < LPT * groups; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int x = __shfl_xor(__builtin_bit_cast(int, m[i]), o);
            m[i] = __builtin_elementwise_max(m[i], __builtin_bit_cast(s16x2, x));
        }
    }
    if (!live || g != 0) return;
    if (ds * 8 < d) {
        int8_t* o = a.bounds + unit * 2 * d + off;
        *reinterpret_cast<int2*>(o) = make_int2(pack4(m[0].x, m[1].x, m[2].x, m[3].x), pack4(m[4].x, m[5].x, m[6].x, m[7].x));
        *reinterpret_cast<int2*>(o + d) =
            make_int2(pack4(-m[0].y, -m[1].y, -m[2].y, -m[3].y), pack4(-m[4].y, -m[5].y, -m[6].y, -m[7].y));
    }
    if (ds == 0) a.scale[unit] = fine ? S : INFINITY;
}

// Lanes a token of bounds_wave takes, and groups a page that leave a group 16 tokens or fewer where it can.
constexpr int bounds_lanes(int d) { return d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32; }
__host__ __device__ inline int bounds_groups(int page_size, int lanes) {
    int g = 1;
    while (g < kWave / lanes && g * 16 < page_size) g *= 2;
    return g;
}

}  // namespace kvq
