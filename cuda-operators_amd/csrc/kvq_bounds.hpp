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

}  // namespace kvq
