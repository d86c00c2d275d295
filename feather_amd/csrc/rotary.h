// Sine and cosine of the rotary angles (decode_step.hip, rope_chunk.hip).
//
// On |r| <= pi/4, with z = r^2:  sin r ~ r + r z (S0 + S1 z + S2 z^2),  cos r ~ 1 - z/2 + z^2 (C0 + C1 z + C2 z^2).  The
// coefficients are minimax fits (Remez exchange in extended precision; the sine's relative, the cosine's absolute error),
// rounded to fp32 one after the other, the rest fitted again each time; tests/test_rotary_fit.py repeats the fit.  Without
// rounding they are off by 2^-27.9 (sine) and 2^-33.1 (cosine); evaluated in fp32 both are within 1.25 * 2^-24.
#pragma once

#include "common.h"

namespace feather {

constexpr float kSin0 = -1.666665524e-01f, kSin1 = 8.332189173e-03f, kSin2 = -1.951829181e-04f;
constexpr float kCos0 = 4.166664556e-02f, kCos1 = -1.388730132e-03f, kCos2 = 2.443067024e-05f;
// pi/2 = kHalfPi0 + kHalfPi1 + kHalfPi2 + 1.1e-23, each the fp32 nearest to what the ones before it leave
constexpr float kHalfPi0 = 1.570796371e+00f, kHalfPi1 = -4.371138829e-08f, kHalfPi2 = -1.715124510e-15f;

// of r + q * pi/2
__device__ __forceinline__ void sincos_quadrant(float r, int q, float &s, float &c) {
    const float z = r * r;
    const float sp = fmaf(r * z, fmaf(z, fmaf(z, kSin2, kSin1), kSin0), r);
    const float cp = fmaf(z, fmaf(z, fmaf(z, fmaf(z, kCos2, kCos1), kCos0), -0.5f), 1.0f);
    const float ss = (q & 1) ? cp : sp, cc = (q & 1) ? sp : cp;
    s = (q & 2) ? -ss : ss;
    c = ((q + 1) & 2) ? -cc : cc;
}

// of a non-negative angle below about 1e5 rad: the nearest multiple of pi/2 is taken off piece by piece with fused
// multiply-adds, which keep what cancels
__device__ __forceinline__ void sincos_small(float x, float &s, float &c) {
    const float k = rintf(x * 0.636619772f);
    sincos_quadrant(fmaf(-k, kHalfPi2, fmaf(-k, kHalfPi1, fmaf(-k, kHalfPi0, x))), (int)k, s, c);
}

}  // namespace feather
