// sigmoid and softplus in fp32, to a few units in the last place over the whole range.
#pragma once

#include "xlane.h"

namespace fw {

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1], with log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3: no
// logarithm near 1 is taken, so for x << 0 the result is e itself, with the relative error of e (|x| 2^-24, the rounding of
// x log2(e)).  2 atanh(s) / s as the polynomial of degree 4 in s^2 through the Chebyshev nodes of [0, 1/9]: off by less
// than 2^-26 of itself.
// sig = sigmoid(x) from the same e.
__device__ __forceinline__ float softplus_sig(float x, float &sig) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
    const float s = e * fast_rcp(2.f + e), s2 = s * s;
    float p = 0.2815778f;
    p = fmaf(p, s2, 0.27965158f);
    p = fmaf(p, s2, 0.40024596f);
    p = fmaf(p, s2, 0.6666632f);
    p = fmaf(p, s2, 2.0f);
    const float r = fast_rcp(1.f + e);
    sig = x >= 0.f ? r : e * r;
    return fmaf(s, p, fmaxf(x, 0.f));
}

// sigmoid(x) = 1 / (1 + exp(-x)); exp overflows to infinity where the result is zero.  For x < 0 the rounding of
// x log2(e) is not made good: a relative error of |x| 2^-24 in a result that is itself exp(x).
__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.f + __builtin_amdgcn_exp2f(-x * kLog2e)); }

}  // namespace fw
