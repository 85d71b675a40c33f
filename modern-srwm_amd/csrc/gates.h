// sigmoid and softplus in fp32, to a few units in the last place over the whole range.
#pragma once

#include "xlane.h"

namespace fw {

// exp(-|x|); the bound keeps an infinite x finite inside exp_2ulp and lets NaN pass (a comparison, not fminf)
__device__ __forceinline__ float exp_minus_abs(float x) {
    const float a = fabsf(x);
    return exp_2ulp(a > 1e30f ? -1e30f : -a);
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1], with log1p(e) = 2 atanh(e / (2 + e)): the argument of
// the series is at most 1/3, so the terms up to s^13 leave a relative error below 2^-24, and no logarithm near 1 is
// taken (for x << 0 the result is e itself, to full relative precision).  sig = sigmoid(x) from the same e.
__device__ __forceinline__ float softplus_sig(float x, float &sig) {
    const float e = exp_minus_abs(x);
    const float s = e * fast_rcp(2.f + e), s2 = s * s;
    float p = 1.f / 13.f;
    p = fmaf(p, s2, 1.f / 11.f);
    p = fmaf(p, s2, 1.f / 9.f);
    p = fmaf(p, s2, 1.f / 7.f);
    p = fmaf(p, s2, 1.f / 5.f);
    p = fmaf(p, s2, 1.f / 3.f);
    p = fmaf(p, s2, 1.f);
    const float r = fast_rcp(1.f + e);
    sig = x >= 0.f ? r : e * r;
    return fmaf(2.f * s, p, fmaxf(x, 0.f));
}
__device__ __forceinline__ float sigmoid(float x) {
    const float e = exp_minus_abs(x), r = fast_rcp(1.f + e);
    return x >= 0.f ? r : e * r;
}

}  // namespace fw
