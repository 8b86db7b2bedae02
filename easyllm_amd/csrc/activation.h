// GELU and its derivative, exact (x Phi(x), Phi the normal distribution function) and with the tanh of the logistic form.
#pragma once
#include "common.h"

constexpr int kActNone = 0, kActGelu = 1, kActGeluTanh = 2;

// Phi(-|x|) = t P(t) exp(-x^2 / 2), t = 1 / (1 + 0.44 |x| / sqrt 2), P of degree 5: a least-squares fit, reweighted to the smallest largest relative
// error, of erfcx(z) / 2 over t(z), z = 0 .. 10; 5.2e-6 off (a bf16 result is off by up to 2^-8).  The negative branch has no
// cancellation, unlike 1 + erf.  `density` gets exp(-x^2 / 2).
__device__ __forceinline__ float normal_cdf(float x, float& density) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.31112698f, fabsf(x), 1.f));
    density = __builtin_amdgcn_exp2f(x * x * -0.72134752f);
    float p = fmaf(-0.07305321f, t, 0.17532738f);
    p = fmaf(p, t, 0.02036425f);
    p = fmaf(p, t, 0.13179392f);
    p = fmaf(p, t, 0.12128457f);
    p = fmaf(p, t, 0.12428053f);
    const float q = p * t * density;
    return x > 0.f ? 1.f - q : q;
}
// (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
__device__ __forceinline__ float tanh_cdf(float x) {
    const float u2 = x * fmaf(x * x, -2.f * 0.79788456f * 0.044715f * 1.44269504f, -2.f * 0.79788456f * 1.44269504f);
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u2));
}

__device__ __forceinline__ float activation(float x, int act) {
    if (act == kActGelu) {
        float d;
        return x * normal_cdf(x, d);
    }
    if (act == kActGeluTanh) return x * tanh_cdf(x);
    return x;
}
__device__ __forceinline__ float activation_slope(float x, int act) {
    if (act == kActGelu) {
        float d;
        const float c = normal_cdf(x, d);
        return fmaf(x * d, 0.39894228f, c);
    }
    if (act == kActGeluTanh) {
        const float s = tanh_cdf(x);
        // (beyond |x| = 100 s (1 - s) is zero; the square would overflow)
        return fmaf(x * s * (1.f - s), fmaf(fminf(x * x, 1e4f), 6.f * 0.79788456f * 0.044715f, 2.f * 0.79788456f), s);
    }
    return 1.f;
}
