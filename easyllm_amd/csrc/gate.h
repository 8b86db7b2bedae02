// What a gated MLP does with its gate: SiLU, either GELU, or ReLU, and the derivative.
#pragma once
#include "activation.h"

#include "../../include/ezl.h"

// act(x) and its derivative.  (SiLU: 1 / (1 + 2^(-x log2 e)) with the bare exp2 / rcp instructions, 1 ulp each; it saturates at both ends.)
template <int ACT>
__device__ __forceinline__ float gate_value(float x) {
    if constexpr (ACT == EZL_GATE_SILU) return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
    else if constexpr (ACT == EZL_GATE_GELU) return activation(x, kActGelu);
    else if constexpr (ACT == EZL_GATE_GELU_TANH) return activation(x, kActGeluTanh);
    else return x <= 0.f ? 0.f : x;  // (NaN stays NaN)
}
template <int ACT>
__device__ __forceinline__ void gate_value_slope(float x, float& y, float& slope) {
    if constexpr (ACT == EZL_GATE_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
        y = x * s;
        slope = fmaf(y, 1.0f - s, s);
    } else if constexpr (ACT == EZL_GATE_GELU) {
        float d;
        const float c = normal_cdf(x, d);
        y = x * c;
        slope = fmaf(x * d, 0.39894228f, c);
    } else if constexpr (ACT == EZL_GATE_GELU_TANH) {
        const float s = tanh_cdf(x);
        y = x * s;
        slope = fmaf(x * s * (1.f - s), fmaf(fminf(x * x, 1e4f), 6.f * 0.79788456f * 0.044715f, 2.f * 0.79788456f), s);
    } else {
        y = x <= 0.f ? 0.f : x;
        slope = x <= 0.f ? 0.f : 1.f;
    }
}
