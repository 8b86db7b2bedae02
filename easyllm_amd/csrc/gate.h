// What a gated MLP does with its gate: SiLU, either GELU, or ReLU, and the derivative.
#pragma once
#include "activation.h"

#include "../../include/ezl.h"

// ---- gate and up as they are kept for the backward pass ----
// In bf16 they would add as much again to the gradients' error as bf16 results have by themselves (relative error of dx and the weights' gradients 3.5e-3 instead of 2.4e-3, of
// which the results' own rounding is 1.7e-3), in fp32 twice the bytes.  So each keeps 12 bits of mantissa: the upper half of its fp32 bits, rounded to 12 bits, in a bf16 tensor, and the
// next four bits in half a byte of a third one, gate's in the lower half: five bytes the two, a sixteenth of the error left.  A value is put together again by one byte
// permutation, as many instructions as widening a bf16; taking it apart costs three more a value.
struct KeptParts {
    bf16_t *gate, *up;
    uint8_t* low;
};
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t kept_bits(float x) { return __float_as_uint(x) + 0x800u; }  // (infinities stay what they are)
// N / 2 words of upper halves, N / 4 of lower bits
template <int N>
__device__ __forceinline__ void keep(const float (&g)[N], const float (&u)[N], uint32_t (&gate)[N / 2], uint32_t (&up)[N / 2], uint32_t (&low)[N / 4]) {
    uint32_t a[N], b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        a[i] = kept_bits(g[i]);
        b[i] = kept_bits(u[i]);
    }
    const auto second_bytes = [](const uint32_t* x) {  // of four words
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(x[3], x[2], 0x0c0c0501u), __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0501u), 0x05040100u);
    };
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        gate[i / 2] = __builtin_amdgcn_perm(a[i + 1], a[i], 0x07060302u);
        up[i / 2] = __builtin_amdgcn_perm(b[i + 1], b[i], 0x07060302u);
    }
#pragma unroll
    for (int i = 0; i < N; i += 4) low[i / 4] = (second_bytes(a + i) >> 4 & 0x0f0f0f0fu) | (second_bytes(b + i) & 0xf0f0f0f0u);
}
template <int N>
__device__ __forceinline__ void kept_values(const uint32_t (&gate)[N / 2], const uint32_t (&up)[N / 2], const uint32_t (&low)[N / 4], float (&g)[N], float (&u)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t selector = (i & 1 ? 0x07060000u : 0x05040000u) | (i & 3) << 8 | 0x0c;  // (0x0c: a byte of zeros)
        g[i] = __uint_as_float(__builtin_amdgcn_perm(gate[i / 2], low[i / 4] << 4 & 0xf0f0f0f0u, selector));
        u[i] = __uint_as_float(__builtin_amdgcn_perm(up[i / 2], low[i / 4] & 0xf0f0f0f0u, selector));
    }
}
__device__ __forceinline__ void keep_one(float g, float u, const KeptParts& to, int64_t at) {
    const uint32_t a = kept_bits(g), b = kept_bits(u);
    to.gate[at] = __builtin_bit_cast(bf16_t, (uint16_t)(a >> 16));
    to.up[at] = __builtin_bit_cast(bf16_t, (uint16_t)(b >> 16));
    to.low[at] = (uint8_t)((a >> 12 & 15) | (b >> 8 & 0xf0));
}

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
