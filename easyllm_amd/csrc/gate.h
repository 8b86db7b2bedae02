// What a gated MLP does with its gate: SiLU, either GELU, or ReLU, and the derivative.
#pragma once
#include "activation.h"

#include "../../include/ezl.h"

// ---- gate and up as they are kept for the backward pass ----
// In bf16 they would add as much again to the gradients' error as bf16 results have by themselves (relative error of dx and the weights' gradients 3.5e-3 instead of 2.4e-3, of
// which the results' own rounding is 1.7e-3), in fp32 twice the bytes.  So each keeps 12 bits of mantissa: the upper half of its fp32 bits, rounded to 12 bits, and the
// next four bits in half a byte for both, gate's in the lower half: five bytes the two, a sixteenth of the error left.  A value is put together again by one byte
// permutation, as many instructions as widening a bf16; taking it apart costs three more a value.
// They lie in blocks of 16 rows and 32 columns, as an epilogue's wave holds them: 64 times gate's eight upper halves, the same of up's, 64 times the eight bytes of lower bits.  A wave's stores
// and loads are whole lines then, in one place instead of sixteen rows of three matrices: keeping costs 4096 x 4096 x 11008 tokens x h x f 33 us instead of 61, 8192 x 128 x 8192 66 instead of
// 110; the way back takes 357 instead of 373 and 219 instead of 228.  The last blocks of rows and columns are whole ones, too.
constexpr int kKeptRows = 16, kKeptCols = 32, kKeptBlock = 2560, kKeptUp = 1024, kKeptLow = 2048;  // (the last three in bytes)
struct Kept {
    char* p;     // null: nothing is kept
    int blocks;  // side by side
    __host__ __device__ __forceinline__ Kept at(int64_t row, int64_t col) const {  // of a block's first row and column
        return {p ? p + (row / kKeptRows * blocks + col / kKeptCols) * kKeptBlock : nullptr, blocks};
    }
};
inline Kept kept_of(const void* p, int64_t f) { return {(char*)p, (int)((f + kKeptCols - 1) / kKeptCols)}; }
// where the eight columns from col / 8 * 8 of a row lie: their upper halves (up's kKeptUp further), their lower bits
struct KeptPlace {
    char *upper, *low;
};
__device__ __forceinline__ KeptPlace kept_place(const Kept& k, int64_t row, int col) {
    char* const block = k.p + (row / kKeptRows * k.blocks + col / kKeptCols) * kKeptBlock;
    const int slot = ((col >> 4 & 1) | (col >> 2 & 2)) * 16 + (int)(row % kKeptRows);
    return {block + slot * 16, block + kKeptLow + slot * 8};
}
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
__device__ __forceinline__ void keep_one(float g, float u, const Kept& to, int64_t row, int col) {
    const uint32_t a = kept_bits(g), b = kept_bits(u);
    const KeptPlace at = kept_place(to, row, col);
    reinterpret_cast<uint16_t*>(at.upper)[col & 7] = (uint16_t)(a >> 16);
    reinterpret_cast<uint16_t*>(at.upper + kKeptUp)[col & 7] = (uint16_t)(b >> 16);
    at.low[col & 7] = (char)((a >> 12 & 15) | (b >> 8 & 0xf0));
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
