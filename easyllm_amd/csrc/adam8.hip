// AdamW with moments of 8 bits: 18 bytes a parameter instead of 30, 6 held instead of 12.
//
// A moment is a code of 8 bits a value and an exponent for every 256 values.  Codes are floating: the second moment has 5 exponent bits and 3 of mantissa
// below the block's largest value (31 binades: gradients apart by 2^15), the first a sign, 4 and 3.  What has to be watched is not the step of an eighth of a
// binade but the average: with beta2 = 0.999 a step moves v by a thousandth of itself, half a code is 3 - 6 %, so a moment rounded to the nearest code never moves at
// all.  Codes are therefore rounded up or down at random, by the share that is cut off: the moments' expected values are exactly those of 32 bits.  The random numbers come
// from a counter (seed, step, tensor, place), so that a step can be repeated.  A second moment above zero is never rounded to zero, which would divide by eps alone.
//
// Bits of an fp32 number grow with it, so the code of x is (bits of |x| 2^(K - e) + random) >> 20: the exponent e of the block moved to the top K of
// the code's range, values below the range denormal by themselves.  A product by a power of two is exact, so the codes are those of whoever computes the moments with the same roundings:
// products and sums below are rounded one by one (no fused multiply-add).
#include "common.h"
#include "dropout.h"  // (the generator)

#include "../../include/ezl.h"

#include <math.h>

namespace {

constexpr int kBlock8 = 256;         // values of one scale
constexpr int kChunk8 = 4096;        // elements a workgroup takes at a time
constexpr int kThreads8 = 256;
constexpr int kListMax8 = 40;        // tensors of a launch (its arguments are at most 4 KB)
constexpr int kTopM = 15, kTopV = 31;

struct MomentsList {
    float* master[kListMax8];
    uint8_t *m[kListMax8], *v[kListMax8], *ms[kListMax8], *vs[kListMax8];
    const float* g[kListMax8];
    bf16_t* param[kListMax8];  // entries may be null
    int64_t n[kListMax8];
    int first[kListMax8];      // launch-wide number of the tensor's first chunk
    uint32_t number[kListMax8];
    int count, chunks;
};
struct Adam8Args {
    float lr, beta1, beta2, one_beta1, one_beta2, eps, weight_decay, inv_bc1, inv_bc2;
    uint32_t key0, key1, step;
};

__device__ __forceinline__ int tensor_of8(const MomentsList& l, int chunk) {  // scalar bisection
    int lo = 0, hi = l.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// what `code` (BITS of magnitude, a sign above) stands for in a block of scale e
template <int BITS, int TOP>
__device__ __forceinline__ float value_of(uint32_t code, int e) {
    const float x = ldexpf(__uint_as_float((code & ((1u << BITS) - 1)) << 20), e - TOP);
    return e == 255 ? __builtin_nanf("") : BITS == 7 && (code & 128) ? -x : x;
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// the scale of a block whose largest magnitude has these bits (NaN is above infinity)
__device__ __forceinline__ int scale_of(uint32_t largest) {
    const uint32_t e = (largest + (1u << 20)) >> 23;
    return e > 255 ? 255 : (int)e;
}
template <int BITS, int TOP, uint32_t LEAST>
__device__ __forceinline__ uint32_t code_of(float x, uint32_t r, int e) {
    if (e == 255) return 0;
    uint32_t c = (__float_as_uint(ldexpf(fabsf(x), TOP - e)) + 16 * r + 8) >> 20;
    if (LEAST && x > 0.f && c < LEAST) c = LEAST;
    return c | (BITS == 7 && x < 0.f ? 128u : 0u);
}

__device__ __forceinline__ void adam8_one(float& p, float& m, float& v, float g, const Adam8Args& a) {
#pragma clang fp contract(off)
    m = m * a.beta1 + g * a.one_beta1;
    v = v * a.beta2 + g * g * a.one_beta2;
    const float update = (m * a.inv_bc1) / (sqrtf(v * a.inv_bc2) + a.eps);
    p = p - (update + p * a.weight_decay) * a.lr;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// A wave takes four blocks of 256, a lane four values of each.
__global__ __launch_bounds__(kThreads8) void adam8_kernel(const MomentsList l, const Adam8Args a, const float* __restrict__ norm_coef) {
    const float coef = norm_coef ? norm_coef[1] : 1.0f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int chunk = blockIdx.x; chunk < l.chunks; chunk += gridDim.x) {
        const int t = tensor_of8(l, chunk);
        const int64_t n = l.n[t], base = (int64_t)(chunk - l.first[t]) * kChunk8;
        for (int u = 0; u < 4; ++u) {
            const int64_t block = base / kBlock8 + wave * 4 + u, at = block * kBlock8 + lane * 4;
            if (block * kBlock8 >= n) break;
            const int64_t group = block / 2 * 64 + lane;
            const u32x4 w = philox_4x32_10((uint32_t)group, (uint32_t)(group >> 32), l.number[t], a.step, a.key0, a.key1);
            const int em = l.ms[t][block], ev = l.vs[t][block];
            float p[4], m[4], v[4];
            uint32_t most_m = 0, most_v = 0;
            for (int k = 0; k < 4; ++k) {
                p[k] = m[k] = v[k] = 0.f;
                if (at + k >= n) continue;
                p[k] = l.master[t][at + k];
                m[k] = value_of<7, kTopM>(l.m[t][at + k], em);
                v[k] = value_of<8, kTopV>(l.v[t][at + k], ev);
                adam8_one(p[k], m[k], v[k], l.g[t][at + k] * coef, a);
                most_m = max(most_m, magnitude(m[k]));
                most_v = max(most_v, magnitude(v[k]));
            }
            const int new_m = scale_of(wave_max_u32(most_m)), new_v = scale_of(wave_max_u32(most_v));
            for (int k = 0; k < 4; ++k) {
                if (at + k >= n) continue;
                const uint32_t word = block & 1 ? w[2 + k / 2] : w[k / 2], r = k & 1 ? word >> 16 : word & 0xffffu;
                l.master[t][at + k] = p[k];
                if (l.param[t]) l.param[t][at + k] = (bf16_t)p[k];
                l.m[t][at + k] = (uint8_t)code_of<7, kTopM, 0>(m[k], r, new_m);
                l.v[t][at + k] = (uint8_t)code_of<8, kTopV, 1>(v[k], r, new_v);
            }
            if (lane == 0) {
                l.ms[t][block] = (uint8_t)new_m;
                l.vs[t][block] = (uint8_t)new_v;
            }
        }
    }
}

// m and v as bf16 values (four significant bits: exact)
struct ValuesList {
    const uint8_t *m[kListMax8], *v[kListMax8], *ms[kListMax8], *vs[kListMax8];
    bf16_t *m_out[kListMax8], *v_out[kListMax8];
    int64_t n[kListMax8];
    int first[kListMax8];
    int count, chunks;
};
__global__ __launch_bounds__(kThreads8) void moments8_kernel(const ValuesList l) {
    for (int chunk = blockIdx.x; chunk < l.chunks; chunk += gridDim.x) {
        int t = 0;
        while (t + 1 < l.count && l.first[t + 1] <= chunk) ++t;
        const int64_t n = l.n[t], base = (int64_t)(chunk - l.first[t]) * kChunk8;
        for (int i = threadIdx.x; i < kChunk8 && base + i < n; i += kThreads8) {
            const int64_t at = base + i;
            l.m_out[t][at] = (bf16_t)value_of<7, kTopM>(l.m[t][at], l.ms[t][at / kBlock8]);
            l.v_out[t][at] = (bf16_t)value_of<8, kTopV>(l.v[t][at], l.vs[t][at / kBlock8]);
        }
    }
}

constexpr int kGrid8 = 2048;

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Whether two of a launch's tensors share memory that one of them writes: they are then updated in two launches, in order.
bool meet(const void* p, int64_t p_bytes, const void* q, int64_t q_bytes) {
    return p && q && (const char*)p < (const char*)q + q_bytes && (const char*)q < (const char*)p + p_bytes;
}

}  // namespace

extern "C" int ezl_adamw8_list(int count, const ezl_adam8_tensor* tensors, const ezl_adam8* how, const void* norm_coef, void* stream) {
    const char* name = "ezl_adamw8_list";
    EZL_REQUIRE(count >= 0 && how && (count == 0 || tensors), EZL_EINVAL, "%s: bad count or null argument", name);
    EZL_REQUIRE(how->step >= 1 && how->step < (1LL << 32), EZL_EINVAL, "%s: step counts from 1, below 2^32", name);
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        EZL_REQUIRE(t.n >= 0 && t.n < (1LL << 40) && (t.n == 0 || (t.master && t.exp_avg && t.exp_avg_sq && t.exp_avg_scale && t.exp_avg_sq_scale && t.grad)), EZL_EINVAL,
                    "%s: null pointer or bad size", name);
        EZL_REQUIRE(ezl_aligned16(t.master) && ezl_aligned16(t.grad) && aligned(t.param_bf16, 8) && aligned(t.exp_avg, 16) && aligned(t.exp_avg_sq, 16) &&
                        aligned(t.exp_avg_scale, 16) && aligned(t.exp_avg_sq_scale, 16),
                    EZL_EINVAL, "%s: the bf16 weight must be 8-byte aligned, the others 16-byte", name);
    }
    Adam8Args a;
    a.lr = (float)how->lr; a.beta1 = (float)how->beta1; a.beta2 = (float)how->beta2; a.eps = (float)how->eps; a.weight_decay = (float)how->weight_decay;
    a.one_beta1 = (float)(1.0 - how->beta1);
    a.one_beta2 = (float)(1.0 - how->beta2);
    a.inv_bc1 = how->bias_correction ? (float)(1.0 / (1.0 - pow(how->beta1, (double)how->step))) : 1.0f;
    a.inv_bc2 = how->bias_correction ? (float)(1.0 / (1.0 - pow(how->beta2, (double)how->step))) : 1.0f;
    a.key0 = (uint32_t)how->seed; a.key1 = (uint32_t)(how->seed >> 32); a.step = (uint32_t)how->step;
    MomentsList l;
    l.count = l.chunks = 0;
    const auto flush = [&]() {
        if (l.count) hipLaunchKernelGGL(adam8_kernel, dim3((unsigned)(l.chunks < kGrid8 ? l.chunks : kGrid8)), dim3(kThreads8), 0, (hipStream_t)stream, l, a, (const float*)norm_coef);
        l.count = l.chunks = 0;
    };
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const int64_t chunks = (t.n + kChunk8 - 1) / kChunk8, blocks = (t.n + kBlock8 - 1) / kBlock8;
        bool again = l.count == kListMax8 || l.chunks + chunks >= (1LL << 30);
        for (int j = 0; j < l.count && !again; ++j) {
            const int64_t other = (l.n[j] + kBlock8 - 1) / kBlock8;
            again = meet(t.master, t.n * 4, l.master[j], l.n[j] * 4) || meet(t.param_bf16, t.n * 2, l.param[j], l.n[j] * 2) || meet(t.exp_avg, t.n, l.m[j], l.n[j]) ||
                    meet(t.exp_avg_sq, t.n, l.v[j], l.n[j]) || meet(t.exp_avg_scale, blocks, l.ms[j], other) || meet(t.exp_avg_sq_scale, blocks, l.vs[j], other);
        }
        if (again) flush();
        const int s = l.count++;
        l.master[s] = (float*)t.master; l.m[s] = (uint8_t*)t.exp_avg; l.v[s] = (uint8_t*)t.exp_avg_sq; l.ms[s] = (uint8_t*)t.exp_avg_scale; l.vs[s] = (uint8_t*)t.exp_avg_sq_scale;
        l.g[s] = (const float*)t.grad; l.param[s] = (bf16_t*)t.param_bf16; l.n[s] = t.n; l.number[s] = t.number; l.first[s] = l.chunks;
        l.chunks += (int)chunks;
    }
    flush();
    EZL_LAUNCH_CHECK(name);
    return EZL_OK;
}

extern "C" int ezl_moments8_list(int count, const ezl_adam8_tensor* tensors, void* const* exp_avg_bf16, void* const* exp_avg_sq_bf16, void* stream) {
    const char* name = "ezl_moments8_list";
    EZL_REQUIRE(count >= 0 && (count == 0 || (tensors && exp_avg_bf16 && exp_avg_sq_bf16)), EZL_EINVAL, "%s: bad count or null argument", name);
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        EZL_REQUIRE(t.n >= 0 && t.n < (1LL << 40) && (t.n == 0 || (t.exp_avg && t.exp_avg_sq && t.exp_avg_scale && t.exp_avg_sq_scale && exp_avg_bf16[i] && exp_avg_sq_bf16[i])),
                    EZL_EINVAL, "%s: null pointer or bad size", name);
        EZL_REQUIRE(aligned(t.exp_avg, 16) && aligned(t.exp_avg_sq, 16) && ezl_aligned16(exp_avg_bf16[i]) && ezl_aligned16(exp_avg_sq_bf16[i]), EZL_EINVAL,
                    "%s: pointers must be 16-byte aligned", name);
    }
    ValuesList l;
    l.count = l.chunks = 0;
    const auto flush = [&]() {
        if (l.count) hipLaunchKernelGGL(moments8_kernel, dim3((unsigned)(l.chunks < kGrid8 ? l.chunks : kGrid8)), dim3(kThreads8), 0, (hipStream_t)stream, l);
        l.count = l.chunks = 0;
    };
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const int64_t chunks = (t.n + kChunk8 - 1) / kChunk8;
        if (l.count == kListMax8 || l.chunks + chunks >= (1LL << 30)) flush();
        const int s = l.count++;
        l.m[s] = (const uint8_t*)t.exp_avg; l.v[s] = (const uint8_t*)t.exp_avg_sq; l.ms[s] = (const uint8_t*)t.exp_avg_scale; l.vs[s] = (const uint8_t*)t.exp_avg_sq_scale;
        l.m_out[s] = (bf16_t*)exp_avg_bf16[i]; l.v_out[s] = (bf16_t*)exp_avg_sq_bf16[i]; l.n[s] = t.n; l.first[s] = l.chunks;
        l.chunks += (int)chunks;
    }
    flush();
    EZL_LAUNCH_CHECK(name);
    return EZL_OK;
}
