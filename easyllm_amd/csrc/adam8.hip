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

#include <type_traits>

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
    const float x = __builtin_amdgcn_ldexpf(__uint_as_float((code & ((1u << BITS) - 1)) << 20), e - TOP);
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
    uint32_t c = (__float_as_uint(__builtin_amdgcn_ldexpf(fabsf(x), TOP - e)) + 16 * r + 8) >> 20;
    if (LEAST && x > 0.f && c < LEAST) c = LEAST;
    return c | (BITS == 7 ? __float_as_uint(x) >> 31 << 7 : 0u);
}

// The root and the quotient correctly rounded, as all else: the weights are their definition's bit by bit.  (25 instructions a value more than the bare ones, which are off by 1 ulp each; 202
// million parameters take 665 us either way but for 3: the memory binds.)
__device__ __forceinline__ void adam8_one(float& p, float& m, float& v, float g, float beta1, float beta2, const Adam8Args& a) {
#pragma clang fp contract(off)
    m = m * beta1 + g * a.one_beta1;
    v = v * beta2 + g * g * a.one_beta2;
    const float update = (m * a.inv_bc1) / (sqrtf(v * a.inv_bc2) + a.eps);
    p = p - (update + p * a.weight_decay) * a.lr;
}

// largest of a wave's values, in a scalar register: rows of 16 lanes, then the rows
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    const auto up = [&](auto CTRL) { v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(CTRL)::value, 0xf, 0xf, false)); };
    up(std::integral_constant<int, 0x111>{});  // row_shr 1, 2, 4, 8
    up(std::integral_constant<int, 0x112>{});
    up(std::integral_constant<int, 0x114>{});
    up(std::integral_constant<int, 0x118>{});
    up(std::integral_constant<int, 0x142>{});  // row_bcast 15, 31
    up(std::integral_constant<int, 0x143>{});
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// where a wave's four blocks of a tensor lie
struct WavePlace {
    float* p;
    const float* g;
    uint8_t *m, *v, *ms, *vs;
    bf16_t* w;
    uint64_t group;  // of the first pair of blocks
    uint32_t number;
};

// Four whole blocks: 16 bytes of the fp32 tensors a lane and load, 4 of the codes, all of them on the way before the first is used.
__device__ __forceinline__ void four_blocks(const WavePlace& at, const Adam8Args& a, float coef, int lane) {
#pragma clang fp contract(off)
    f32x4 p[4], g[4];
    uint32_t cm[4], cv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        cm[u] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(at.m) + u * 64 + lane);
        cv[u] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(at.v) + u * 64 + lane);
        g[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(at.g) + u * 64 + lane);
        p[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(at.p) + u * 64 + lane);
    }
    const uint32_t old_ms = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t*>(at.ms));
    const uint32_t old_vs = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t*>(at.vs));
    uint32_t new_ms = 0, new_vs = 0;
#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {
        const uint64_t group = at.group + 64 * pair + lane;
        const u32x4 words = philox_4x32_10((uint32_t)group, (uint32_t)(group >> 32), at.number, a.step, a.key0, a.key1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int u = 2 * pair + half;
            const int em = old_ms >> 8 * u & 255, ev = old_vs >> 8 * u & 255;
            // (a block that is not finite: NaN by its factor)
            const float beta1 = em == 255 ? __builtin_nanf("") : a.beta1, beta2 = ev == 255 ? __builtin_nanf("") : a.beta2;
            float m[4], v[4];
            uint32_t most_m = 0, most_v = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t c = cm[u] >> 8 * k;
                m[k] = __builtin_amdgcn_ldexpf(__uint_as_float((c & 127) << 20 | (c & 128) << 24), em - kTopM);
                v[k] = __builtin_amdgcn_ldexpf(__uint_as_float((cv[u] >> 8 * k & 255) << 20), ev - kTopV);
                const float gk = g[u][k] * coef;
                float pk = p[u][k];
                adam8_one(pk, m[k], v[k], gk, beta1, beta2, a);
                p[u][k] = pk;
                most_m = max(most_m, magnitude(m[k]));
                most_v = max(most_v, magnitude(v[k]));
            }
            const int nm = scale_of(wave_max_u32(most_m)), nv = scale_of(wave_max_u32(most_v));
            uint32_t code_m = 0, code_v = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t word = words[2 * half + k / 2], r = k & 1 ? word >> 16 : word & 0xffffu;
                code_m |= (((magnitude(__builtin_amdgcn_ldexpf(m[k], kTopM - nm)) + 8 + 16 * r) >> 20) | __float_as_uint(m[k]) >> 31 << 7) << 8 * k;
                const uint32_t c = (magnitude(__builtin_amdgcn_ldexpf(v[k], kTopV - nv)) + 8 + 16 * r) >> 20;
                code_v |= max(c, min(__float_as_uint(v[k]), 1u)) << 8 * k;
            }
            code_m = nm == 255 ? 0 : code_m;
            code_v = nv == 255 ? 0 : code_v;
            new_ms |= (uint32_t)nm << 8 * u;
            new_vs |= (uint32_t)nv << 8 * u;
            __builtin_nontemporal_store(p[u], reinterpret_cast<f32x4*>(at.p) + u * 64 + lane);
            __builtin_nontemporal_store(code_m, reinterpret_cast<uint32_t*>(at.m) + u * 64 + lane);
            __builtin_nontemporal_store(code_v, reinterpret_cast<uint32_t*>(at.v) + u * 64 + lane);
            if (at.w) {
                bf16x4 o;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = (bf16_t)p[u][k];
                reinterpret_cast<bf16x4*>(at.w)[u * 64 + lane] = o;
            }
        }
    }
    if (lane == 0) {
        *reinterpret_cast<uint32_t*>(at.ms) = new_ms;
        *reinterpret_cast<uint32_t*>(at.vs) = new_vs;
    }
}

// The end of a tensor, `left` elements of up to four blocks, one by one.
__device__ void last_blocks(const WavePlace& at, const Adam8Args& a, float coef, int lane, int left) {
    for (int u = 0; u < 4 && u * kBlock8 < left; ++u) {
        const int i0 = u * kBlock8 + lane * 4;
        const uint64_t group = at.group + 64 * (u / 2) + lane;
        const u32x4 w = philox_4x32_10((uint32_t)group, (uint32_t)(group >> 32), at.number, a.step, a.key0, a.key1);
        const int em = at.ms[u], ev = at.vs[u];
        float p[4], m[4], v[4];
        uint32_t most_m = 0, most_v = 0;
        for (int k = 0; k < 4; ++k) {
            p[k] = m[k] = v[k] = 0.f;
            if (i0 + k >= left) continue;
            p[k] = at.p[i0 + k];
            m[k] = value_of<7, kTopM>(at.m[i0 + k], em);
            v[k] = value_of<8, kTopV>(at.v[i0 + k], ev);
            adam8_one(p[k], m[k], v[k], at.g[i0 + k] * coef, a.beta1, a.beta2, a);
            most_m = max(most_m, magnitude(m[k]));
            most_v = max(most_v, magnitude(v[k]));
        }
        const int nm = scale_of(wave_max_u32(most_m)), nv = scale_of(wave_max_u32(most_v));
        for (int k = 0; k < 4; ++k) {
            if (i0 + k >= left) continue;
            const uint32_t word = w[(u & 1) * 2 + k / 2], r = k & 1 ? word >> 16 : word & 0xffffu;
            at.p[i0 + k] = p[k];
            if (at.w) at.w[i0 + k] = (bf16_t)p[k];
            at.m[i0 + k] = (uint8_t)code_of<7, kTopM, 0>(m[k], r, nm);
            at.v[i0 + k] = (uint8_t)code_of<8, kTopV, 1>(v[k], r, nv);
        }
        if (lane == 0) {
            at.ms[u] = (uint8_t)nm;
            at.vs[u] = (uint8_t)nv;
        }
    }
}

// A wave takes four blocks of 256, a lane four values of each: a block's largest value is a wave's.  Chunks go out from the last to the first: a norm of the gradients that went through them
// in the other direction has left the last ones in the last-level cache.
// Bound by HBM: 18 bytes a parameter.  A workgroup per chunk; 202 million parameters in nine tensors 665 us, 5.5 TB/s (a large copy 5.3; with 2048 workgroups that walk over the chunks
// a sixth longer, with 8192 a tenth): a new workgroup's loads are out while the old ones compute.
__global__ __launch_bounds__(kThreads8) void adam8_kernel(const MomentsList l, const Adam8Args a, const float* __restrict__ norm_coef) {
    const float coef = norm_coef ? norm_coef[1] : 1.0f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = l.chunks - 1 - (int)blockIdx.x, t = tensor_of8(l, chunk);
    const int64_t base = (int64_t)(chunk - l.first[t]) * kChunk8 + wave * (kChunk8 / 4), left = l.n[t] - base, block = base / kBlock8;
    if (left <= 0) return;
    const WavePlace at = {l.master[t] + base, l.g[t] + base, l.m[t] + base, l.v[t] + base, l.ms[t] + block, l.vs[t] + block,
                          l.param[t] ? l.param[t] + base : nullptr, (uint64_t)block * 32, l.number[t]};
    if (left >= kChunk8 / 4) four_blocks(at, a, coef, lane);
    else last_blocks(at, a, coef, lane, (int)left);
}

// m and v as bf16 values (four significant bits: exact).  6 bytes a parameter, 16-byte stores: 202 million 216 us, 5.6 TB/s.
struct ValuesList {
    const uint8_t *m[kListMax8], *v[kListMax8], *ms[kListMax8], *vs[kListMax8];
    bf16_t *m_out[kListMax8], *v_out[kListMax8];
    int64_t n[kListMax8];
    int first[kListMax8];
    int count, chunks;
};
__global__ __launch_bounds__(kThreads8) void moments8_kernel(const ValuesList l) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const int chunk = blockIdx.x;
    int t = 0;
    while (t + 1 < l.count && l.first[t + 1] <= chunk) ++t;
#pragma unroll
    for (int part = 0; part < 2; ++part) {  // a thread's 8 values of either moment: of one block
        const int64_t at = (int64_t)(chunk - l.first[t]) * kChunk8 + (part * kThreads8 + threadIdx.x) * 8, left = l.n[t] - at;
        if (left <= 0) continue;
        const int em = l.ms[t][at / kBlock8], ev = l.vs[t][at / kBlock8];
        if (left < 8) {
            for (int i = 0; i < left; ++i) {
                l.m_out[t][at + i] = (bf16_t)value_of<7, kTopM>(l.m[t][at + i], em);
                l.v_out[t][at + i] = (bf16_t)value_of<8, kTopV>(l.v[t][at + i], ev);
            }
            continue;
        }
        const u32x2 cm = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(l.m[t] + at)), cv = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(l.v[t] + at));
        bf16x8 m, v;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = (bf16_t)value_of<7, kTopM>(cm[i / 4] >> 8 * (i & 3) & 255, em);
            v[i] = (bf16_t)value_of<8, kTopV>(cv[i / 4] >> 8 * (i & 3) & 255, ev);
        }
        st_bf16x8(l.m_out[t] + at, m);
        st_bf16x8(l.v_out[t] + at, v);
    }
}

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
        EZL_REQUIRE(t.n >= 0 && t.n < (1LL << 35) && (t.n == 0 || (t.master && t.exp_avg && t.exp_avg_sq && t.exp_avg_scale && t.exp_avg_sq_scale && t.grad)), EZL_EINVAL,
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
        if (l.count) hipLaunchKernelGGL(adam8_kernel, dim3((unsigned)l.chunks), dim3(kThreads8), 0, (hipStream_t)stream, l, a, (const float*)norm_coef);
        l.count = l.chunks = 0;
    };
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const int64_t chunks = (t.n + kChunk8 - 1) / kChunk8, blocks = (t.n + kBlock8 - 1) / kBlock8;
        bool again = l.count == kListMax8 || l.chunks + chunks >= (1LL << 23);
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
    if (l.count == 0) return EZL_OK;  // (the last one ends a list that is not empty)
    flush();
    EZL_LAUNCH_CHECK(name);
    return EZL_OK;
}

extern "C" int ezl_moments8_list(int count, const ezl_adam8_tensor* tensors, void* const* exp_avg_bf16, void* const* exp_avg_sq_bf16, void* stream) {
    const char* name = "ezl_moments8_list";
    EZL_REQUIRE(count >= 0 && (count == 0 || (tensors && exp_avg_bf16 && exp_avg_sq_bf16)), EZL_EINVAL, "%s: bad count or null argument", name);
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        EZL_REQUIRE(t.n >= 0 && t.n < (1LL << 35) && (t.n == 0 || (t.exp_avg && t.exp_avg_sq && t.exp_avg_scale && t.exp_avg_sq_scale && exp_avg_bf16[i] && exp_avg_sq_bf16[i])),
                    EZL_EINVAL, "%s: null pointer or bad size", name);
        EZL_REQUIRE(aligned(t.exp_avg, 16) && aligned(t.exp_avg_sq, 16) && ezl_aligned16(exp_avg_bf16[i]) && ezl_aligned16(exp_avg_sq_bf16[i]), EZL_EINVAL,
                    "%s: pointers must be 16-byte aligned", name);
    }
    ValuesList l;
    l.count = l.chunks = 0;
    const auto flush = [&]() {
        if (l.count) hipLaunchKernelGGL(moments8_kernel, dim3((unsigned)l.chunks), dim3(kThreads8), 0, (hipStream_t)stream, l);
        l.count = l.chunks = 0;
    };
    for (int i = 0; i < count; ++i) {
        const ezl_adam8_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const int64_t chunks = (t.n + kChunk8 - 1) / kChunk8;
        if (l.count == kListMax8 || l.chunks + chunks >= (1LL << 23)) flush();
        const int s = l.count++;
        l.m[s] = (const uint8_t*)t.exp_avg; l.v[s] = (const uint8_t*)t.exp_avg_sq; l.ms[s] = (const uint8_t*)t.exp_avg_scale; l.vs[s] = (const uint8_t*)t.exp_avg_sq_scale;
        l.m_out[s] = (bf16_t*)exp_avg_bf16[i]; l.v_out[s] = (bf16_t*)exp_avg_sq_bf16[i]; l.n[s] = t.n; l.first[s] = l.chunks;
        l.chunks += (int)chunks;
    }
    if (l.count == 0) return EZL_OK;  // (the last one ends a list that is not empty)
    flush();
    EZL_LAUNCH_CHECK(name);
    return EZL_OK;
}
