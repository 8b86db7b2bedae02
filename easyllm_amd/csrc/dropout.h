// Dropout from a counter: which elements of a tensor are dropped follows from their index and two numbers, so the mask is computed
// where it is needed, in the forward and in the backward pass, and never stored.
//
// Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): elements 8 g .. 8 g + 7 of a tensor
// take the 128 bits of the counter (g low, g high, offset, step) under the key `seed` as eight 16-bit numbers, the low half of a word first, and
// an element is dropped where its number is below drop_of_65536.  16 bits an element: the share is a multiple of 2^-16 (and
// kept elements are scaled by what is exactly its counterpart), one generator call serves the 16 bytes of a lane's vector.
// (32 bits, two calls: 8192 x 8192 forward with a residual 73.5 -> 74.8 us, backward 43.0 -> 49.7, the norm's backward 131 -> 142.)
#pragma once
#include "common.h"

#include "../../include/ezl.h"

struct DropArgs {
    uint32_t key0, key1, offset, threshold;
    float scale;
    const long long* step;  // device word, or null: 0
};

// host: the kernels' form of a caller's description (NULL: nothing is dropped)
inline int drop_args(const char* name, const ezl_dropout* d, DropArgs& a) {
    a = {0, 0, 0, 0, 1.f, nullptr};
    if (!d) return EZL_OK;
    EZL_REQUIRE(d->drop_of_65536 >= 0 && d->drop_of_65536 <= 65536, EZL_EINVAL, "%s: drop_of_65536 must be 0 .. 65536", name);
    EZL_REQUIRE((reinterpret_cast<uintptr_t>(d->step) & 7) == 0, EZL_EINVAL, "%s: step must be 8-byte aligned", name);
    a.key0 = (uint32_t)d->seed;
    a.key1 = (uint32_t)(d->seed >> 32);
    a.offset = d->offset;
    a.threshold = (uint32_t)d->drop_of_65536;
    a.scale = d->drop_of_65536 == 65536 ? 0.f : 65536.f / (float)(65536 - d->drop_of_65536);
    a.step = (const long long*)d->step;
    return EZL_OK;
}

#ifdef __HIPCC__
__device__ __forceinline__ uint32_t drop_step(const DropArgs& a) { return a.step ? (uint32_t)*a.step : 0u; }

__device__ __forceinline__ u32x4 philox_4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// v[j] = dropout(v[j]) of the eight elements of `group`.  Dropped ones are zero whatever they held.
__device__ __forceinline__ void drop8(float (&v)[8], int64_t group, const DropArgs& a, uint32_t step) {
    const u32x4 w = philox_4x32_10((uint32_t)group, (uint32_t)(group >> 32), a.offset, step, a.key0, a.key1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = (w[j] & 0xffffu) < a.threshold ? 0.f : v[2 * j] * a.scale;
        v[2 * j + 1] = (w[j] >> 16) < a.threshold ? 0.f : v[2 * j + 1] * a.scale;
    }
}
#endif
