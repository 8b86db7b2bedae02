// Rotary positions of any pairing: the first `turned` elements of a head are pairs (j, j + turned / 2), or (2 j, 2 j + 1), turned by the angle
// position * inv_freq[j]; the rest of the head passes through.  out = scale * (x1 cos - x2 sin, x2 cos + x1 sin); backward turns the other way.
//
// No table: an angle is position times frequency in 64 bits, reduced to a turn there, so that a position of a million is as exact as one of ten (in 32 bits its angle
// is off by up to 0.03), and no length has to be known beforehand.
#include "common.h"

#include "../../include/ezl.h"

namespace {

constexpr int kRotaryBlock = 256;

struct RotarySide {
    const bf16_t* x;
    bf16_t* out;
    int64_t seq, batch, head;  // strides of x in elements
    int heads;
};
struct RotaryArgs {
    RotarySide q, k;
    const void* inv_freq;
    const int64_t* position_ids;  // null: the place in the sequence
    int64_t pos_seq, pos_batch;
    int64_t tokens;  // s * b, s-major
    int b, d, turned, f64;
    float scale, sign;
};

// cosine and sine of position * frequency, times scale; the sine with the direction's sign
__device__ __forceinline__ void angle_of(const RotaryArgs& a, double position, int j, float& c, float& s) {
    const double f = a.f64 ? ((const double*)a.inv_freq)[j] : (double)((const float*)a.inv_freq)[j];
    const double t = position * f * 0.15915494309189535;  // turns
    const float r = (float)(t - rint(t));
    c = __builtin_amdgcn_cosf(r) * a.scale;
    s = __builtin_amdgcn_sinf(r) * (a.scale * a.sign);
}

template <bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryBlock) void rotary_kernel(const RotaryArgs a) {
    const int half = a.turned >> 1, heads = a.q.heads + a.k.heads;
    const int per_head = half + (a.d - a.turned);  // pairs, then single elements
    const int64_t items = a.tokens * heads * per_head;
    for (int64_t it = (int64_t)blockIdx.x * kRotaryBlock + threadIdx.x; it < items; it += (int64_t)gridDim.x * kRotaryBlock) {
        const int j = (int)(it % per_head);
        const int64_t th = it / per_head;
        int head = (int)(th % heads);
        const int64_t token = th / heads, si = token / a.b, bi = token % a.b;
        const bool second = head >= a.q.heads;
        const RotarySide& side = second ? a.k : a.q;
        head -= second ? a.q.heads : 0;
        const bf16_t* x = side.x + si * side.seq + bi * side.batch + head * side.head;
        bf16_t* out = side.out + (token * side.heads + head) * a.d;
        if (j >= half) {
            out[j + half] = x[j + half];
            continue;
        }
        const int64_t position = a.position_ids ? a.position_ids[bi * a.pos_batch + si * a.pos_seq] : si;
        float c, s;
        angle_of(a, (double)position, j, c, s);
        const int i1 = INTERLEAVED ? 2 * j : j, i2 = INTERLEAVED ? 2 * j + 1 : j + half;
        const float x1 = (float)x[i1], x2 = (float)x[i2];
        out[i1] = (bf16_t)(x1 * c - x2 * s);
        out[i2] = (bf16_t)(x2 * c + x1 * s);
    }
}

}  // namespace

extern "C" int ezl_rotary(const ezl_rotary_side* q, const ezl_rotary_side* k, const void* inv_freq, int inv_freq_f64, const void* position_ids,
                          int64_t pos_seq_stride, int64_t pos_batch_stride, int64_t s, int64_t b, int64_t d, int64_t turned, int interleaved, float scale,
                          int backward, void* stream) {
    EZL_REQUIRE(q && s >= 0 && b >= 0 && s < (1LL << 31) && b < (1LL << 31) && s * b < (1LL << 40), EZL_EINVAL, "ezl_rotary: bad size");
    EZL_REQUIRE(d > 0 && d % 8 == 0 && d <= (1 << 16) && turned > 0 && turned % 2 == 0 && turned <= d, EZL_EUNSUPPORTED,
                "ezl_rotary: the head's width must be a multiple of 8, what is turned of it even and not more (got %lld, %lld)", (long long)d, (long long)turned);
    RotaryArgs a = {};
    int64_t heads = 0;
    for (const ezl_rotary_side* side : {q, k}) {
        if (!side) continue;
        EZL_REQUIRE(side->heads >= 0 && side->heads < (1 << 20), EZL_EINVAL, "ezl_rotary: bad number of heads");
        heads += side->heads;
        if (side->heads == 0 || s * b == 0) continue;
        EZL_REQUIRE(side->x && side->out && ezl_aligned16(side->x) && ezl_aligned16(side->out), EZL_EINVAL, "ezl_rotary: null or misaligned pointer");
        EZL_REQUIRE(side->seq_stride % 8 == 0 && side->batch_stride % 8 == 0 && side->head_stride % 8 == 0 && side->seq_stride >= 0 && side->batch_stride >= 0 &&
                        side->head_stride >= 0,
                    EZL_EINVAL, "ezl_rotary: strides must be multiples of 8");
        (side == q ? a.q : a.k) = {(const bf16_t*)side->x, (bf16_t*)side->out, side->seq_stride, side->batch_stride, side->head_stride, (int)side->heads};
    }
    if (s * b == 0 || heads == 0) return EZL_OK;
    EZL_REQUIRE(inv_freq && (reinterpret_cast<uintptr_t>(inv_freq) & (inv_freq_f64 ? 7 : 3)) == 0 && (reinterpret_cast<uintptr_t>(position_ids) & 7) == 0, EZL_EINVAL,
                "ezl_rotary: null or misaligned pointer");
    a.inv_freq = inv_freq;
    a.position_ids = (const int64_t*)position_ids;
    a.pos_seq = pos_seq_stride;
    a.pos_batch = pos_batch_stride;
    a.tokens = s * b;
    a.b = (int)b; a.d = (int)d; a.turned = (int)turned; a.f64 = inv_freq_f64 != 0;
    a.scale = scale;
    a.sign = backward ? -1.f : 1.f;
    const int64_t items = a.tokens * heads * (turned / 2 + d - turned), blocks = (items + kRotaryBlock - 1) / kRotaryBlock;
    hipLaunchKernelGGL(interleaved ? rotary_kernel<true> : rotary_kernel<false>, dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), dim3(kRotaryBlock), 0,
                       (hipStream_t)stream, a);
    EZL_LAUNCH_CHECK("ezl_rotary");
    return EZL_OK;
}
