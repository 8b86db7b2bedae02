// Rotary positions of any pairing: the first `turned` elements of a head are pairs (j, j + turned / 2), or (2 j, 2 j + 1), turned by the angle
// position * inv_freq[j]; the rest of the head passes through.  out = scale * (x1 cos - x2 sin, x2 cos + x1 sin); backward turns the other way.
//
// No table: an angle is position times frequency in 64 bits, reduced to a turn there, so that a position of a million is as exact as one of ten (in 32 bits its angle
// is off by up to 0.03), and no length has to be known beforehand.
//
// Long calls are bound by HBM, every byte once each way: q and k of 16384 tokens, 32 heads of 128 each, 101 us a direction (5.3 TB/s; the angles, computed once per token and pair for four heads or more, cost
// nothing there); 8192 tokens of 64 and 8 heads, half of each turned, read out of the projection's packed result 61.8 (4.9).  Short ones are bound by the launch: a token's 40 heads
// 3.2 us, 1167 tokens of 24 heads, 24 of 64 elements turned in neighbouring pairs, 4.8.
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
    int slots, turned_slots;       // of a head
    int head_lanes, block_tokens;  // threads of a block: [block_tokens][head_lanes][slots]
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

typedef bf16x8 __attribute__((aligned(2))) bf16x8_any;  // (a half of a head that is no multiple of 8 starts anywhere)

// n <= 8 elements from p on; WHOLE: n is 8 and p on 16 bytes
template <bool WHOLE>
__device__ __forceinline__ bf16x8 load8(const bf16_t* p, int n) {
    if constexpr (WHOLE) return ld_bf16x8_nt(p);
    if (n == 8) return *reinterpret_cast<const bf16x8_any*>(p);
    bf16x8 v = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) v[i] = p[i];
    return v;
}
template <bool WHOLE, bool STREAM>
__device__ __forceinline__ void store8(bf16_t* p, bf16x8 v, int n) {
    if constexpr (WHOLE) {
        st_result<STREAM>(p, v);
        return;
    }
    if (n == 8) {
        *reinterpret_cast<bf16x8_any*>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = v[i];
}

// A thread owns one slot of a head - eight pairs j (of neighbours: four), or eight elements that are copied - for HEADS heads of one token, and computes its
// angles once, while their elements are on the way.
template <bool INTERLEAVED, bool WHOLE, int HEADS, bool STREAM>
__global__ __launch_bounds__(kRotaryBlock) void rotary_kernel(const RotaryArgs a) {
    const int half = a.turned >> 1, heads = a.q.heads + a.k.heads;
    const int lane = (int)(threadIdx.x / (unsigned)a.slots), slot = threadIdx.x - lane * a.slots;
    const int token_in = (int)((unsigned)lane / (unsigned)a.head_lanes);
    const int head0 = lane - token_in * a.head_lanes + blockIdx.y * (HEADS * a.head_lanes);
    if (token_in >= a.block_tokens) return;
    const int64_t token = (int64_t)blockIdx.x * a.block_tokens + token_in;
    if (token >= a.tokens) return;
    const int64_t si = a.b == 1 ? token : token / a.b, bi = a.b == 1 ? 0 : token - si * a.b;
    const bool turns = slot < a.turned_slots;
    // Its first element, in the part of the head that its like share (of halves: the first of both).  The last slot of a part that is no multiple of 8 reaches back into the one before, whose
    // thread writes the same there: every access is 16 bytes.
    const int part = turns ? (INTERLEAVED ? a.turned : half) : a.d - a.turned;
    int e = (turns ? slot : slot - a.turned_slots) * 8;
    if (!WHOLE && part >= 8) e = min(e, part - 8);
    const int n = WHOLE ? 8 : min(8, part - e), e0 = turns ? e : a.turned + e;
    const int j0 = INTERLEAVED ? e / 2 : e;  // its first pair
    const bf16_t* x[HEADS];
    bf16_t* out[HEADS];
    bf16x8 v[HEADS], w[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        int head = head0 + i * a.head_lanes;
        const bool second = head >= a.q.heads;
        const RotarySide& side = second ? a.k : a.q;
        head -= second ? a.q.heads : 0;
        x[i] = side.x + si * side.seq + bi * side.batch + head * side.head + e0;
        out[i] = side.out + (token * side.heads + head) * a.d + e0;
        if (head0 + i * a.head_lanes < heads) {
            v[i] = load8<WHOLE>(x[i], n);
            if (!INTERLEAVED && turns) w[i] = load8<WHOLE>(x[i] + half, n);
        }
    }
    float c[INTERLEAVED ? 4 : 8], s[INTERLEAVED ? 4 : 8];
    if (turns) {
        const double position = (double)(a.position_ids ? a.position_ids[bi * a.pos_batch + si * a.pos_seq] : si);
#pragma unroll
        for (int p = 0; p < (INTERLEAVED ? 4 : 8); ++p) angle_of(a, position, WHOLE ? j0 + p : min(j0 + p, half - 1), c[p], s[p]);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        if (head0 + i * a.head_lanes >= heads) break;
        if (turns) {
            float f[8], g[8], y[8], z[8];
            unpack8(v[i], f);
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    y[2 * p] = f[2 * p] * c[p] - f[2 * p + 1] * s[p];
                    y[2 * p + 1] = f[2 * p + 1] * c[p] + f[2 * p] * s[p];
                }
            } else {
                unpack8(w[i], g);
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    y[p] = f[p] * c[p] - g[p] * s[p];
                    z[p] = g[p] * c[p] + f[p] * s[p];
                }
                store8<WHOLE, STREAM>(out[i] + half, pack8(z), n);
            }
            v[i] = pack8(y);
        }
        store8<WHOLE, STREAM>(out[i], v[i], n);
    }
}

// (stream_out: only results of many pieces are more than the caches hold)
template <bool INTERLEAVED, bool WHOLE>
void launch_heads(const RotaryArgs& a, int per_thread, dim3 grid, dim3 block, bool stream_out, hipStream_t st) {
    constexpr int MANY = INTERLEAVED ? 8 : 4;
    if (per_thread == 1) hipLaunchKernelGGL((rotary_kernel<INTERLEAVED, WHOLE, 1, false>), grid, block, 0, st, a);
    else if (per_thread == 2) hipLaunchKernelGGL((rotary_kernel<INTERLEAVED, WHOLE, 2, false>), grid, block, 0, st, a);
    else if (stream_out) hipLaunchKernelGGL((rotary_kernel<INTERLEAVED, WHOLE, MANY, WHOLE>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rotary_kernel<INTERLEAVED, WHOLE, MANY, false>), grid, block, 0, st, a);
}

}  // namespace

extern "C" int ezl_rotary(const ezl_rotary_side* q, const ezl_rotary_side* k, const void* inv_freq, int inv_freq_f64, const void* position_ids,
                          int64_t pos_seq_stride, int64_t pos_batch_stride, int64_t s, int64_t b, int64_t d, int64_t turned, int interleaved, float scale,
                          int backward, void* stream) {
    EZL_REQUIRE(q && s >= 0 && b >= 0 && s < (1LL << 31) && b < (1LL << 31) && s * b < (1LL << 31), EZL_EINVAL, "ezl_rotary: bad size");
    EZL_REQUIRE(d > 0 && d % 8 == 0 && d <= 8 * kRotaryBlock && turned > 0 && turned % 2 == 0 && turned <= d, EZL_EUNSUPPORTED,
                "ezl_rotary: the head's width must be a multiple of 8 up to 2048, what is turned of it even and not more (got %lld, %lld)", (long long)d, (long long)turned);
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
    a.turned_slots = (int)(interleaved ? (turned + 7) / 8 : (turned / 2 + 7) / 8);
    a.slots = a.turned_slots + (int)((d - turned + 7) / 8);
    EZL_REQUIRE(a.slots <= kRotaryBlock, EZL_EUNSUPPORTED, "ezl_rotary: a head's %lld elements, %lld of them turned, are more than %d pieces of 8", (long long)d, (long long)turned,
                kRotaryBlock);
    const int most = kRotaryBlock / a.slots;  // heads a block has threads for
    // Heads of a thread: few items want threads, many want one set of angles and several loads each.  us with 1, 2, 4, 8, heads of 128, 32 + 8 of them: 1 token 3.0, 3.3, 3.9,
    // 4.9; 256 4.0, 3.8, 4.5, 5.5; 512 5.6, 4.5, 4.8, 6.0; 1024 8.4, 6.1, 6.3, 6.7; 2048 17.4, 10.8, 9.8, 10.2; 16384 of 32 + 32 136, 106, 91, 92; neighbours, which
    // need half the angles and registers a slot, 138, 114, 94, 87.
    const int64_t items = a.tokens * heads * a.slots;
    const int per_thread = items <= 1 << 16 ? 1 : items <= 3 << 17 ? 2 : interleaved ? 8 : 4;
    const int64_t lanes = (heads + per_thread - 1) / per_thread;
    a.head_lanes = (int)(lanes < most ? lanes : most);
    a.block_tokens = most / a.head_lanes;
    const dim3 grid((unsigned)((a.tokens + a.block_tokens - 1) / a.block_tokens), (unsigned)((heads + per_thread * a.head_lanes - 1) / (per_thread * a.head_lanes)));
    const dim3 block((unsigned)((a.block_tokens * a.head_lanes * a.slots + 63) / 64 * 64));
    const bool whole = turned % (interleaved ? 8 : 16) == 0, stream_out = ezl_streams(a.tokens * heads * d * 2);
    (interleaved ? whole ? launch_heads<true, true> : launch_heads<true, false> : whole ? launch_heads<false, true> : launch_heads<false, false>)(
        a, per_thread, grid, block, stream_out, (hipStream_t)stream);
    EZL_LAUNCH_CHECK("ezl_rotary");
    return EZL_OK;
}
