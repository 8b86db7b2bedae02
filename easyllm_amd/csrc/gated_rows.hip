// Products of up to 16 rows whose weights are streamed once: act(X W^T) * (X W2^T) and X W^T, a handful of tokens through a gated MLP.
//
// What bounds them is the weights' way from memory.  Every CU takes the same number of columns, to the column (as whole tiles of 16 some would take a fifth more), eight of W
// and the same eight of W2 at a time, or sixteen of W alone: what a fragment has rows for past the CU's last column is read from that again, which costs
// no traffic.  The eight waves of a workgroup own the 64-wide blocks of K in turn; a wave has up to 16 of them in registers and the same of what comes next - the rest of a long K, or the next
// columns - on the way into each as soon as it is used.  The tokens lie in LDS.  A tile's eight sums meet there too, double buffered: one barrier per tile, behind which the
// waves take turns to add them, in wave order, and to write the result.
// One row through 4096 x 11008: both first products 35.6 us (5.1 TB/s of the 5.3 that a copy reaches), the whole block 58 (4.6); eight rows 39.7 and 64.
#include "gated_rows.h"

namespace {

constexpr int kWaves = 8;

// SB: 64-wide blocks of K that a wave has in registers
template <int SB, bool PAIRS>
__global__ __launch_bounds__(kWaves * 64) void stream_rows_kernel(const bf16_t* __restrict__ X, const bf16_t* __restrict__ W, const bf16_t* __restrict__ W2, bf16_t* __restrict__ C,
                                                                  const Kept kept, int M, int cols, int K, int64_t ldx, int64_t ldw, int act, int segments) {
    constexpr int COLS = PAIRS ? 8 : 16;  // of a tile
    __shared__ __attribute__((aligned(16))) bf16_t tokens[kStreamLdsBytes / 2];
    __shared__ f32x4 sums[2][kWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int first = (int)((int64_t)cols * blockIdx.x / gridDim.x), end = (int)((int64_t)cols * (blockIdx.x + 1) / gridDim.x);
    const int blocks = (K + 511) / 512, row_elements = blocks * 512 + 8;  // (eight waves' blocks of K; rows apart by 4 banks)
    const auto k_of = [&](int u, int h) { return (wave + u * kWaves) * 64 + h * 32 + g * 8; };
    const auto row_of = [&](int col) {
        const bf16_t* w = PAIRS && r >= 8 ? W2 : W;
        return w + (int64_t)min(col + (PAIRS ? r & 7 : r), end - 1) * ldw;
    };
    bf16x8 w[SB][2];
    // what lies past K is read from the row's start and cleared
    const auto load = [&](bf16x8 (&dst)[2], const bf16_t* row, int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) dst[h] = ld_bf16x8(row + (k_of(u, h) < K ? k_of(u, h) : 0));
    };
    // The tokens are on the way before the first weights: behind them they would come last, and nothing be fetched meanwhile.  What is more than EARLY pieces of a thread is brought first.
    constexpr int EARLY = 8;
    const int row_pieces = row_elements / 8, pieces = M * row_pieces;
    const auto fetch = [&](int i) {
        const int m = min(i, pieces - 1) / row_pieces, k = (min(i, pieces - 1) - m * row_pieces) * 8;
        bf16x8 x = ld_bf16x8(X + m * ldx + (k < K ? k : 0));
        if (k >= K) x = bf16x8{};
        return x;
    };
    for (int i = threadIdx.x + EARLY * kWaves * 64; i < pieces; i += kWaves * 64) *reinterpret_cast<bf16x8*>(tokens + i * 8) = fetch(i);
    bf16x8 early[EARLY];
#pragma unroll
    for (int j = 0; j < EARLY; ++j)
        if (j * kWaves * 64 < pieces) early[j] = fetch(threadIdx.x + j * kWaves * 64);
    asm volatile("" ::: "memory");
    const bf16_t* row = row_of(first);
#pragma unroll
    for (int v = 0; v < SB; ++v) load(w[v], row, v);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < EARLY; ++j) {
        const int i = threadIdx.x + j * kWaves * 64;
        if (i < pieces) *reinterpret_cast<bf16x8*>(tokens + i * 8) = early[j];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the weights stay on the way across the barrier)
    wave_barrier();
    const bf16_t* const mine = tokens + min(r, M - 1) * row_elements + wave * 64 + g * 8;
    int buf = 0, turn = 0;
    for (int col = first; col < end; col += COLS) {
        f32x4 a0 = {0.f, 0.f, 0.f, 0.f}, a1 = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < segments; ++s) {
            // (Loads are made in any case: where one may be left out, the compiler waits for all of them.  Behind the last column it is a row that was just read.)
            const bool last = s + 1 == segments;
            const int u0 = s * SB, next_u0 = last ? 0 : u0 + SB;
            if (last) row = row_of(col + COLS);
#pragma unroll
            for (int v = 0; v < SB; ++v) {
                const int u = u0 + v;
                const bf16_t* const at = mine + min(u, blocks - 1) * 512;
                bf16x8 x[2] = {*reinterpret_cast<const bf16x8*>(at), *reinterpret_cast<const bf16x8*>(at + 32)};
                if ((wave + u * kWaves) * 64 + 64 > K) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (k_of(u, h) >= K) w[v][h] = x[h] = bf16x8{};
                }
                a0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[v][0], x[0], a0, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[v][1], x[1], a1, 0, 0, 0);
                load(w[v], row, next_u0 + v);
            }
        }
        // The sum below may not read the products' registers before they are written: wait states that the compiler leaves out where a branch goes past the loads.
        asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a0), "+v"(a1));
        sums[buf][wave][lane] = a0 + a1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wave_barrier();
        // a register e of lane l is the product of row l & 15 with the tile's weight row 4 (l >> 4) + e.  (A buffer is written again two tiles on, behind a barrier that its reader has passed.)
        if (wave == turn && r < M && (!PAIRS || g < 2)) {
            const auto sum = [&](int from) {
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < kWaves; ++q) {
                    const f32x4 x = sums[buf][q][from];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += x[e];
                }
                return v;
            };
            const f32x4 a = sum(lane);
            f32x4 b = a;
            if constexpr (PAIRS) b = sum(lane + 32);
            const int n = col + g * 4;
            const int64_t at = (int64_t)r * cols + n;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (n + e >= end) break;
                float y = a[e];
                if constexpr (PAIRS) {
                    y = (act == EZL_GATE_SILU ? gate_value<EZL_GATE_SILU>(y) : act == EZL_GATE_GELU ? gate_value<EZL_GATE_GELU>(y)
                         : act == EZL_GATE_GELU_TANH ? gate_value<EZL_GATE_GELU_TANH>(y) : gate_value<EZL_GATE_RELU>(y)) * b[e];
                    if (kept.p) keep_one(a[e], b[e], kept, r, n + e);
                }
                C[at + e] = (bf16_t)y;
            }
        }
        buf ^= 1;
        turn = (turn + 1) & (kWaves - 1);
    }
}

template <bool PAIRS>
void launch_stream(const void* X, const void* W, const void* W2, void* C, const Kept& kept, int M, int cols, int K, int64_t ldx, int64_t ldw, int act, hipStream_t st) {
    const int tiles = (cols + (PAIRS ? 7 : 15)) / (PAIRS ? 8 : 16), blocks = (K + 64 * kWaves - 1) / (64 * kWaves);
    const int segments = (blocks + 15) / 16, sb = (blocks + segments - 1) / segments;
    const dim3 grid((unsigned)(tiles < 256 ? tiles : 256));
#define EZL_STREAM(SB)                                                                                                                                                       \
    hipLaunchKernelGGL((stream_rows_kernel<SB, PAIRS>), grid, dim3(kWaves * 64), 0, st, (const bf16_t*)X, (const bf16_t*)W, (const bf16_t*)W2, (bf16_t*)C, kept, M, \
                       cols, K, ldx, ldw, act, (blocks + SB - 1) / SB);                                                                                                     \
    break
    switch (sb) {  // (blocks past K cost loads of a line that is there)
        case 1: EZL_STREAM(1);
        case 2: EZL_STREAM(2);
        case 3: EZL_STREAM(3);
        case 4: EZL_STREAM(4);
        case 5: case 6: EZL_STREAM(6);
        case 7: case 8: EZL_STREAM(8);
        case 9: case 10: case 11: EZL_STREAM(11);
        default: EZL_STREAM(16);
    }
#undef EZL_STREAM
}

}  // namespace

void stream_rows_launch(const void* X, const void* W, const void* W2, void* C, const Kept& kept, int M, int cols, int K, int64_t ldx, int64_t ldw, int act, hipStream_t st) {
    (W2 ? launch_stream<true> : launch_stream<false>)(X, W, W2, C, kept, M, cols, K, ldx, ldw, act, st);
}
