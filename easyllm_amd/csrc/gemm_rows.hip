// Forward products of up to 16 rows, C[M,N] = X[M,K] W[N,K]^T with an epilogue: a handful of tokens through a layer.
//
// What bounds them is the weights' way from memory, each of which is used M times only: nothing is gained by staging them in LDS, and few columns per workgroup
// bring every CU to the memory.  A workgroup walks over tiles of 16 columns.  Its eight waves own the 64-wide blocks of K in turn (together they read a row
// of W in pieces of 1 KiB); a wave keeps its blocks of X in registers for all tiles and the next tile's weights on the way while the current ones are
// multiplied.  (X loaded anew per tile costs as much as W: 16 rows 29 us at 11008 x 4096, so 24.)  The eight sums of a tile meet in LDS, double buffered: one
// barrier per tile, behind which the waves take turns to add them, in wave order, and to write the result.
#include "gemm_rows.h"

namespace {

constexpr int kWaves = 8;

// KB: 64-wide blocks of K a wave owns
template <int KB>
__global__ __launch_bounds__(kWaves * 64) void gemm_rows_kernel(const bf16_t* __restrict__ X, const bf16_t* __restrict__ W, bf16_t* __restrict__ C, int M, int N,
                                                                int K, int64_t ldx, int64_t ldw, int64_t ldc, const Epilogue epi) {
    __shared__ f32x4 sums[2][kWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int tiles = (N + 15) >> 4;
    bf16x8 x[KB][2], w[KB][2];
    // rows past the last are read from the last, their results are not stored; what lies past K is read from the row's start and cleared
    const bf16_t* const xrow = X + (int64_t)min(r, M - 1) * ldx;
    const auto row_of = [&](int tile) { return W + (int64_t)min(tile * 16 + r, N - 1) * ldw; };
    const auto k_of = [&](int u, int h) { return (wave + u * kWaves) * 64 + h * 32 + g * 8; };
    const auto load = [&](bf16x8 (&dst)[2], const bf16_t* row, int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) dst[h] = ld_bf16x8(row + (k_of(u, h) < K ? k_of(u, h) : 0));
    };
    const auto clear_tail = [&](bf16x8 (&v)[2], int u) {
        if ((wave + u * kWaves) * 64 + 64 > K)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (k_of(u, h) >= K) v[h] = bf16x8{};
    };
    int tile = blockIdx.x;
    {
        const bf16_t* row = row_of(tile);
#pragma unroll
        for (int u = 0; u < KB; ++u) load(w[u], row, u);
    }
#pragma unroll
    for (int u = 0; u < KB; ++u) load(x[u], xrow, u);
#pragma unroll
    for (int u = 0; u < KB; ++u) clear_tail(x[u], u);
    int buf = 0, turn = 0;
    for (; tile < tiles; tile += gridDim.x) {
        const int next = tile + (int)gridDim.x;
        const bf16_t* row = row_of(next);
        f32x4 a0 = {0.f, 0.f, 0.f, 0.f}, a1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < KB; ++u) {
            if (u + 2 >= KB) clear_tail(w[u], u);  // (K ends in the last two)
            a0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u][0], x[u][0], a0, 0, 0, 0);
            a1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u][1], x[u][1], a1, 0, 0, 0);
            if (next < tiles) load(w[u], row, u);
        }
        // The sum below may not read the products' registers before they are written, which takes the hardware wait states that the compiler leaves out where the branch
        // above goes past the loads (seen as wrong last elements; tests/test_mfma_wait_states.py looks for such reads).
        asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a0), "+v"(a1));
        sums[buf][wave][lane] = a0 + a1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // written; the next tile's loads stay on the way across the barrier
        wave_barrier();
        // a register q of lane l is C[l & 15][16 tile + 4 (l >> 4) + q].  (A buffer is written again two tiles on, behind a barrier that its reader has passed.)
        const int n = tile * 16 + g * 4;
        if (wave == turn && r < M && n < N) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < kWaves; ++q) {
                const f32x4 s = sums[buf][q][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += s[e];
            }
            store_epilogue<4>(v, C, ldc, r, n, epi);
        }
        buf ^= 1;
        turn = (turn + 1) & (kWaves - 1);
    }
}

}  // namespace

void gemm_rows_launch(const void* X, const void* W, void* C, int M, int N, int K, int64_t ldx, int64_t ldw, int64_t ldc, const Epilogue& epi, hipStream_t st) {
    static_assert(kRowsMaxK <= 10 * 64 * kWaves, "blocks of K in registers");
    const int tiles = (N + 15) / 16, kb = (K + 64 * kWaves - 1) / (64 * kWaves);
    // One workgroup per CU where it has 24 loads per wave and more on the way, two where fewer: 8 rows, 8192 x 1000 6.2 -> 5.7 us, but 11008 x 4096 21.6 -> 24.2.
    const int most = kb <= 2 ? 512 : 256;
    const dim3 grid((unsigned)(tiles < most ? tiles : most));
#define EZL_ROWS(KB)                                                                                                                                   \
    hipLaunchKernelGGL((gemm_rows_kernel<KB>), grid, dim3(kWaves * 64), 0, st, (const bf16_t*)X, (const bf16_t*)W, (bf16_t*)C, M, N, K, ldx, ldw, ldc, epi); \
    break
    switch (kb) {  // (blocks past K cost loads of a line that is there)
        case 1: EZL_ROWS(1);
        case 2: EZL_ROWS(2);
        case 3: EZL_ROWS(3);
        case 4: EZL_ROWS(4);
        case 5: case 6: EZL_ROWS(6);
        case 7: case 8: EZL_ROWS(8);
        default: EZL_ROWS(10);
    }
#undef EZL_ROWS
}
