// Forward products of a few rows with an epilogue (gemm_rows.hip); what ezl_gemm_bf16_epilogue checks holds.
#pragma once
#include "gemm_tile.h"

// Up to 16 rows (one MFMA fragment), whose K fits the registers of a workgroup, and few enough columns: where N / 16 tiles leave most of a last round of workgroups
// empty, or the weights' stream is long, or many rows have to come into registers first, the tiles do better.  us of the tiles and of this kernel, weights from HBM, GELU, bias and a
// residual, N x K, at 1, 8 and 16 rows:  256 x 256 4.2, 3.1  4.4, 3.4  4.4, 3.4;  2048 x 2048 10.7, 5.5  10.6, 6.2  10.8, 6.9;  8192 x 2560 17.3, 13.3  15.5, 13.7  15.9, 14.7;
// 4096 x 4096 15.0, 10.7  14.7, 11.1  15.0, 12.6;  8192 x 4096 20.7, 17.5  20.0, 17.3  20.3, 18.7;  4096 x 5120 16.7, 12.3  16.4, 13.0  16.8, 15.1.  What the rule
// takes and should not: 5120 x 3584 15.9, 15.7  15.7, 16.5;  5120 x 5120 at 8 rows 18.5, 19.5;  256 x 4096 at 16 rows 9.0, 9.8.  What it leaves to the tiles:  5120 x 3584 at 16 rows 15.2, 17.7;
// 8192 x 4096 at 16 rows, as above;  512 x 6144 10.7, 11.2  10.7, 12.9  10.9, 15.0;  6144 x 6144 23.0, 24.7  22.4, 26.4  22.8, 28.3;  11008 x 4096 23.4, 22.7  22.5, 22.4  22.8, 23.9;
// 13696 x 5120 30.7, 33.7  29.9, 33.5  30.4, 35.7;  16384 x 4096 32.0, 29.9  31.0, 29.5  31.1, 30.9;  32000 x 512 10.5, 11.5  10.6, 12.1  10.2, 12.4.
constexpr int kRowsMaxK = 5120;
inline bool gemm_rows_pays(int64_t M, int64_t N, int64_t K) {
    if (M <= 8) return N <= 8192 && K <= kRowsMaxK;
    return M <= 16 && ((N <= 4096 && K <= 4096) || (N <= 8192 && K <= 2560));
}
__attribute__((visibility("hidden"))) void gemm_rows_launch(const void* X, const void* W, void* C, int M, int N, int K, int64_t ldx, int64_t ldw, int64_t ldc,
                                                            const Epilogue& epi, hipStream_t st);
