// Forward products of a few rows with an epilogue (gemm_rows.hip); what ezl_gemm_bf16_epilogue checks holds.
#pragma once
#include "gemm_tile.h"

// Up to 16 rows (one MFMA fragment), whose K fits the registers of a workgroup.  us of the tiles and of this kernel, 8 rows, weights from HBM, GELU and a residual: N x K
// 688 x 256 4.3, 3.4; 2048 x 2048 9.8, 5.8; 1024 x 4096 9.8, 8.8; 4096 x 4096 14.6, 11.1; 8192 x 5120 23.7, 21.2; the longer the weights' stream the less:
// 5120 x 5120 19.7, 19.8; 11008 x 4096 23.2, 22.8; 28672 x 6144 72.9, 71.8.  (One row 14.6, 10.4 and 22.8, 21.9 at 4096 and 11008 x 4096; 16 rows 15.0, 12.5 and 22.9,
// 23.8.)
constexpr int kRowsMax = 16, kRowsMaxK = 6144;
inline bool gemm_rows_pays(int64_t M, int64_t K) { return M <= kRowsMax && K <= kRowsMaxK; }
__attribute__((visibility("hidden"))) void gemm_rows_launch(const void* X, const void* W, void* C, int M, int N, int K, int64_t ldx, int64_t ldw, int64_t ldc,
                                                            const Epilogue& epi, hipStream_t st);
