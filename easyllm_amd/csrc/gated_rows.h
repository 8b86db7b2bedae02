// The products of a gated MLP for a handful of tokens (gated_rows.hip).
#pragma once
#include "gemm_tile.h"

// Rows x K that fit: the tokens lie in LDS, each in whole blocks of 512 elements.
constexpr int kStreamLdsBytes = 147456, kStreamMaxRows = 16;
constexpr int64_t stream_row_elements(int64_t K) { return (K + 511) / 512 * 512 + 8; }
inline bool stream_rows_fit(int64_t M, int64_t K) { return M <= kStreamMaxRows && K < (1 << 17) && M * stream_row_elements(K) * 2 <= kStreamLdsBytes; }
// Whether they beat the tiles (and, alone, gemm_rows.hip).  us of the tiles and of this, weights from HBM, h x f, at 1, 4, 8 and 16 rows: the gate's products
//   256 x 688    3.7, 3.7  3.8, 3.9  3.8, 4.0  3.8, 4.1     768 x 2048  6.6, 4.6  6.6, 5.1  6.6, 5.2  6.7, 5.6     2048 x 5504   13.4, 12.8  13.3, 12.6  13.2, 13.2  13.6, 13.5
//   4096 x 1024  11.6, 8.7  11.8, 9.2  11.8, 9.5  11.9, 12.0  4096 x 11008  42.4, 37.8  40.6, 37.0  40.5, 37.5  41.2, 40.6  5120 x 13696  57.0, 54.3  53.3, 53.6  54.7, 55.2  56.2, 55.7
//   8192 x 3584  34.4, 27.8  31.7, 26.2  31.8, 28.6  32.1, 32.0
// and the down projection, K x N: 5504 x 2048 12.4, 10.3  12.4, 10.8  12.4, 11.8  12.5, 12.7;  11008 x 4096 23.4, 21.6  23.6, 22.7;  13696 x 5120 33.2, 32.9  33.2, 34.9.
// Pairs up to 8 rows: 30 % faster at best, 5 % slower at worst (0.2 us of 256 x 688; 5120 x 13696 1 %).  16 rows would be 16 % faster at 768 x 2048, 8 % slower at 256 x 688, and within 1.5 % elsewhere.
inline bool stream_pairs_pay(int64_t M, int64_t K) { return M <= 8 && stream_rows_fit(M, K); }
inline bool stream_down_pays(int64_t M, int64_t K) { return M * K <= 48 * 1024 && stream_rows_fit(M, K); }
// C[M, cols] = act(X W^T) * (X W2^T), or with W2 null X W^T; all rows on 16 bytes, C contiguous
__attribute__((visibility("hidden"))) void stream_rows_launch(const void* X, const void* W, const void* W2, void* C, const Kept& kept, int M, int cols, int K, int64_t ldx, int64_t ldw, int act,
                                                              hipStream_t st);
