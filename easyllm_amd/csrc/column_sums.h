// Gradients that are column sums: the kernels that walk over the rows leave fp32 partial rows, one launch adds up to three sets of them.
#pragma once
#include "common.h"

#include "../../include/ezl.h"

struct ColumnSum {
    const float* partials;  // [blocks][n]
    void *bf16, *f32;       // where the sum goes (both null: nowhere)
    int accumulate;
};
inline bool wanted(const ezl_layer_grad* g) { return g && (g->f32 || g->bf16); }
inline ColumnSum column_sum(const float* partials, const ezl_layer_grad* g) {
    if (!wanted(g)) return {partials, nullptr, nullptr, 0};
    return {partials, g->f32 ? nullptr : g->bf16, g->f32, g->f32 && g->accumulate};
}
constexpr int64_t kMaxRows = (1LL << 31) - (1 << 16);  // row numbers are 32-bit, with room for one step past the last
constexpr int64_t kMaxSumColumns = 1LL << 27;                // of the launch that adds them: a block of 1024 threads per 64 columns, fewer than 2^32 threads
constexpr int kColumnSums = 3;
// `count` of them, the rows of each in index order, one after the other where two targets share memory
__attribute__((visibility("hidden"))) int column_sums(const char* name, const ColumnSum* sums, int count, int blocks, int64_t n, hipStream_t stream);
