// Dropout with bias and residual sum, the backward passes of it and of the activations, and their column sums (HBM-bound).
//
//   out = residual + dropout(x + bias);   dx = dropout'(dy), dbias = sum over rows of dx;   dpre = dy act'(pre), dbias = sum over rows of dpre
//
// Each byte moves once: 8192 x 8192 with bias and residual forward 73.5 us (5.5 TB/s; a copy of 2 GiB runs at 5.0), backward with the bias's gradient 47.0 (5.7, the launch
// that adds the partial rows included), without 43.0 (6.2).
#include "activation.h"
#include "column_sums.h"
#include "dropout.h"

namespace {

struct DropAdd {
    const bf16_t *x, *bias, *res;
    bf16_t* out;
    int64_t groups;  // of 8 elements
    int cols8;       // groups of a row
    DropArgs drop;
};

// A thread takes every gridDim.x * 256-th group of 8 elements; its column advances with it.
template <bool DROP, bool BIAS>
__global__ __launch_bounds__(256) void dropout_add_kernel(const DropAdd a) {
    const int64_t stride = (int64_t)gridDim.x * 256;
    int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int col = 0, col_step = 0;
    if constexpr (BIAS) {
        col = (int)(g % a.cols8);
        col_step = (int)(stride % a.cols8);
    }
    uint32_t step = 0;
    if constexpr (DROP) step = drop_step(a.drop);
    for (; g < a.groups; g += stride) {
        float v[8];
        unpack8(ld_bf16x8(a.x + g * 8), v);
        float r[8];
        if (a.res) unpack8(ld_bf16x8(a.res + g * 8), r);
        if constexpr (BIAS) {
            float b[8];
            unpack8(ld_bf16x8(a.bias + col * 8), b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += b[i];
            col += col_step;
            if (col >= a.cols8) col -= a.cols8;
        }
        if constexpr (DROP) drop8(v, g, a.drop, step);
        if (a.res)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += r[i];
        st_bf16x8(a.out + g * 8, pack8(v));
    }
}

// dx = f(dy) with the column sums of f(dy) before rounding: a block owns 512 columns (64 lanes of 8) and every gridDim.y * 4-th row from its four
// waves' on, and leaves one partial row of them.
constexpr int kSumBlocks = 256;  // partial rows at most
struct DropSum {
    const bf16_t* dy;
    bf16_t* dx;
    float* partial;
    int rows, n;
    DropArgs drop;
};
template <class F>
__device__ __forceinline__ void rows_with_column_sums(int rows, int n, float* partial, F&& f) {
    __shared__ float fold[4][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = (blockIdx.x * 64 + lane) * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (col < n)
        for (int row = blockIdx.y * 4 + wave; row < rows; row += gridDim.y * 4) {
            float v[8];
            f((int64_t)row * n + col, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += v[i];
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) fold[wave][lane * 8 + i] = acc[i];
    __syncthreads();
    for (int j = threadIdx.x; j < 512; j += 256)
        if (blockIdx.x * 512 + j < n) partial[(int64_t)blockIdx.y * n + blockIdx.x * 512 + j] = fold[0][j] + fold[1][j] + fold[2][j] + fold[3][j];
}
template <bool DROP>
__global__ __launch_bounds__(256) void dropout_sum_kernel(const DropSum a) {
    uint32_t step = 0;
    if constexpr (DROP) step = drop_step(a.drop);
    rows_with_column_sums(a.rows, a.n, a.partial, [&](int64_t at, float (&v)[8]) {
        unpack8(ld_bf16x8(a.dy + at), v);
        if constexpr (DROP) {
            drop8(v, at >> 3, a.drop, step);
            st_bf16x8(a.dx + at, pack8(v));
        }
    });
}

// pre is kept in bf16 (half the bytes of fp32; its rounding moves the slope, and shows in the bias's gradient: 0.0018 off 64 bits where one rounding leaves 0.0017, norms of
// 1531 x 4096 x 11008) and dpre is written in bf16, the operand of both gradients' products: dx and dW are two roundings off, 0.0024.  The bias's gradient is summed before dpre is rounded.
struct ActBwd {
    const bf16_t *dy, *pre;
    bf16_t* dpre;
    float* partial;
    int64_t groups;  // of 8 elements
    int rows, n;
};
template <int ACT>
__device__ __forceinline__ void act_bwd8(const ActBwd& a, int64_t at, float (&v)[8]) {
    float p[8];
    unpack8(ld_bf16x8(a.dy + at), v);
    unpack8(ld_bf16x8(a.pre + at), p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= activation_slope(p[i], ACT);
    st_bf16x8(a.dpre + at, pack8(v));
}
template <int ACT, bool SUMS>
__global__ __launch_bounds__(256) void act_bwd_kernel(const ActBwd a) {
    if constexpr (SUMS) {
        rows_with_column_sums(a.rows, a.n, a.partial, [&](int64_t at, float (&v)[8]) { act_bwd8<ACT>(a, at, v); });
    } else {
        for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < a.groups; g += (int64_t)gridDim.x * 256) {
            float v[8];
            act_bwd8<ACT>(a, g * 8, v);
        }
    }
}

struct SumsArgs {
    ColumnSum s[kColumnSums];
};
__global__ __launch_bounds__(kColsumThreads) void column_sums_kernel(const SumsArgs a, int blocks, int n) {
    const ColumnSum s = a.s[blockIdx.y];
    ezl_colsum(s.partials, blocks, n, (bf16_t*)s.bf16, (float*)s.f32, s.accumulate);
}

dim3 sum_grid(int64_t rows, int64_t n) {
    const int64_t slabs = (n + 511) / 512;
    int64_t segs = (2048 + slabs - 1) / slabs;
    const int64_t most = (rows + 3) / 4;
    segs = segs > kSumBlocks ? kSumBlocks : segs;
    segs = segs > most ? most : segs;
    return dim3((unsigned)slabs, (unsigned)(segs < 1 ? 1 : segs));
}
unsigned elementwise_grid(int64_t groups) {
    const int64_t g = (groups + 255) / 256;
    return (unsigned)(g > 256 * 16 ? 256 * 16 : g);
}
int sizes_check(const char* name, int64_t rows, int64_t n) {
    EZL_REQUIRE(rows >= 0 && rows <= kMaxRows && n > 0 && n % 8 == 0 && n <= kMaxRows && (rows == 0 || n <= (1LL << 60) / rows), EZL_EUNSUPPORTED,
                "%s: need n %% 8 == 0, rows and n <= %lld (got %lld x %lld)", name, (long long)kMaxRows, (long long)rows, (long long)n);
    return EZL_OK;
}

}  // namespace

int column_sums(const char* name, const ColumnSum* sums, int count, int blocks, int64_t n, hipStream_t stream) {
    // (one parameter in two places has one buffer, which is overwritten first and added to then)
    for (int i = 1; i < count; ++i)
        for (int j = 0; j < i; ++j)
            if (sums[i].f32 && sums[j].f32 && (char*)sums[i].f32 < (char*)sums[j].f32 + 4 * n && (char*)sums[j].f32 < (char*)sums[i].f32 + 4 * n) {
                for (int k = 0; k < count; ++k)
                    if (const int rc = column_sums(name, sums + k, 1, blocks, n, stream)) return rc;
                return EZL_OK;
            }
    SumsArgs a = {};
    for (int i = 0; i < count; ++i) a.s[i] = sums[i];
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((n + 63) / 64), (unsigned)count), dim3(kColsumThreads), 0, stream, a, blocks, (int)n);
    EZL_LAUNCH_CHECK(name);
    return EZL_OK;
}

extern "C" int ezl_dropout_add_fwd(const void* x, const void* bias, const void* residual, const ezl_dropout* drop, void* out, int64_t rows, int64_t n,
                                   void* stream) {
    const char* name = "ezl_dropout_add_fwd";
    if (const int rc = sizes_check(name, rows, n)) return rc;
    EZL_REQUIRE(rows == 0 || (x && out), EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(ezl_aligned16(x) && ezl_aligned16(bias) && ezl_aligned16(residual) && ezl_aligned16(out), EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    DropAdd a = {(const bf16_t*)x, (const bf16_t*)bias, (const bf16_t*)residual, (bf16_t*)out, rows * (n / 8), (int)(n / 8), {}};
    if (const int rc = drop_args(name, drop, a.drop)) return rc;
    if (rows == 0) return EZL_OK;
    const dim3 grid(elementwise_grid(a.groups));
    hipStream_t st = (hipStream_t)stream;
    if (a.drop.threshold && bias) hipLaunchKernelGGL((dropout_add_kernel<true, true>), grid, dim3(256), 0, st, a);
    else if (a.drop.threshold) hipLaunchKernelGGL((dropout_add_kernel<true, false>), grid, dim3(256), 0, st, a);
    else if (bias) hipLaunchKernelGGL((dropout_add_kernel<false, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((dropout_add_kernel<false, false>), grid, dim3(256), 0, st, a);
    EZL_LAUNCH_CHECK("ezl_dropout_add_fwd");
    return EZL_OK;
}

extern "C" int64_t ezl_column_sum_workspace_bytes(int64_t rows, int64_t n) {
    return rows < 0 || n <= 0 ? 0 : (int64_t)sum_grid(rows, n).y * n * (int64_t)sizeof(float);
}

extern "C" int ezl_dropout_add_bwd(const void* dy, const ezl_dropout* drop, void* dx, const ezl_layer_grad* dbias, void* workspace, int64_t workspace_bytes,
                                   int64_t rows, int64_t n, void* stream) {
    const char* name = "ezl_dropout_add_bwd";
    if (const int rc = sizes_check(name, rows, n)) return rc;
    EZL_REQUIRE(rows == 0 || (dy && (dx != nullptr) == (drop != nullptr)), EZL_EINVAL, "%s: null pointer, or a dx without drop", name);
    EZL_REQUIRE(drop || wanted(dbias), EZL_EINVAL, "%s: nothing to do", name);
    EZL_REQUIRE(ezl_aligned16(dy) && ezl_aligned16(dx) && ezl_aligned16(workspace), EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    DropArgs d;
    if (const int rc = drop_args(name, drop, d)) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (!wanted(dbias)) {
        if (rows == 0) return EZL_OK;
        const DropAdd a = {(const bf16_t*)dy, nullptr, nullptr, (bf16_t*)dx, rows * (n / 8), (int)(n / 8), d};
        hipLaunchKernelGGL((dropout_add_kernel<true, false>), dim3(elementwise_grid(a.groups)), dim3(256), 0, st, a);
        EZL_LAUNCH_CHECK("ezl_dropout_add_bwd");
        return EZL_OK;
    }
    EZL_REQUIRE(n <= kMaxSumColumns, EZL_EUNSUPPORTED, "%s: column sums of n <= %lld (got %lld)", name, (long long)kMaxSumColumns, (long long)n);
    EZL_REQUIRE(workspace && workspace_bytes >= ezl_column_sum_workspace_bytes(rows, n), EZL_EINVAL, "%s: workspace missing or too small", name);
    const DropSum a = {(const bf16_t*)dy, (bf16_t*)dx, (float*)workspace, (int)rows, (int)n, d};
    const dim3 grid = sum_grid(rows, n);
    if (drop) hipLaunchKernelGGL(dropout_sum_kernel<true>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(dropout_sum_kernel<false>, grid, dim3(256), 0, st, a);
    EZL_LAUNCH_CHECK("ezl_dropout_add_bwd");
    const ColumnSum s = column_sum((const float*)workspace, dbias);
    return column_sums(name, &s, 1, (int)grid.y, n, st);
}

extern "C" int ezl_act_bwd(int act, const void* dy, const void* pre, void* dpre, const ezl_layer_grad* dbias, void* workspace, int64_t workspace_bytes,
                           int64_t rows, int64_t n, void* stream) {
    const char* name = "ezl_act_bwd";
    EZL_REQUIRE(act == kActGelu || act == kActGeluTanh, EZL_EINVAL, "%s: act must be EZL_ACT_GELU or EZL_ACT_GELU_TANH", name);
    if (const int rc = sizes_check(name, rows, n)) return rc;
    EZL_REQUIRE(rows == 0 || (dy && pre && dpre), EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(ezl_aligned16(dy) && ezl_aligned16(pre) && ezl_aligned16(dpre) && ezl_aligned16(workspace), EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    hipStream_t st = (hipStream_t)stream;
    const ActBwd a = {(const bf16_t*)dy, (const bf16_t*)pre, (bf16_t*)dpre, (float*)workspace, rows * (n / 8), (int)rows, (int)n};
    if (!wanted(dbias)) {
        if (rows == 0) return EZL_OK;
        const dim3 grid(elementwise_grid(a.groups));
        if (act == kActGelu) hipLaunchKernelGGL((act_bwd_kernel<kActGelu, false>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((act_bwd_kernel<kActGeluTanh, false>), grid, dim3(256), 0, st, a);
        EZL_LAUNCH_CHECK("ezl_act_bwd");
        return EZL_OK;
    }
    EZL_REQUIRE(n <= kMaxSumColumns, EZL_EUNSUPPORTED, "%s: column sums of n <= %lld (got %lld)", name, (long long)kMaxSumColumns, (long long)n);
    EZL_REQUIRE(workspace && workspace_bytes >= ezl_column_sum_workspace_bytes(rows, n), EZL_EINVAL, "%s: workspace missing or too small", name);
    const dim3 grid = sum_grid(rows, n);
    if (act == kActGelu) hipLaunchKernelGGL((act_bwd_kernel<kActGelu, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((act_bwd_kernel<kActGeluTanh, true>), grid, dim3(256), 0, st, a);
    EZL_LAUNCH_CHECK("ezl_act_bwd");
    const ColumnSum s = column_sum((const float*)workspace, dbias);
    return column_sums(name, &s, 1, (int)grid.y, n, st);
}
