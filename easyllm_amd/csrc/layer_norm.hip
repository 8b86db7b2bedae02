// Layer norm, and either norm behind dropout and the residual sum, forward / backward for gfx950 (HBM-bound).
//
//   s = x, or residual + dropout(x + x_bias)
//   layer norm   xhat = (s - mean) rstd, y = xhat w + b        RMSNorm   xhat = s rstd, y = xhat w
//   ds = rstd (g - [mean(g)] - xhat mean(g xhat)) + dsum, g = dy w;   dw = sum dy xhat, db = sum dy, dx = dropout'(ds), dx_bias = sum dx
//
// A row is held in registers (h <= 8192) and read from HBM once: the variance is of the centred values, not a difference of two large sums.
// y and the statistics are of the fp32 sum.  The backward pass has the sum as it was stored, in bf16, and dw's terms dy xhat carry that rounding, |s| rstd 2^-9 at most
// (ds, where xhat enters with a mean over the row only, hardly shows it: 0.0025 at a hundred times below).  dw against 64 bits, norms: 0.0022 to 0.0028 for rows around zero where one rounding
// leaves 0.0017; 0.013 where a row's mean is ten times its spread and 0.10 at a hundred times, as far as a norm of the stored sum would be off in y.  The gradient is that
// of the tensor that the call returned.  (The sum made anew from x, the mask and the residual leaves dw at one rounding everywhere and costs the backward pass a quarter more to read: 16384 x 5120
// 117 -> 146 us, with dropout and a bias 173 -> 206.)
#include "column_sums.h"
#include "dropout.h"

#include <type_traits>

namespace {

constexpr int kMaxH = 8192;

struct NormFwd {
    const bf16_t *x, *x_bias, *res, *w, *b;
    bf16_t *y, *sum;
    float *mean, *rstd;
    int T, h;
    float eps;
    DropArgs drop;
};

// A row is shared by NSPLIT waves: wave part p owns the NCHUNK * 512 columns from p * NCHUNK * 512 on, lane l the 8 columns at l * 8 of each 512.  A
// wave's next row is loaded before the current one is worked on, and where a wave holds whole rows no barrier ties it to others.  Rate of the bytes read and
// written, x + residual -> sum + y, call after call: 16384 x 5120 5.4 TB/s, 8192 x 8192 5.3, 32768 x 1024 6.2; a copy of 2 GiB runs at 5.0.  (Between backward passes of
// the same size 4.5, 150 us with dropout and a bias for 126, while those take 142 us for 173: each finds some of what the other left in the last-level cache.)  (A block per row
// that loads, reduces and stores in turn, up to 512 threads: 4.6, 5.5, 5.9.  Streaming hints on any of the loads or stores: within 1 %.)
template <int NCHUNK, int NSPLIT, bool CENTER, bool RES, bool DROP>
__global__ __launch_bounds__(256) void norm_fwd_kernel(const NormFwd a) {
    constexpr int RPB = 4 / NSPLIT;
    __shared__ float cell[2][RPB][NSPLIT];
    const int lane = threadIdx.x & 63, h = a.h;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = wave / NSPLIT, part = wave % NSPLIT;
    const int col0 = (part * NCHUNK * 64 + lane) * 8;
    bf16x8 wv[NCHUNK], bv[NCHUNK], xb[NCHUNK];
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
        const int col = col0 + c * 512;
#pragma unroll
        for (int i = 0; i < 8; ++i) wv[c][i] = bv[c][i] = xb[c][i] = (bf16_t)0.0f;
        if (col < h) {
            wv[c] = ld_bf16x8(a.w + col);
            if (CENTER && a.b) bv[c] = ld_bf16x8(a.b + col);
            if (RES && a.x_bias) xb[c] = ld_bf16x8(a.x_bias + col);
        }
    }
    uint32_t step = 0;
    if constexpr (DROP) step = drop_step(a.drop);
    int parity = 0;
    auto row_sum = [&](float v) {
        v = wave_sum(v);
        if constexpr (NSPLIT > 1) {
            if (lane == 0) cell[parity][slot][part] = v;
            __syncthreads();
            v = cell[parity][slot][0];
#pragma unroll
            for (int q = 1; q < NSPLIT; ++q) v += cell[parity][slot][q];
            parity ^= 1;
        }
        return v;
    };
    const float inv_h = 1.0f / (float)h;
    bf16x8 nx[NCHUNK], nr[NCHUNK];
    auto fetch = [&](int row) {
        const int64_t at = (int64_t)row * h + col0;
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) nx[c][i] = nr[c][i] = (bf16_t)0.0f;
            if (row < a.T && col0 + c * 512 < h) {
                nx[c] = ld_bf16x8(a.x + at + c * 512);
                if (RES) nr[c] = ld_bf16x8(a.res + at + c * 512);
            }
        }
    };
    fetch(blockIdx.x * RPB + slot);
    for (int row0 = blockIdx.x * RPB; row0 < a.T; row0 += gridDim.x * RPB) {
        const int row = row0 + slot;
        const bool live = row < a.T;
        const int64_t at = (int64_t)row * h + col0;
        bf16x8 x[NCHUNK], r[NCHUNK];
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            x[c] = nx[c];
            r[c] = nr[c];
        }
        if (row0 + (int)gridDim.x * RPB < a.T) fetch(row + gridDim.x * RPB);
        float v[NCHUNK][8];
        float s1 = 0.f;
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            unpack8(x[c], v[c]);
            if constexpr (RES) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += (float)xb[c][i];
                if constexpr (DROP) drop8(v[c], (at + c * 512) >> 3, a.drop, step);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += (float)r[c][i];
                if (live && col0 + c * 512 < h) st_bf16x8(a.sum + at + c * 512, pack8(v[c]));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s1 += CENTER ? v[c][i] : v[c][i] * v[c][i];
        }
        s1 = row_sum(s1) * inv_h;
        float mean = 0.f, var = s1;
        if constexpr (CENTER) {
            mean = s1;
            float s2 = 0.f;
#pragma unroll
            for (int c = 0; c < NCHUNK; ++c)
                if (col0 + c * 512 < h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[c][i] -= mean;
                        s2 += v[c][i] * v[c][i];
                    }
            var = row_sum(s2) * inv_h;
        }
        const float rs = rsqrtf(var + a.eps);
        if (live && part == 0 && lane == 0) {
            a.rstd[row] = rs;
            if (CENTER) a.mean[row] = mean;
        }
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c)
            if (live && col0 + c * 512 < h) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = v[c][i] * rs * (float)wv[c][i] + (float)bv[c][i];
                st_bf16x8(a.y + at + c * 512, pack8(o));
            }
    }
}

struct NormBwd {
    const bf16_t *dy, *dsum, *s, *w;
    const float *mean, *rstd;
    bf16_t *dx, *dres;
    float *dw, *db, *dxb;  // partial rows
    int T, h;
    DropArgs drop;
};

// Rows, columns and loads ahead as in the forward kernel.  Each wave keeps the column sums of its lanes' columns over the rows it
// visits; the waves of a block that hold the same columns are added through LDS in a fixed order and one partial row per block goes to HBM.
template <int NCHUNK, int NSPLIT, bool CENTER, bool DROP, bool XB>
__global__ __launch_bounds__(256, 2) void norm_bwd_kernel(const NormBwd a) {
    constexpr int RPB = 4 / NSPLIT, NSUMS = 1 + CENTER + XB;
    constexpr bool AHEAD = NCHUNK < 4 || NSUMS < 3;  // dsum is loaded a row ahead too, where the registers hold it
    extern __shared__ float fold[];  // RPB rows of h
    __shared__ float cell[2][RPB][NSPLIT][2];  // [parity][row slot][part]
    const int lane = threadIdx.x & 63, h = a.h;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = wave / NSPLIT, part = wave % NSPLIT;
    const int col0 = (part * NCHUNK * 64 + lane) * 8;
    bf16x8 wr[NCHUNK];
    float acc[NSUMS][NCHUNK][8];
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
        const int col = col0 + c * 512;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            wr[c][i] = (bf16_t)0.0f;
#pragma unroll
            for (int q = 0; q < NSUMS; ++q) acc[q][c][i] = 0.f;
        }
        if (col < h) wr[c] = ld_bf16x8(a.w + col);
    }
    uint32_t step = 0;
    if constexpr (DROP) step = drop_step(a.drop);
    const float inv_h = 1.0f / (float)h;
    int parity = 0;
    bf16x8 ns[NCHUNK], ndy[NCHUNK], nds[NCHUNK];
    float nrs = 0.f, nmean = 0.f;
    auto fetch = [&](int row) {
        const bool live = row < a.T;
        const int64_t at = (int64_t)row * h + col0;
        nrs = live ? a.rstd[row] : 0.f;
        if (CENTER) nmean = live ? a.mean[row] : 0.f;
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) ns[c][i] = ndy[c][i] = nds[c][i] = (bf16_t)0.0f;
            if (live && col0 + c * 512 < h) {
                ns[c] = ld_bf16x8_nt(a.s + at + c * 512);
                ndy[c] = ld_bf16x8_nt(a.dy + at + c * 512);
                if (AHEAD && a.dsum) nds[c] = ld_bf16x8_nt(a.dsum + at + c * 512);
            }
        }
    };
    fetch(blockIdx.x * RPB + slot);
    for (int row0 = blockIdx.x * RPB; row0 < a.T; row0 += gridDim.x * RPB) {
        const int row = row0 + slot;
        const bool live = row < a.T;
        bf16x8 sr[NCHUNK], dyr[NCHUNK], dsr[NCHUNK];
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            sr[c] = ns[c];
            dyr[c] = ndy[c];
            dsr[c] = nds[c];
            if (!AHEAD && a.dsum && live && col0 + c * 512 < h) dsr[c] = ld_bf16x8_nt(a.dsum + (int64_t)row * h + col0 + c * 512);
        }
        const float rs = nrs, mean = nmean;
        if (row0 + (int)gridDim.x * RPB < a.T) fetch(row + gridDim.x * RPB);
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float g = (float)dyr[c][i] * (float)wr[c][i];
                d2 += g * (((float)sr[c][i] - mean) * rs);
                if (CENTER) d1 += g;
            }
        d2 = wave_sum(d2);
        if (CENTER) d1 = wave_sum(d1);
        if constexpr (NSPLIT > 1) {
            if (lane == 0) {
                cell[parity][slot][part][0] = d2;
                cell[parity][slot][part][1] = d1;
            }
            __syncthreads();
            d2 = cell[parity][slot][0][0];
            d1 = cell[parity][slot][0][1];
#pragma unroll
            for (int q = 1; q < NSPLIT; ++q) {  // the same order in every wave of the row
                d2 += cell[parity][slot][q][0];
                d1 += cell[parity][slot][q][1];
            }
            parity ^= 1;
        }
        const float m2 = d2 * inv_h, m1 = CENTER ? d1 * inv_h : 0.f;
        const int64_t at = (int64_t)row * h + col0;
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            // opaque: the fp32 copies made for the sums above must not be kept alive (they would not fit)
            asm volatile("" : "+v"(sr[c]), "+v"(dyr[c]));
            if (live && col0 + c * 512 < h) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float xhat = ((float)sr[c][i] - mean) * rs, dyv = (float)dyr[c][i];
                    o[i] = rs * (dyv * (float)wr[c][i] - m1 - xhat * m2) + (float)dsr[c][i];
                    acc[0][c][i] += dyv * xhat;
                    if constexpr (CENTER) acc[1][c][i] += dyv;
                }
                if constexpr (DROP) {
                    st_bf16x8(a.dres + at + c * 512, pack8(o));
                    drop8(o, (at + c * 512) >> 3, a.drop, step);
                }
                if constexpr (XB)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[NSUMS - 1][c][i] += o[i];
                st_bf16x8(a.dx + at + c * 512, pack8(o));
            }
        }
    }
    float* const out[3] = {a.dw, CENTER ? a.db : a.dxb, a.dxb};
#pragma unroll
    for (int q = 0; q < NSUMS; ++q) {
        float* const dst = RPB > 1 ? fold + slot * h : out[q] + (int64_t)blockIdx.x * h;  // (a block of one row: its waves' columns are apart)
        if (RPB > 1 && q > 0) __syncthreads();
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            const int col = col0 + c * 512;
            if (col < h)
#pragma unroll
                for (int k = 0; k < 8; k += 4) *reinterpret_cast<f32x4*>(dst + col + k) = f32x4{acc[q][c][k], acc[q][c][k + 1], acc[q][c][k + 2], acc[q][c][k + 3]};
        }
        if constexpr (RPB > 1) {
            __syncthreads();
            for (int j = threadIdx.x * 4; j < h; j += 1024) {
                f32x4 v = *reinterpret_cast<const f32x4*>(fold + j);
#pragma unroll
                for (int s2 = 1; s2 < RPB; ++s2) v += *reinterpret_cast<const f32x4*>(fold + s2 * h + j);
                *reinterpret_cast<f32x4*>(out[q] + (int64_t)blockIdx.x * h + j) = v;
            }
        }
    }
}

constexpr int64_t kFwdBlocks = 4096, kBwdBlocks = 512;  // at most

// waves that share a row, and with it rows of a block of four
int split_of(int64_t h) { return h <= 2048 ? 1 : (h <= 4096 ? 2 : 4); }

// launch(NCHUNK, NSPLIT) for rows of h
template <class L>
void by_width(int64_t h, L&& launch) {
    const int split = split_of(h), nchunk = ((int)h + 512 * split - 1) / (512 * split);
    typedef std::integral_constant<int, 1> one;
    typedef std::integral_constant<int, 2> two;
    typedef std::integral_constant<int, 3> three;
    typedef std::integral_constant<int, 4> four;
    if (split == 1 && nchunk == 1) launch(one{}, one{});
    else if (split == 1 && nchunk == 2) launch(two{}, one{});
    else if (split == 1 && nchunk == 3) launch(three{}, one{});
    else if (split == 1) launch(four{}, one{});
    else if (split == 2 && nchunk == 3) launch(three{}, two{});
    else if (split == 2) launch(four{}, two{});
    else if (nchunk == 3) launch(three{}, four{});
    else launch(four{}, four{});
}
unsigned blocks_for(int64_t rows, int64_t h, int64_t most) {
    const int rpb = 4 / split_of(h);
    const int64_t blocks = (rows + rpb - 1) / rpb;
    return (unsigned)(blocks > most ? most : (blocks < 1 ? 1 : blocks));
}

// Every block leaves partial rows of h floats, which few rows feel, and wide ones, which cost most per block; the others gain by two blocks per CU.  256
// against 512, us: 1167 x 1000 9.1, 9.6; 4000 x 2048 20.7, 21.6 (with dropout and a bias 26.1, 27.2); 8000 x 2048 30.8, 29.9; 2048 x 4096 22.5, 24.4; 4096 x 5120 42.6,
// 39.3; 16384 x 5120 138, 116; 32768 x 1024 50.5, 48.9 (67.5, 63.0); 4096 x 8192 53.0, 56.0; 8192 x 8192 91.8, 95.7.
unsigned bwd_blocks(int64_t rows, int64_t h) {
    const bool few = rows * split_of(h) <= 8192 || h > 6144;
    return blocks_for(rows, h, few ? kBwdBlocks / 2 : kBwdBlocks);  // (no rows still give zero sums)
}

template <bool CENTER, bool RES, bool DROP>
void launch_fwd(const NormFwd& a, hipStream_t st) {
    by_width(a.h, [&](auto nc, auto ns) {
        hipLaunchKernelGGL((norm_fwd_kernel<decltype(nc)::value, decltype(ns)::value, CENTER, RES, DROP>), dim3(blocks_for(a.T, a.h, kFwdBlocks)), dim3(256), 0, st, a);
    });
}
template <bool CENTER, bool DROP, bool XB>
void launch_bwd(unsigned grid, const NormBwd& a, hipStream_t st) {
    by_width(a.h, [&](auto nc, auto ns) {
        hipLaunchKernelGGL((norm_bwd_kernel<decltype(nc)::value, decltype(ns)::value, CENTER, DROP, XB>), dim3(grid), dim3(256),
                           decltype(ns)::value == 4 ? 0 : (size_t)a.h * (4 / decltype(ns)::value) * sizeof(float), st, a);
    });
}

}  // namespace

extern "C" int ezl_norm_fwd(int kind, const void* x, const void* x_bias, const void* residual, const ezl_dropout* drop, const void* weight, const void* bias,
                            void* y, void* sum_out, void* mean, void* rstd, int64_t rows, int64_t h, float eps, void* stream) {
    const char* name = "ezl_norm_fwd";
    const bool layer = kind == EZL_LAYER_NORM;
    EZL_REQUIRE(layer || kind == EZL_RMS_NORM, EZL_EINVAL, "%s: kind must be EZL_LAYER_NORM or EZL_RMS_NORM", name);
    EZL_REQUIRE(rows >= 0 && rows <= kMaxRows && h > 0 && h % 8 == 0 && h <= kMaxH, EZL_EUNSUPPORTED, "%s: need h %% 8 == 0, h <= %d and rows <= %lld (got %lld x %lld)",
                name, kMaxH, (long long)kMaxRows, (long long)rows, (long long)h);
    EZL_REQUIRE((residual != nullptr) == (sum_out != nullptr) || rows == 0, EZL_EINVAL, "%s: residual and sum_out go together", name);
    EZL_REQUIRE(residual || (layer && !x_bias && !drop) || rows == 0, EZL_EINVAL, "%s: x_bias, drop and EZL_RMS_NORM need a residual", name);
    EZL_REQUIRE(layer || !bias, EZL_EINVAL, "%s: an RMSNorm has no bias", name);
    EZL_REQUIRE(rows == 0 || (x && weight && y && rstd && (mean || !layer)), EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(ezl_aligned16(x) && ezl_aligned16(x_bias) && ezl_aligned16(residual) && ezl_aligned16(weight) && ezl_aligned16(bias) && ezl_aligned16(y) && ezl_aligned16(sum_out),
                EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    NormFwd a = {(const bf16_t*)x, (const bf16_t*)x_bias, (const bf16_t*)residual, (const bf16_t*)weight, (const bf16_t*)bias, (bf16_t*)y, (bf16_t*)sum_out,
                 (float*)mean, (float*)rstd, (int)rows, (int)h, eps, {}};
    if (const int rc = drop_args(name, drop, a.drop)) return rc;
    if (rows == 0) return EZL_OK;
    hipStream_t st = (hipStream_t)stream;
    const bool dropping = drop && drop->drop_of_65536 > 0;
    if (layer && !residual) launch_fwd<true, false, false>(a, st);
    else if (layer && !dropping) launch_fwd<true, true, false>(a, st);
    else if (layer) launch_fwd<true, true, true>(a, st);
    else if (!dropping) launch_fwd<false, true, false>(a, st);
    else launch_fwd<false, true, true>(a, st);
    EZL_LAUNCH_CHECK("ezl_norm_fwd");
    return EZL_OK;
}

extern "C" int64_t ezl_norm_bwd_workspace_bytes(int64_t rows, int64_t h) {
    return rows < 0 || h <= 0 ? 0 : kColumnSums * bwd_blocks(rows, h) * h * (int64_t)sizeof(float);
}

extern "C" int ezl_norm_bwd(int kind, const void* dy, const void* dsum, const void* s, const void* weight, const void* mean, const void* rstd,
                            const ezl_dropout* drop, void* dx, void* dresidual, const ezl_layer_grad* dweight, const ezl_layer_grad* dbias,
                            const ezl_layer_grad* dx_bias, void* workspace, int64_t workspace_bytes, int64_t rows, int64_t h, void* stream) {
    const char* name = "ezl_norm_bwd";
    const bool layer = kind == EZL_LAYER_NORM;
    EZL_REQUIRE(layer || kind == EZL_RMS_NORM, EZL_EINVAL, "%s: kind must be EZL_LAYER_NORM or EZL_RMS_NORM", name);
    EZL_REQUIRE(rows >= 0 && rows <= kMaxRows && h > 0 && h % 8 == 0 && h <= kMaxH, EZL_EUNSUPPORTED, "%s: need h %% 8 == 0, h <= %d and rows <= %lld (got %lld x %lld)",
                name, kMaxH, (long long)kMaxRows, (long long)rows, (long long)h);
    EZL_REQUIRE(weight && (rows == 0 || (dy && s && rstd && dx && (mean || !layer))), EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(wanted(dweight), EZL_EINVAL, "%s: dweight is always written", name);
    EZL_REQUIRE(layer || !wanted(dbias), EZL_EINVAL, "%s: an RMSNorm has no bias", name);
    EZL_REQUIRE((drop != nullptr) == (dresidual != nullptr) || rows == 0, EZL_EINVAL, "%s: drop and dresidual go together", name);
    EZL_REQUIRE(ezl_aligned16(dy) && ezl_aligned16(dsum) && ezl_aligned16(s) && ezl_aligned16(weight) && ezl_aligned16(dx) && ezl_aligned16(dresidual) && ezl_aligned16(workspace),
                EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    EZL_REQUIRE(workspace && workspace_bytes >= ezl_norm_bwd_workspace_bytes(rows, h), EZL_EINVAL, "%s: workspace missing or too small", name);
    const unsigned grid = bwd_blocks(rows, h);
    const int64_t set = grid * h;  // partial rows of one sum
    float* part = (float*)workspace;
    NormBwd a = {(const bf16_t*)dy, (const bf16_t*)dsum, (const bf16_t*)s, (const bf16_t*)weight, (const float*)mean, (const float*)rstd, (bf16_t*)dx,
                 (bf16_t*)dresidual, part, part + set, part + 2 * set, (int)rows, (int)h, {}};
    if (const int rc = drop_args(name, drop, a.drop)) return rc;
    hipStream_t st = (hipStream_t)stream;
    const bool xb = wanted(dx_bias);
#define EZL_LAUNCH_BWD(L)                                          \
    do {                                                           \
        if (drop && xb) launch_bwd<L, true, true>(grid, a, st);        \
        else if (drop) launch_bwd<L, true, false>(grid, a, st);        \
        else if (xb) launch_bwd<L, false, true>(grid, a, st);          \
        else launch_bwd<L, false, false>(grid, a, st);                 \
    } while (0)
    if (layer) EZL_LAUNCH_BWD(true);
    else EZL_LAUNCH_BWD(false);
#undef EZL_LAUNCH_BWD
    EZL_LAUNCH_CHECK("ezl_norm_bwd");
    ColumnSum sums[kColumnSums];
    int count = 0;
    sums[count++] = column_sum(a.dw, dweight);
    if (wanted(dbias)) sums[count++] = column_sum(a.db, dbias);
    if (xb) sums[count++] = column_sum(a.dxb, dx_bias);
    return column_sums(name, sums, count, (int)grid, h, st);
}
