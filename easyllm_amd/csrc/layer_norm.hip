// Layer norm, and either norm behind dropout and the residual sum, forward / backward for gfx950 (HBM-bound).
//
//   s = x, or residual + dropout(x + x_bias)
//   layer norm   xhat = (s - mean) rstd, y = xhat w + b        RMSNorm   xhat = s rstd, y = xhat w
//   ds = rstd (g - [mean(g)] - xhat mean(g xhat)) + dsum, g = dy w;   dw = sum dy xhat, db = sum dy, dx = dropout'(ds), dx_bias = sum dx
//
// A row is held in registers (h <= 8192) and read from HBM once: the variance is of the centred values, not a difference of two large sums.
// y and the statistics are of the fp32 sum; the backward pass has the sum as it was stored, in bf16.
#include "column_sums.h"
#include "dropout.h"

namespace {

constexpr int kMaxH = 8192;

struct NormFwd {
    const bf16_t *x, *x_bias, *res, *w, *b;
    bf16_t *y, *sum;
    float *mean, *rstd;
    int T, h, tpr;
    float eps;
    DropArgs drop;
};

// tpr threads (whole waves) per row, 256 / tpr rows per block; thread t holds the chunks of 8 columns at (c * tpr + t) * 8.
template <int NCHUNK, bool CENTER, bool RES, bool DROP>
__global__ __launch_bounds__(256) void norm_fwd_kernel(const NormFwd a) {
    __shared__ float red[2][4][4];  // [parity][row slot][wave in slot]
    const int tpr = a.tpr, h = a.h;
    const int slot = threadIdx.x / tpr, tin = threadIdx.x % tpr, wis = tin >> 6, nws = tpr >> 6, lane = threadIdx.x & 63;
    const int rpb = 256 / tpr;
    bf16x8 wv[NCHUNK], bv[NCHUNK], xb[NCHUNK];
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
        const int col = (c * tpr + tin) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) bv[c][i] = xb[c][i] = (bf16_t)0.0f;
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
        if (nws > 1) {
            if (lane == 0) red[parity][slot][wis] = v;
            __syncthreads();
            v = 0.f;
            for (int i = 0; i < nws; ++i) v += red[parity][slot][i];
            parity ^= 1;
        }
        return v;
    };
    const float inv_h = 1.0f / (float)h;
    // every thread of the block runs the same number of iterations (barriers inside)
    for (int row0 = blockIdx.x * rpb; row0 < a.T; row0 += gridDim.x * rpb) {
        const int row = row0 + slot;
        const bool live = row < a.T;
        const int64_t base = (int64_t)row * h;
        float v[NCHUNK][8];
        float s1 = 0.f;
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            const int col = (c * tpr + tin) * 8;
            if (live && col < h) {
                unpack8(ld_bf16x8(a.x + base + col), v[c]);
                if constexpr (RES) {
                    float r[8];
                    unpack8(ld_bf16x8(a.res + base + col), r);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[c][i] += (float)xb[c][i];
                    if constexpr (DROP) drop8(v[c], (base + col) >> 3, a.drop, step);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[c][i] += r[i];
                    st_bf16x8(a.sum + base + col, pack8(v[c]));
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) s1 += CENTER ? v[c][i] : v[c][i] * v[c][i];
            }
        }
        s1 = row_sum(s1) * inv_h;
        float mean = 0.f, var = s1;
        if constexpr (CENTER) {
            mean = s1;
            float s2 = 0.f;
#pragma unroll
            for (int c = 0; c < NCHUNK; ++c)
                if (live && (c * tpr + tin) * 8 < h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[c][i] -= mean;
                        s2 += v[c][i] * v[c][i];
                    }
            var = row_sum(s2) * inv_h;
        }
        const float rs = rsqrtf(var + a.eps);
        if (live && tin == 0) {
            a.rstd[row] = rs;
            if (CENTER) a.mean[row] = mean;
        }
#pragma unroll
        for (int c = 0; c < NCHUNK; ++c) {
            const int col = (c * tpr + tin) * 8;
            if (live && col < h) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = v[c][i] * rs * (float)wv[c][i] + (float)bv[c][i];
                st_bf16x8(a.y + base + col, pack8(o));
            }
        }
    }
}

struct NormBwd {
    const bf16_t *dy, *dsum, *s, *w;
    const float *mean, *rstd;
    bf16_t *dx, *dres;
    float *dw, *db, *dxb;  // partial rows
    int T, h;
    bool stream;
    DropArgs drop;
};

// A row is shared by NSPLIT waves: wave part p owns the NCHUNK * 512 columns from p * NCHUNK * 512 on, lane l the 8 columns at l * 8 of each 512.  The
// operands of a wave's next row are loaded before the current row is worked on.  Each wave keeps the column sums of its lanes' columns over the rows it
// visits; the rows of a block are folded through LDS in a fixed order and one partial row per block goes to HBM.
template <int NCHUNK, int NSPLIT, bool CENTER, bool DROP, bool XB>
__global__ __launch_bounds__(256, 2) void norm_bwd_kernel(const NormBwd a) {
    constexpr int RPB = 4 / NSPLIT, NSUMS = 1 + CENTER + XB;
    extern __shared__ float fold[];  // h floats
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
                if (a.dsum) nds[c] = ld_bf16x8_nt(a.dsum + at + c * 512);
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
                    if (a.stream) st_bf16x8_nt(a.dres + at + c * 512, pack8(o));
                    else st_bf16x8(a.dres + at + c * 512, pack8(o));
                    drop8(o, (at + c * 512) >> 3, a.drop, step);
                }
                if constexpr (XB)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[NSUMS - 1][c][i] += o[i];
                if (a.stream) st_bf16x8_nt(a.dx + at + c * 512, pack8(o));
                else st_bf16x8(a.dx + at + c * 512, pack8(o));
            }
        }
    }
    float* const out[3] = {a.dw, CENTER ? a.db : a.dxb, a.dxb};
#pragma unroll
    for (int q = 0; q < NSUMS; ++q) {
        __syncthreads();
        for (int s2 = 0; s2 < RPB; ++s2) {  // row slot 0 stores, the others add in turn
            if (slot == s2) {
#pragma unroll
                for (int c = 0; c < NCHUNK; ++c) {
                    const int col = col0 + c * 512;
                    if (col < h) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (s2 == 0) fold[col + i] = acc[q][c][i];
                            else fold[col + i] += acc[q][c][i];
                        }
                    }
                }
            }
            __syncthreads();
        }
        for (int j = threadIdx.x; j < h; j += 256) out[q][(size_t)blockIdx.x * h + j] = fold[j];
    }
}

constexpr int64_t kBwdBlocks = 512;  // partial rows at most: two blocks per CU

template <bool CENTER, bool RES, bool DROP>
void launch_fwd(int nchunk, unsigned grid, unsigned threads, const NormFwd& a, hipStream_t st) {
    if (nchunk == 1) hipLaunchKernelGGL((norm_fwd_kernel<1, CENTER, RES, DROP>), dim3(grid), dim3(threads), 0, st, a);
    else if (nchunk == 2) hipLaunchKernelGGL((norm_fwd_kernel<2, CENTER, RES, DROP>), dim3(grid), dim3(threads), 0, st, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<4, CENTER, RES, DROP>), dim3(grid), dim3(threads), 0, st, a);
}

int bwd_split(int64_t h) { return h <= 2048 ? 1 : (h <= 4096 ? 2 : 4); }

template <bool CENTER, bool DROP, bool XB>
void launch_bwd(unsigned grid, const NormBwd& a, hipStream_t st) {
    const size_t smem = (size_t)a.h * sizeof(float);
#define EZL_BWD(NC, NS) hipLaunchKernelGGL((norm_bwd_kernel<NC, NS, CENTER, DROP, XB>), dim3(grid), dim3(256), smem, st, a)
    const int split = bwd_split(a.h), nchunk = (a.h + 512 * split - 1) / (512 * split);
    if (split == 1) {
        if (nchunk == 1) EZL_BWD(1, 1);
        else if (nchunk == 2) EZL_BWD(2, 1);
        else EZL_BWD(4, 1);
    } else if (split == 2) {
        if (nchunk == 3) EZL_BWD(3, 2);
        else EZL_BWD(4, 2);
    } else {
        if (nchunk == 3) EZL_BWD(3, 4);
        else EZL_BWD(4, 4);
    }
#undef EZL_BWD
}

}  // namespace

extern "C" int ezl_norm_fwd(int kind, const void* x, const void* x_bias, const void* residual, const ezl_dropout* drop, const void* weight, const void* bias,
                            void* y, void* sum_out, void* mean, void* rstd, int64_t rows, int64_t h, float eps, void* stream) {
    const char* name = "ezl_norm_fwd";
    const bool layer = kind == EZL_LAYER_NORM;
    EZL_REQUIRE(layer || kind == EZL_RMS_NORM, EZL_EINVAL, "%s: kind must be EZL_LAYER_NORM or EZL_RMS_NORM", name);
    EZL_REQUIRE(rows >= 0 && rows < (1LL << 31) && h > 0 && h % 8 == 0 && h <= kMaxH, EZL_EUNSUPPORTED, "%s: need h %% 8 == 0, h <= %d and rows < 2^31 (got %lld x %lld)",
                name, kMaxH, (long long)rows, (long long)h);
    EZL_REQUIRE((residual != nullptr) == (sum_out != nullptr) || rows == 0, EZL_EINVAL, "%s: residual and sum_out go together", name);
    EZL_REQUIRE(residual || (layer && !x_bias && !drop) || rows == 0, EZL_EINVAL, "%s: x_bias, drop and EZL_RMS_NORM need a residual", name);
    EZL_REQUIRE(layer || !bias, EZL_EINVAL, "%s: an RMSNorm has no bias", name);
    EZL_REQUIRE(rows == 0 || (x && weight && y && rstd && (mean || !layer)), EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(ezl_aligned16(x) && ezl_aligned16(x_bias) && ezl_aligned16(residual) && ezl_aligned16(weight) && ezl_aligned16(bias) && ezl_aligned16(y) && ezl_aligned16(sum_out),
                EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    NormFwd a = {(const bf16_t*)x, (const bf16_t*)x_bias, (const bf16_t*)residual, (const bf16_t*)weight, (const bf16_t*)bias, (bf16_t*)y, (bf16_t*)sum_out,
                 (float*)mean, (float*)rstd, (int)rows, (int)h, 0, eps, {}};
    if (const int rc = drop_args(name, drop, a.drop)) return rc;
    if (rows == 0) return EZL_OK;
    hipStream_t st = (hipStream_t)stream;
    int tpr = ((int)h / 8 + 63) / 64 * 64;
    if (tpr > 256) tpr = 256;
    a.tpr = tpr;
    const int nchunk = ((int)h + tpr * 8 - 1) / (tpr * 8), rpb = 256 / tpr;
    int64_t grid = (rows + rpb - 1) / rpb;
    if (grid > 256 * 16) grid = 256 * 16;
    const unsigned threads = (unsigned)(rpb * tpr);  // whole row slots only
    const bool dropping = drop && drop->drop_of_65536 > 0;
    if (layer && !residual) launch_fwd<true, false, false>(nchunk, (unsigned)grid, threads, a, st);
    else if (layer && !dropping) launch_fwd<true, true, false>(nchunk, (unsigned)grid, threads, a, st);
    else if (layer) launch_fwd<true, true, true>(nchunk, (unsigned)grid, threads, a, st);
    else if (!dropping) launch_fwd<false, true, false>(nchunk, (unsigned)grid, threads, a, st);
    else launch_fwd<false, true, true>(nchunk, (unsigned)grid, threads, a, st);
    EZL_LAUNCH_CHECK("ezl_norm_fwd");
    return EZL_OK;
}

extern "C" int64_t ezl_norm_bwd_workspace_bytes(int64_t rows, int64_t h) {
    (void)rows;
    return kColumnSums * kBwdBlocks * h * (int64_t)sizeof(float);
}

extern "C" int ezl_norm_bwd(int kind, const void* dy, const void* dsum, const void* s, const void* weight, const void* mean, const void* rstd,
                            const ezl_dropout* drop, void* dx, void* dresidual, const ezl_layer_grad* dweight, const ezl_layer_grad* dbias,
                            const ezl_layer_grad* dx_bias, void* workspace, int64_t workspace_bytes, int64_t rows, int64_t h, void* stream) {
    const char* name = "ezl_norm_bwd";
    const bool layer = kind == EZL_LAYER_NORM;
    EZL_REQUIRE(layer || kind == EZL_RMS_NORM, EZL_EINVAL, "%s: kind must be EZL_LAYER_NORM or EZL_RMS_NORM", name);
    EZL_REQUIRE(rows >= 0 && rows < (1LL << 31) && h > 0 && h % 8 == 0 && h <= kMaxH, EZL_EUNSUPPORTED, "%s: need h %% 8 == 0, h <= %d and rows < 2^31 (got %lld x %lld)",
                name, kMaxH, (long long)rows, (long long)h);
    EZL_REQUIRE(weight && (rows == 0 || (dy && s && rstd && dx && (mean || !layer))), EZL_EINVAL, "%s: null pointer", name);
    EZL_REQUIRE(wanted(dweight), EZL_EINVAL, "%s: dweight is always written", name);
    EZL_REQUIRE(layer || !wanted(dbias), EZL_EINVAL, "%s: an RMSNorm has no bias", name);
    EZL_REQUIRE((drop != nullptr) == (dresidual != nullptr) || rows == 0, EZL_EINVAL, "%s: drop and dresidual go together", name);
    EZL_REQUIRE(ezl_aligned16(dy) && ezl_aligned16(dsum) && ezl_aligned16(s) && ezl_aligned16(weight) && ezl_aligned16(dx) && ezl_aligned16(dresidual) && ezl_aligned16(workspace),
                EZL_EINVAL, "%s: pointers must be 16-byte aligned", name);
    EZL_REQUIRE(workspace && workspace_bytes >= ezl_norm_bwd_workspace_bytes(rows, h), EZL_EINVAL, "%s: workspace missing or too small", name);
    float* part = (float*)workspace;
    NormBwd a = {(const bf16_t*)dy, (const bf16_t*)dsum, (const bf16_t*)s, (const bf16_t*)weight, (const float*)mean, (const float*)rstd, (bf16_t*)dx,
                 (bf16_t*)dresidual, part, part + kBwdBlocks * h, part + 2 * kBwdBlocks * h, (int)rows, (int)h, false, {}};
    if (const int rc = drop_args(name, drop, a.drop)) return rc;
    a.stream = ezl_streams(rows * h * (drop ? 4 : 2));
    hipStream_t st = (hipStream_t)stream;
    const int rpb = 4 / bwd_split(h);
    int64_t grid = (rows + rpb - 1) / rpb;
    grid = grid > kBwdBlocks ? kBwdBlocks : (grid < 1 ? 1 : grid);  // (no rows still give zero sums)
    const bool xb = wanted(dx_bias);
#define EZL_LAUNCH_BWD(L)                                          \
    do {                                                           \
        if (drop && xb) launch_bwd<L, true, true>((unsigned)grid, a, st);        \
        else if (drop) launch_bwd<L, true, false>((unsigned)grid, a, st);        \
        else if (xb) launch_bwd<L, false, true>((unsigned)grid, a, st);          \
        else launch_bwd<L, false, false>((unsigned)grid, a, st);                 \
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
