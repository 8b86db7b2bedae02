// The way back through the gate of an MLP as a pass of its own, where no product of the framework's stands in front of it.  HBM-bound: 11 bytes a value.
#include "common.h"
#include "gate.h"

namespace {

constexpr int kGateBlock = 256;

// dgate = d * up * act'(gate), dup = d * act(gate): a workgroup takes a row of four blocks of what was kept, a wave eight rows of two, so that d and the results are read and written in whole
// lines as what was kept is.  Workgroups i, i + 8, i + 16, .. - an XCD's - are neighbours in a stripe of 16 rows: where rows end inside a line, both of its halves come together in one L2.
// 4096 x 11008 in 88 us (5.6 TB/s), 8192 x 2816 46.8, 1531 x 11008 34.8; 15094 x 15336, whose rows end inside lines, 490 (5.2 TB/s; with an XCD's workgroups apart 647, past the caches 750, with a wave on
// one block 963).
template <int ACT>
__global__ __launch_bounds__(kGateBlock) void gate_bwd_kernel(const bf16_t* d_in, const Kept kept, bf16_t* dgate, bf16_t* dup, int64_t M, int f, int across) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = (wave & 1) * 8 + (lane >> 3), col = ((int)(blockIdx.x / 8) % across * 2 + (wave >> 1)) * 2 * kKeptCols + (lane & 7) * 8;
    if (col >= f) return;
    const int stripes = gridDim.x / across;
    for (int64_t rows = (int)(blockIdx.x / 8) / across * 8 + blockIdx.x % 8; rows * kKeptRows + row < M; rows += stripes) {
        const KeptPlace from = kept_place(kept, rows * kKeptRows + row, col);
        const u32x4 kg = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from.upper)), ku = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from.upper + kKeptUp));
        const u32x2 kl = *reinterpret_cast<const u32x2*>(from.low);
        const int64_t at = (rows * kKeptRows + row) * f + col;
        float gate[8], up[8], d[8], dg[8], du[8];
        unpack8(ld_bf16x8(d_in + at), d);
        kept_values<8>({kg[0], kg[1], kg[2], kg[3]}, {ku[0], ku[1], ku[2], ku[3]}, {kl[0], kl[1]}, gate, up);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float y, slope;
            gate_value_slope<ACT>(gate[k], y, slope);
            dg[k] = d[k] * up[k] * slope;
            du[k] = d[k] * y;
        }
        st_bf16x8(dgate + at, pack8(dg));
        st_bf16x8(dup + at, pack8(du));
    }
}

}  // namespace

extern "C" int ezl_gate_bwd(int act, const void* d, const void* kept, void* dgate, void* dup, int64_t M, int64_t f, void* stream) {
    EZL_REQUIRE(act >= EZL_GATE_SILU && act <= EZL_GATE_RELU, EZL_EINVAL, "ezl_gate_bwd: act must be one of EZL_GATE_*");
    EZL_REQUIRE(M >= 0 && f >= 0 && f % 8 == 0 && f < (1LL << 21), EZL_EUNSUPPORTED, "ezl_gate_bwd: the width must be a multiple of 8 below 2^21");
    if (M == 0 || f == 0) return EZL_OK;
    EZL_REQUIRE(d && kept && dgate && dup && ezl_aligned16(d) && ezl_aligned16(kept) && ezl_aligned16(dgate) && ezl_aligned16(dup), EZL_EINVAL, "ezl_gate_bwd: null or misaligned pointer");
    constexpr decltype(&gate_bwd_kernel<0>) kernels[] = {gate_bwd_kernel<0>, gate_bwd_kernel<1>, gate_bwd_kernel<2>, gate_bwd_kernel<3>};
    const Kept from = kept_of(kept, f);
    const int64_t rows = (M + kKeptRows - 1) / kKeptRows;
    const int across = (from.blocks + 3) / 4;  // workgroups of a stripe of 16 rows
    const int64_t most = (1 << 24) / across / 8 * 8, stripes = (rows + 7) / 8 * 8;
    hipLaunchKernelGGL(kernels[act], dim3((unsigned)((stripes < most ? stripes : most) * across)), dim3(kGateBlock), 0, (hipStream_t)stream, (const bf16_t*)d, from, (bf16_t*)dgate, (bf16_t*)dup, M,
                       (int)f, across);
    EZL_LAUNCH_CHECK("ezl_gate_bwd");
    return EZL_OK;
}
