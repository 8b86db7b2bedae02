// The gate of an MLP as passes of their own: out = act(gate) * up and its backward, HBM-bound.
#include "common.h"
#include "gate.h"

namespace {

constexpr int kGateBlock = 256;

template <int ACT>
__global__ __launch_bounds__(kGateBlock) void gate_fwd_kernel(const bf16_t* __restrict__ gate, const bf16_t* __restrict__ up, bf16_t* __restrict__ out, int64_t n8) {
    for (int64_t i = (int64_t)blockIdx.x * kGateBlock + threadIdx.x; i < n8; i += (int64_t)gridDim.x * kGateBlock) {
        float g[8], u[8], o[8];
        unpack8(ld_bf16x8_nt(gate + i * 8), g);
        unpack8(ld_bf16x8_nt(up + i * 8), u);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = gate_value<ACT>(g[k]) * u[k];
        st_bf16x8(out + i * 8, pack8(o));
    }
}

// dgate = dout * up * act'(gate), dup = dout * act(gate); out, if given, once more
template <int ACT, bool STREAM>
__global__ __launch_bounds__(kGateBlock) void gate_bwd_kernel(const bf16_t* __restrict__ dout, const bf16_t* __restrict__ gate, const bf16_t* __restrict__ up,
                                                              bf16_t* __restrict__ dgate, bf16_t* __restrict__ dup, bf16_t* __restrict__ out, int64_t n8) {
    for (int64_t i = (int64_t)blockIdx.x * kGateBlock + threadIdx.x; i < n8; i += (int64_t)gridDim.x * kGateBlock) {
        float g[8], u[8], d[8], dg[8], du[8], o[8];
        unpack8(ld_bf16x8_nt(gate + i * 8), g);
        unpack8(ld_bf16x8_nt(up + i * 8), u);
        unpack8(ld_bf16x8_nt(dout + i * 8), d);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float y, slope;
            gate_value_slope<ACT>(g[k], y, slope);
            dg[k] = d[k] * u[k] * slope;
            du[k] = d[k] * y;
            o[k] = y * u[k];
        }
        st_result<STREAM>(dgate + i * 8, pack8(dg));
        st_result<STREAM>(dup + i * 8, pack8(du));
        if (out) st_result<STREAM>(out + i * 8, pack8(o));
    }
}

unsigned gate_grid(int64_t n8) {
    const int64_t blocks = (n8 + kGateBlock - 1) / kGateBlock;
    return (unsigned)(blocks < 8192 ? blocks : 8192);
}

}  // namespace

extern "C" int ezl_gate_fwd(int act, const void* gate, const void* up, void* out, int64_t n, void* stream) {
    EZL_REQUIRE(act >= EZL_GATE_SILU && act <= EZL_GATE_RELU, EZL_EINVAL, "ezl_gate_fwd: act must be one of EZL_GATE_*");
    EZL_REQUIRE(n >= 0 && n % 8 == 0, EZL_EUNSUPPORTED, "ezl_gate_fwd: n must be a multiple of 8");
    EZL_REQUIRE(ezl_aligned16(gate) && ezl_aligned16(up) && ezl_aligned16(out) && (n == 0 || (gate && up && out)), EZL_EINVAL, "ezl_gate_fwd: null or misaligned pointer");
    if (n == 0) return EZL_OK;
    constexpr decltype(&gate_fwd_kernel<0>) kernels[] = {gate_fwd_kernel<0>, gate_fwd_kernel<1>, gate_fwd_kernel<2>, gate_fwd_kernel<3>};
    hipLaunchKernelGGL(kernels[act], dim3(gate_grid(n / 8)), dim3(kGateBlock), 0, (hipStream_t)stream, (const bf16_t*)gate, (const bf16_t*)up, (bf16_t*)out, n / 8);
    EZL_LAUNCH_CHECK("ezl_gate_fwd");
    return EZL_OK;
}

extern "C" int ezl_gate_bwd(int act, const void* dout, const void* gate, const void* up, void* dgate, void* dup, void* out, int64_t n, void* stream) {
    EZL_REQUIRE(act >= EZL_GATE_SILU && act <= EZL_GATE_RELU, EZL_EINVAL, "ezl_gate_bwd: act must be one of EZL_GATE_*");
    EZL_REQUIRE(n >= 0 && n % 8 == 0, EZL_EUNSUPPORTED, "ezl_gate_bwd: n must be a multiple of 8");
    EZL_REQUIRE(ezl_aligned16(dout) && ezl_aligned16(gate) && ezl_aligned16(up) && ezl_aligned16(dgate) && ezl_aligned16(dup) && ezl_aligned16(out) &&
                    (n == 0 || (dout && gate && up && dgate && dup)),
                EZL_EINVAL, "ezl_gate_bwd: null or misaligned pointer");
    if (n == 0) return EZL_OK;
    constexpr decltype(&gate_bwd_kernel<0, false>) kernels[][2] = {{gate_bwd_kernel<0, false>, gate_bwd_kernel<0, true>}, {gate_bwd_kernel<1, false>, gate_bwd_kernel<1, true>},
                                                                    {gate_bwd_kernel<2, false>, gate_bwd_kernel<2, true>}, {gate_bwd_kernel<3, false>, gate_bwd_kernel<3, true>}};
    hipLaunchKernelGGL(kernels[act][ezl_streams(n * (out ? 6 : 4))], dim3(gate_grid(n / 8)), dim3(kGateBlock), 0, (hipStream_t)stream, (const bf16_t*)dout,
                       (const bf16_t*)gate, (const bf16_t*)up, (bf16_t*)dgate, (bf16_t*)dup, (bf16_t*)out, n / 8);
    EZL_LAUNCH_CHECK("ezl_gate_bwd");
    return EZL_OK;
}
