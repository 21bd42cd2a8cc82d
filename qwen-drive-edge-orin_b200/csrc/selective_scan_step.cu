// Selective scan, token by token: the state of a few rows stays in registers while the tokens of a
// sequence pass (the decode form, usually one token; and prompts).
//   S <- e^{d A} S + d x_t B_t^T;   y_t = S C_t + D x_t
//
// Bound for one token: the state's bytes, 8 P NS per head, read and written once. Eight lanes share
// a state row (a float4 each per 32 columns, so a warp's access covers four rows by 128 contiguous
// bytes); the sum over the columns takes three shuffles for four rows. fp32 state and sums.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gdn_ssm.h"
#include "selective_scan.cuh"
#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

constexpr int STEP_THREADS = 128;

// KN: float4 column groups per lane (32 KN >= NS). R: rows per lane.
template <int KN, int R>
__global__ void __launch_bounds__(STEP_THREADS) scan_step_kernel(const ScanArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane & 7, rl = lane >> 3;
    const int h = blockIdx.y, seq = blockIdx.z;
    const int g = h / (a.H / a.G);
    const int p0 = (blockIdx.x * (STEP_THREADS / 32) + warp) * 4 * R + rl;
    if (p0 - rl >= a.P) return;  // whole warps
    const int64_t sbase = ((int64_t)seq * a.H + h) * a.P * a.NS;
    int64_t row, end;
    seq_range(a.cu, seq, a.T, row, end);

    float s[R][KN][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < KN; ++k) {
            const int p = p0 + 4 * r, n = 4 * sub + 32 * k;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            // a plain load: the state may be the output buffer
            if (a.s0 != nullptr && p < a.P && n < a.NS)
                v = *reinterpret_cast<const float4*>(a.s0 + sbase + (int64_t)p * a.NS + n);
            s[r][k][0] = v.x; s[r][k][1] = v.y; s[r][k][2] = v.z; s[r][k][3] = v.w;
        }
    const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.f, D = a.D ? a.D[h] : 0.f;
    for (; row < end; ++row) {
        float d = scan_dt(a, row, h) + bias;
        if (a.softplus) d = softplus(d);
        const float decay = expf(d * A);
        float bv[KN][4], cv[KN][4];
#pragma unroll
        for (int k = 0; k < KN; ++k) {
            const int n = 4 * sub + 32 * k;
            Vec<__nv_bfloat16, 4> b4, c4;
            uint2 ub = make_uint2(0u, 0u), uc = ub;
            if (n < a.NS) {
                ub = __ldg(reinterpret_cast<const uint2*>(a.B + row * a.bs + (int64_t)g * a.NS + n));
                uc = __ldg(reinterpret_cast<const uint2*>(a.C + row * a.cs + (int64_t)g * a.NS + n));
            }
            b4 = *reinterpret_cast<Vec<__nv_bfloat16, 4>*>(&ub);
            c4 = *reinterpret_cast<Vec<__nv_bfloat16, 4>*>(&uc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bv[k][i] = to_float(b4.v[i]);
                cv[k][i] = to_float(c4.v[i]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int p = p0 + 4 * r;
            const float x = p < a.P ? to_float(a.x[row * a.xs + (int64_t)h * a.P + p]) : 0.f;
            const float dx = d * x;
            float y = 0.f;
#pragma unroll
            for (int k = 0; k < KN; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[r][k][i] = fmaf(dx, bv[k][i], decay * s[r][k][i]);
                    y = fmaf(s[r][k][i], cv[k][i], y);
                }
            y += __shfl_xor_sync(0xffffffffu, y, 1);
            y += __shfl_xor_sync(0xffffffffu, y, 2);
            y += __shfl_xor_sync(0xffffffffu, y, 4);
            if (sub == 0 && p < a.P) a.y[(row * a.H + h) * a.P + p] = __float2bfloat16_rn(fmaf(D, x, y));
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < KN; ++k) {
            const int p = p0 + 4 * r, n = 4 * sub + 32 * k;
            if (p < a.P && n < a.NS)
                *reinterpret_cast<float4*>(a.sf + sbase + (int64_t)p * a.NS + n) =
                    make_float4(s[r][k][0], s[r][k][1], s[r][k][2], s[r][k][3]);
        }
}

template <int KN>
static cudaError_t step_rows(const ScanArgs& a, cudaStream_t stream) {
    // Four rows per lane keep 16 loads of 16 bytes in flight; one row per lane where four would not
    // give every SM a block (one request: latency counts, not bytes).
    const int64_t wide = (int64_t)((a.P + 63) / 64) * a.H * a.N;
    if (wide >= 2 * 148)
        scan_step_kernel<KN, 4><<<dim3((a.P + 63) / 64, a.H, a.N), STEP_THREADS, 0, stream>>>(a);
    else
        scan_step_kernel<KN, 1><<<dim3((a.P + 15) / 16, a.H, a.N), STEP_THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_scan_step(const ScanArgs& a, cudaStream_t stream) {
    switch ((a.NS + 31) / 32) {
        case 1: return step_rows<1>(a, stream);
        case 2: return step_rows<2>(a, stream);
        case 3: return step_rows<3>(a, stream);
        default: return step_rows<4>(a, stream);
    }
}

}  // namespace ssm
}  // namespace gdn
