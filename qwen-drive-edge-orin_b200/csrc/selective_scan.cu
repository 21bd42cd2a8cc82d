// Selective scan over prompts: entry points, argument checks and the choice of kernel.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "gdn_ssm.h"
#include "selective_scan.cuh"
#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

// Calls of up to this many tokens a sequence run token by token, packed ones of up to this many token rows in all
// (their lengths are on the device): 128 packed single tokens take the chunks, 408 us against 85 as a decode (64 heads
// of 64). Measured (64 heads of 64, state 128, 64 sequences):
// 115 us at 8 tokens and 197 at 16 against 194 for one chunk; one sequence of 24 heads: 6.0 and 10.3
// against 9.8.
constexpr int STEP_TOKENS = 15;

static int sm_count() {
    static std::atomic<int> known[64] = {};  // per device; threads that race here store the same value
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if ((sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

static bool scan_args_ok(const ScanArgs& a, int64_t rows) {
    if (a.N < 0 || a.T < 0 || a.H < 1 || a.G < 1 || a.H % a.G != 0 || a.H > 65535 || a.N > 65535) return false;
    if (a.P < 8 || a.P > 128 || a.P % 8 != 0 || a.NS < 8 || a.NS > 128 || a.NS % 8 != 0) return false;
    if (a.xs < (int64_t)a.H * a.P || a.bs < (int64_t)a.G * a.NS || a.cs < (int64_t)a.G * a.NS || a.dts < a.H) return false;
    if (a.xs % 8 != 0 || a.bs % 8 != 0 || a.cs % 8 != 0) return false;
    if (a.N == 0) return true;
    if (!a.A || !a.sf || !aligned_to(a.sf, 16) || !aligned_to(a.s0, 16)) return false;
    if (rows > 0 && (!a.x || !a.dt || !a.B || !a.C || !a.y)) return false;
    return aligned_to(a.x, 16) && aligned_to(a.B, 16) && aligned_to(a.C, 16) && aligned_to(a.y, 16);
}

// withhold: see launch_scan_chunks; such a call never runs token by token.
static cudaError_t scan_prefill(const ScanArgs& a, void* workspace, size_t workspace_bytes, void* scratch, size_t scratch_bytes,
                                int withhold, cudaStream_t stream) {
    const int64_t rows = a.cu ? a.T : (int64_t)a.N * a.T;
    if (!scan_args_ok(a, rows)) return cudaErrorInvalidValue;
    if (!workspace || workspace_bytes < 256) return cudaErrorInvalidValue;
    if (a.N == 0) return cudaSuccess;
    if (a.T <= STEP_TOKENS) return withhold < 0 ? launch_scan_step(a, stream) : cudaErrorInvalidValue;
    if (rows > 0x7fffffffLL - 128) return cudaErrorInvalidValue;  // token rows are 32-bit tile coordinates
    const ChunkPlan pl = plan_scan_chunks(a.N, a.T, a.cu != nullptr, a.H, a.P, a.G, sm_count());
    if (pl.part_bytes > 0 && (!scratch || !aligned_to(scratch, 256) || scratch_bytes < pl.log_bytes + pl.part_bytes))
        return cudaErrorInvalidValue;
    return launch_scan_chunks(a, pl, rows, workspace, scratch, withhold, stream);
}

}  // namespace ssm
}  // namespace gdn

extern "C" size_t selective_scan_scratch_size(int N, int T, int packed, int H, int P, int G, int n_state) {
    using namespace gdn::ssm;
    if (N <= 0 || T <= STEP_TOKENS || H < 1 || G < 1 || H % G != 0 || P < 1) return 0;
    const ChunkPlan pl = plan_scan_chunks(N, T, packed != 0, H, P, G, sm_count());
    return pl.log_bytes + pl.part_bytes;
}

extern "C" cudaError_t selective_scan_prefill(const void* x, int64_t x_stride, const void* dt, int64_t dt_stride,
                                              int dt_bf16, const float* A, const void* B, int64_t B_stride,
                                              const void* C, int64_t C_stride, const float* D, const float* dt_bias,
                                              int dt_softplus, const float* s0, void* y, float* sf,
                                              const int* cu_seqlens, int N, int T, int H, int P, int G, int n_state,
                                              void* workspace, size_t workspace_bytes, void* scratch,
                                              size_t scratch_bytes, cudaStream_t stream) {
    using bf16 = __nv_bfloat16;
    gdn::ssm::ScanArgs a{static_cast<const bf16*>(x), static_cast<const bf16*>(B), static_cast<const bf16*>(C), dt, A, D,
                         dt_bias, s0, sf, static_cast<bf16*>(y), cu_seqlens, x_stride, dt_stride, B_stride, C_stride, N, T,
                         H, P, G, n_state, dt_bf16, dt_softplus};
    return gdn::ssm::scan_prefill(a, workspace, workspace_bytes, scratch, scratch_bytes, -1, stream);
}

// Test hook for the bounded waits: the x tiles of one chunk never arrive, so that the waits for them run out.
// No fault, trap or unbounded wait is involved.
extern "C" cudaError_t selective_scan_test_withheld_load(const void* x, const void* dt, const float* A, const void* B,
                                                         const void* C, void* y, float* sf, int N, int T, int H, int P,
                                                         int G, int n_state, void* workspace, size_t workspace_bytes,
                                                         void* scratch, size_t scratch_bytes, cudaStream_t stream,
                                                         int withheld_chunk) {
    using bf16 = __nv_bfloat16;
    if (withheld_chunk < 0) return cudaErrorInvalidValue;
    gdn::ssm::ScanArgs a{static_cast<const bf16*>(x), static_cast<const bf16*>(B), static_cast<const bf16*>(C), dt, A, nullptr,
                         nullptr, nullptr, sf, static_cast<bf16*>(y), nullptr, (int64_t)H * P, H, (int64_t)G * n_state,
                         (int64_t)G * n_state, N, T, H, P, G, n_state, 0, 0};
    return gdn::ssm::scan_prefill(a, workspace, workspace_bytes, scratch, scratch_bytes, withheld_chunk, stream);
}

extern "C" cudaError_t selective_scan_decode(const void* x, int64_t x_stride, const void* dt, int64_t dt_stride,
                                             int dt_bf16, const float* A, const void* B, int64_t B_stride, const void* C,
                                             int64_t C_stride, const float* D, const float* dt_bias, int dt_softplus,
                                             float* state, void* y, int N, int T, int H, int P, int G, int n_state,
                                             cudaStream_t stream) {
    using bf16 = __nv_bfloat16;
    gdn::ssm::ScanArgs a{static_cast<const bf16*>(x), static_cast<const bf16*>(B), static_cast<const bf16*>(C), dt, A, D,
                         dt_bias, state, state, static_cast<bf16*>(y), nullptr, x_stride, dt_stride, B_stride, C_stride, N,
                         T, H, P, G, n_state, dt_bf16, dt_softplus};
    if (!gdn::ssm::scan_args_ok(a, (int64_t)N * T)) return cudaErrorInvalidValue;
    if (N == 0 || T == 0) return cudaSuccess;
    return gdn::ssm::launch_scan_step(a, stream);
}
