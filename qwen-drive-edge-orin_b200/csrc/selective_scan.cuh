// Arguments of the selective scan, shared by its token-by-token kernel
// (selective_scan_step.cu) and the chunked one (selective_scan_chunk.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace gdn {
namespace ssm {

struct ScanArgs {
    const __nv_bfloat16 *x, *B, *C;
    const void* dt;
    const float *A, *D, *dt_bias;
    const float* s0;   // [N, H, P, NS] or null
    float* sf;         // [N, H, P, NS]
    __nv_bfloat16* y;  // [rows, H, P]
    const int* cu;     // packed offsets or null
    int64_t xs, dts, bs, cs;  // row strides, elements
    int N, T, H, P, G, NS;
    int dt_bf16, softplus;
};

// Token by token against a state in registers (one launch); any supported size.
cudaError_t launch_scan_step(const ScanArgs& a, cudaStream_t stream);

// In 128-token chunks on the tensor cores. The plan: units = slot pairs (two tiles of up to 64
// channels) over all groups, segments over all sequences (seg_tokens = 0: one each), and the
// scratch for the segments' states and log decays.
struct ChunkPlan {
    int pairs, units, seg_tokens;
    int64_t segments;
    size_t part_bytes, log_bytes;
};
ChunkPlan plan_scan_chunks(int N, int T, bool packed, int H, int P, int G, int sms);
// withhold: test hook, the chunk of each segment whose x tiles are never loaded (-1: none).
cudaError_t launch_scan_chunks(const ScanArgs& a, const ChunkPlan& pl, int64_t rows, void* workspace, void* scratch,
                               int withhold, cudaStream_t stream);

// Step size of (row, head) before the bias and the softplus.
__device__ __forceinline__ float scan_dt(const ScanArgs& a, int64_t row, int h) {
    return a.dt_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.dt)[row * a.dts + h])
                     : static_cast<const float*>(a.dt)[row * a.dts + h];
}

}  // namespace ssm
}  // namespace gdn
