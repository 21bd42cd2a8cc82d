/*
 * gdn_b200 C ABI, state-space operators for NVIDIA B200 (sm_100a): the short
 * causal convolution, the selective scan (prompts and single tokens) and the
 * gated group norm of hybrid layers. They stand beside the gated delta rule of
 * gdn_prefill.h and follow its conventions: caller-owned device memory, calls
 * asynchronous and stream-ordered, nothing allocated, cudaErrorInvalidValue for
 * bad arguments before any device work, otherwise the launch error, if any.
 * No counterparts in the reference.
 *
 * Sequences. cu_seqlens == NULL: N sequences of T tokens, sequence i at token
 * rows [i T, (i + 1) T). Otherwise (packed) T is the number of token rows and
 * sequence i covers rows [cu_seqlens[i], cu_seqlens[i + 1]) (int32, device
 * memory, non-decreasing, cu_seqlens[0] >= 0, cu_seqlens[N] <= T; values are
 * clamped to [0, T]). Rows that no sequence covers are not written. A sequence
 * may be empty: its final state is its initial state.
 *
 * Token rows of an input may be further apart than they are wide (a slice of a
 * wider projection): *_stride is the distance of consecutive rows in elements.
 * Outputs are contiguous. dtype: 0 fp16, 1 bf16, 2 fp32.
 */
#ifndef GDN_B200_GDN_SSM_H_
#define GDN_B200_GDN_SSM_H_

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Short causal depthwise convolution over tokens, channels last:
 *   y[t, c] = act( bias[c] + sum_{j < W} w[c, j] x[t - W + 1 + j, c] ),  act = silu or none
 * x [rows, C] (x_stride), w [C, W], bias [C] or NULL, y [rows, C], all of `dtype`, fp32 math.
 * Inputs before a sequence's start are s0 [N, W - 1, C] (oldest first) or, with s0 NULL, zeros;
 * sf [N, W - 1, C] receives each sequence's last W - 1 inputs (of s0 and x together).
 * 2 <= W <= 4. sf must not overlap s0 or x. */
cudaError_t causal_conv_prefill(const void* x, int64_t x_stride, const void* w, const void* bias, const void* s0,
                                void* y, void* sf, const int* cu_seqlens, int N, int T, int C, int W, int silu,
                                int dtype, cudaStream_t stream);

/* The same for the next T tokens (usually one) of B sequences, x [B, T, C], with the last W - 1
 * inputs in `state` [B, W - 1, C], read and updated in place. */
cudaError_t causal_conv_decode(const void* x, int64_t x_stride, const void* w, const void* bias, void* state, void* y,
                               int B, int T, int C, int W, int silu, int dtype, cudaStream_t stream);

/* Selective state space scan with a scalar decay per head. Per sequence, head h and token t, with
 * d = dt[t, h] + dt_bias[h], softplus'ed if dt_softplus != 0:
 *   S <- exp(d A[h]) S + d x[t, h, :] B[t, g, :]^T;   y[t, h, :] = S C[t, g, :] + D[h] x[t, h, :]
 * x [rows, H, P], B and C [rows, G, N_STATE] bf16 (heads and groups contiguous inside a row), head h
 * uses group h / (H / G); dt [rows, H] fp32 (dt_bf16 = 0) or bf16 (1); A, D (or NULL), dt_bias (or
 * NULL) fp32 [H]; y bf16 [rows, H, P]; s0 (or NULL: zeros) and sf fp32 [N, H, P, N_STATE].
 * d A <= 0 (a decay). P and N_STATE are multiples of 8 up to 128, N and H at most 65535, token rows at
 * most 2^31 - 129; x, B, C rows 16-byte aligned. sf must not overlap s0. An x that is not finite makes its
 * channel's outputs NaN from the start of its 128 tokens (counted from the sequence's start) on, not
 * from its own token on; no value of any input reaches another sequence.
 * workspace: at least 256 bytes, zero before its first use, whose first word is the status word
 * (deltanet_read_status: 0, or bits 0 and 16 where a bounded wait of the scan ran out); calls may share it. scratch: selective_scan_scratch_size(...) bytes for the
 * same sizes on the same device, 256-byte aligned (NULL where that is 0); calls that may overlap in
 * time need scratch of their own. */
size_t selective_scan_scratch_size(int N, int T, int packed, int H, int P, int G, int n_state);
cudaError_t selective_scan_prefill(const void* x, int64_t x_stride, const void* dt, int64_t dt_stride, int dt_bf16,
                                   const float* A, const void* B, int64_t B_stride, const void* C, int64_t C_stride,
                                   const float* D, const float* dt_bias, int dt_softplus, const float* s0, void* y,
                                   float* sf, const int* cu_seqlens, int N, int T, int H, int P, int G, int n_state,
                                   void* workspace, size_t workspace_bytes, void* scratch, size_t scratch_bytes,
                                   cudaStream_t stream);

/* Test hook for failure detection: selective_scan_prefill of N sequences of T tokens (at least 16; contiguous
 * inputs, fp32 dt, no D, dt_bias, softplus or s0) with the x tiles of chunk `withheld_chunk` (of 128 tokens, counted in
 * each segment) never loaded. The waits for them run out, the status word says so, the kernels stop, wait (bounded)
 * for what they have in flight and return; y and sf are then undefined. Returns the launch status. */
cudaError_t selective_scan_test_withheld_load(const void* x, const void* dt, const float* A, const void* B,
                                              const void* C, void* y, float* sf, int N, int T, int H, int P, int G,
                                              int n_state, void* workspace, size_t workspace_bytes, void* scratch,
                                              size_t scratch_bytes, cudaStream_t stream, int withheld_chunk);

/* The next T tokens (usually one) of `N` sequences, x [N, T, H, P], with the state [N, H, P, N_STATE]
 * read and updated in place. Continues a prefill from its final state. */
cudaError_t selective_scan_decode(const void* x, int64_t x_stride, const void* dt, int64_t dt_stride, int dt_bf16,
                                  const float* A, const void* B, int64_t B_stride, const void* C, int64_t C_stride,
                                  const float* D, const float* dt_bias, int dt_softplus, float* state, void* y,
                                  int N, int T, int H, int P, int G, int n_state, cudaStream_t stream);

/* Gated RMSNorm over channel groups, the gate before the norm:
 *   u = x silu(z);  y = w u rsqrt(mean over the row's group of C / groups channels of u^2 + eps)
 * x, z [rows, C] (row strides), w [C], y [rows, C], all of `dtype`; fp32 math, one rounding.
 * (gated_rmsnorm_forward of gdn_prefill.h has the gate behind the norm.) */
cudaError_t gated_group_rmsnorm_forward(const void* x, int64_t x_stride, const void* z, int64_t z_stride, const void* w,
                                        void* y, int64_t rows, int C, int groups, float eps, int dtype,
                                        cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GDN_B200_GDN_SSM_H_ */
