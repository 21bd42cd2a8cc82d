// Helpers shared by the state-space operators (causal_conv.cu, selective_scan*.cu,
// gated_group_norm.cu): conversions, 16-byte vectors of a storage type, silu and
// softplus, and the token range of a sequence.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace gdn {
namespace ssm {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// VEC consecutive elements: one access of 16 or 8 bytes, or one element (VEC = 1).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> ldg(const T* p) {
    Vec<T, VEC> r;
    if constexpr (sizeof(T) * VEC == 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        r = *reinterpret_cast<const Vec<T, VEC>*>(&u);
    } else if constexpr (sizeof(T) * VEC == 8) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        r = *reinterpret_cast<const Vec<T, VEC>*>(&u);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = p[i];
    }
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void stg(T* p, const Vec<T, VEC>& r) {
    if constexpr (sizeof(T) * VEC == 16) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
    } else if constexpr (sizeof(T) * VEC == 8) {
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&r);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[i] = r.v[i];
    }
}

// silu(v) = v / (1 + e^-v). 16-bit outputs take the fast exponential (off by 2 fp32 ulp and one more for each
// unit of |v|: 2^-17 at most, far below the output's rounding) and division (0 for divisors above 2^126: below
// v = -87.3, where silu is under 2^-119); fp32 outputs the full-precision ones. e^-v = inf gives 0.
template <typename T>
__device__ __forceinline__ float silu(float v) {
    if constexpr (sizeof(T) == 4) return v / (1.f + expf(-v));
    return __fdividef(v, 1.f + __expf(-v));
}

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }

// Token rows [begin, end) of sequence i. Packed offsets are clamped to [0, T] and to order, so
// that a bad offset never becomes an access outside the buffers.
__device__ __forceinline__ void seq_range(const int* cu, int i, int T, int64_t& begin, int64_t& end) {
    if (cu == nullptr) {
        begin = (int64_t)i * T;
        end = begin + T;
    } else {
        const int b = min(max(cu[i], 0), T);
        begin = b;
        end = max(min(max(cu[i + 1], 0), T), b);
    }
}

}  // namespace ssm

inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace gdn
