// Gated RMSNorm over channel groups, the gate before the norm:
//   u = x silu(z);  y = w u rsqrt(mean_group(u^2) + eps)
// the norm behind a selective scan (gated_rmsnorm.cu has the gate behind the norm, one group a row).
//
// Bound: bytes, three streams. A team of threads owns one group of one row: a warp for groups of up to
// 64 vectors of 16 bytes, then 64, 128 and 256 threads. The team keeps u in registers between the sum of
// squares and the store, so x and z are read once; elements beyond the registers (groups wider than
// 256 x 8 vectors) are read and gated a second time. Few threads with several vectors each have more loads
// in flight per synchronisation: 32768 rows of 4096 bf16 take 138 us with 128 threads x 4 vectors, 156 with
// 256 x 2, 182 with 512 x 1; 8192 rows of 8192 77 us with 128 x 8, 86 with 256 x 2 and re-reads; 16384 rows
// of 8 groups of 1024 149 us with 64 x 2, 171 with a warp x 4. fp32 math, one rounding at the store.
#include <cuda_runtime.h>
#include <stdint.h>

#include "gdn_ssm.h"
#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

// Blocks of NT threads hold NT / TEAM teams.
template <typename T, int VEC, int TEAM, int KEEP, int NT = (TEAM > 32 ? TEAM : 128)>
__global__ void __launch_bounds__(NT) group_norm_kernel(const T* __restrict__ x, int64_t xs,
                                                                  const T* __restrict__ z, int64_t zs,
                                                                  const T* __restrict__ w, T* __restrict__ y,
                                                                  int64_t units, int C, int groups, float eps) {
    __shared__ float part[NT / 32];
    const int team = threadIdx.x / TEAM, me = threadIdx.x % TEAM;
    const int64_t unit = (int64_t)blockIdx.x * (NT / TEAM) + team;
    if (TEAM == 32 && unit >= units) return;  // whole warps; block teams are launched exactly
    const int64_t row = unit / groups;
    const int gs = C / groups, c0 = (int)(unit - row * groups) * gs;
    const T* xr = x + row * xs + c0;
    const T* zr = z + row * zs + c0;
    T* yr = y + row * C + c0;
    const T* wr = w + c0;
    const int nv = gs / VEC;  // vectors of the group
    float u[KEEP][VEC];
    float ss = 0.f;
    {
        Vec<T, VEC> xv[KEEP], zv[KEEP];
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            if (me + k * TEAM < nv) {
                xv[k] = ldg<T, VEC>(xr + (int64_t)(me + k * TEAM) * VEC);
                zv[k] = ldg<T, VEC>(zr + (int64_t)(me + k * TEAM) * VEC);
            }
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            if (me + k * TEAM < nv) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    u[k][i] = to_float(xv[k].v[i]) * silu<T>(to_float(zv[k].v[i]));
                    ss = fmaf(u[k][i], u[k][i], ss);
                }
            }
    }
    for (int j = me + KEEP * TEAM; j < nv; j += TEAM) {
        const Vec<T, VEC> xv = ldg<T, VEC>(xr + (int64_t)j * VEC), zv = ldg<T, VEC>(zr + (int64_t)j * VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float v = to_float(xv.v[i]) * silu<T>(to_float(zv.v[i]));
            ss = fmaf(v, v, ss);
        }
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if constexpr (TEAM > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) ss += part[i];
    }
    const float rstd = rsqrtf(ss / (float)gs + eps);
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (me + k * TEAM < nv) {
            const Vec<T, VEC> wv = ldg<T, VEC>(wr + (me + k * TEAM) * VEC);
            Vec<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.v[i] = from_float<T>(to_float(wv.v[i]) * (u[k][i] * rstd));
            stg<T, VEC>(yr + (int64_t)(me + k * TEAM) * VEC, o);
        }
    for (int j = me + KEEP * TEAM; j < nv; j += TEAM) {
        const Vec<T, VEC> xv = ldg<T, VEC>(xr + (int64_t)j * VEC), zv = ldg<T, VEC>(zr + (int64_t)j * VEC);
        const Vec<T, VEC> wv = ldg<T, VEC>(wr + j * VEC);
        Vec<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            o.v[i] = from_float<T>(to_float(wv.v[i]) * (to_float(xv.v[i]) * silu<T>(to_float(zv.v[i])) * rstd));
        stg<T, VEC>(yr + (int64_t)j * VEC, o);
    }
}

template <typename T, int VEC, int TEAM, int KEEP, int NT = (TEAM > 32 ? TEAM : 128)>
static cudaError_t norm_launch(const void* x, int64_t xs, const void* z, int64_t zs, const void* w, void* y, int64_t units,
                               int C, int groups, float eps, cudaStream_t stream) {
    const int64_t per = NT / TEAM, blocks = (units + per - 1) / per;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    group_norm_kernel<T, VEC, TEAM, KEEP, NT><<<(unsigned)blocks, NT, 0, stream>>>(
        static_cast<const T*>(x), xs, static_cast<const T*>(z), zs, static_cast<const T*>(w), static_cast<T*>(y), units, C,
        groups, eps);
    return cudaGetLastError();
}

template <typename T, int VEC>
static cudaError_t norm_vec(const void* x, int64_t xs, const void* z, int64_t zs, const void* w, void* y, int64_t rows, int C,
                            int groups, float eps, cudaStream_t stream) {
    const int nv = C / groups / VEC;
    const int64_t units = rows * groups;
#define GDN_NORM(TEAM, KEEP) norm_launch<T, VEC, TEAM, KEEP>(x, xs, z, zs, w, y, units, C, groups, eps, stream)
    if (nv <= 32) return GDN_NORM(32, 1);
    if (nv <= 64) return GDN_NORM(32, 2);
    if (nv <= 128) return GDN_NORM(64, 2);
    if (nv <= 256) return GDN_NORM(128, 2);
    if (nv <= 512) return GDN_NORM(128, 4);
    if (nv <= 1024) return GDN_NORM(128, 8);
    return GDN_NORM(256, 8);
#undef GDN_NORM
}

template <typename T>
static cudaError_t norm_type(const void* x, int64_t xs, const void* z, int64_t zs, const void* w, void* y, int64_t rows, int C,
                             int groups, float eps, cudaStream_t stream) {
    constexpr int VEC = 16 / sizeof(T);
    // 16-byte accesses where every group starts on 16 bytes, else one element at a time
    const bool wide = (C / groups) % VEC == 0 && xs % VEC == 0 && zs % VEC == 0 && aligned_to(x, 16) && aligned_to(z, 16) &&
                      aligned_to(w, 16) && aligned_to(y, 16);
    return wide ? norm_vec<T, VEC>(x, xs, z, zs, w, y, rows, C, groups, eps, stream)
                : norm_vec<T, 1>(x, xs, z, zs, w, y, rows, C, groups, eps, stream);
}

}  // namespace ssm
}  // namespace gdn

extern "C" cudaError_t gated_group_rmsnorm_forward(const void* x, int64_t x_stride, const void* z, int64_t z_stride,
                                                   const void* w, void* y, int64_t rows, int C, int groups, float eps,
                                                   int dtype, cudaStream_t stream) {
    if (rows < 0 || C < 1 || groups < 1 || C % groups != 0 || dtype < 0 || dtype > 2 || x_stride < C || z_stride < C)
        return cudaErrorInvalidValue;
    if (rows == 0) return cudaSuccess;
    if (!x || !z || !w || !y) return cudaErrorInvalidValue;
    switch (dtype) {
        case 0: return gdn::ssm::norm_type<__half>(x, x_stride, z, z_stride, w, y, rows, C, groups, eps, stream);
        case 1: return gdn::ssm::norm_type<__nv_bfloat16>(x, x_stride, z, z_stride, w, y, rows, C, groups, eps, stream);
        default: return gdn::ssm::norm_type<float>(x, x_stride, z, z_stride, w, y, rows, C, groups, eps, stream);
    }
}
