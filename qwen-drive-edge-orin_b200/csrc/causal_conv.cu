// Short causal depthwise convolution over tokens, channels last, with a carried state:
//   y[t, c] = act( b[c] + sum_{j < W} w[c, j] x[t - W + 1 + j, c] )
// the layer in front of the recurrence (prompts and single tokens).
//
// Bound: bytes. Each input is read once and each output written once for 2 W flops, so a thread
// takes 8 bytes of channels and marches over a tile of tokens with the last W - 1 inputs in
// registers; the W - 1 rows in front of a tile are read twice (from L2). Products and sums are
// fp32, one rounding at the store. Eight bytes and eight tokens in flight at 24 warps an SM measured
// best (19592 x 6144 bf16: 105 us; 16 bytes at 12 warps 117, four tokens 138): 16-byte vectors keep
// twice the weights and inputs in registers. 15 us of the 105 are the silu's two special-function
// operations per element.
#include <cuda_runtime.h>
#include <stdint.h>

#include "gdn_common.cuh"
#include "gdn_ssm.h"
#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

constexpr int CONV_THREADS = 128;
constexpr int CONV_UNROLL = 8;  // tokens loaded ahead per thread

struct ConvArgs {
    const void *x, *w, *bias, *s0;
    void *y, *sf;
    const int* cu;
    int64_t xs;     // row stride of x, elements
    int64_t rows;   // token rows in all
    int N, T, C, silu;
    int tile;       // tokens per block
    int tiles;      // blocks along the tokens; blocks behind them write the final states
};

// Position q of a sequence's input stream: x for q >= 0, the initial state (or zero) before.
template <typename T, int VEC, int W>
__device__ __forceinline__ Vec<T, VEC> conv_input(const ConvArgs& a, int64_t begin, int64_t q, int seq, int c) {
    if (q >= 0) return ldg<T, VEC>(static_cast<const T*>(a.x) + (begin + q) * a.xs + c);
    Vec<T, VEC> r;
    if (a.s0 != nullptr) {
        r = ldg<T, VEC>(static_cast<const T*>(a.s0) + ((int64_t)seq * (W - 1) + (W - 1 + q)) * a.C + c);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = from_float<T>(0.f);
    }
    return r;
}

// Channels go in pairs (sm_100 multiplies and adds two fp32 values in one instruction); VEC = 1 leaves
// the second half idle.
template <typename T, int VEC, int W>
struct Taps {
    static constexpr int NP = (VEC + 1) / 2;
    uint64_t w[W][NP], b[NP], h[W - 1][NP];  // weights, bias, the last W - 1 inputs (oldest first)
    static __device__ __forceinline__ float at(const Vec<T, VEC>& v, int i) { return i < VEC ? to_float(v.v[i < VEC ? i : 0]) : 0.f; }
    __device__ __forceinline__ Taps(const void* wp, const void* bp, int c) {
        // the weights of VEC channels are W vectors in a row
        Vec<T, VEC> v[W], bv;
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = ldg<T, VEC>(static_cast<const T*>(wp) + (int64_t)c * W + j * VEC);
        if (bp) bv = ldg<T, VEC>(static_cast<const T*>(bp) + c);
        auto weight = [&](int i, int j) { return i < VEC ? to_float(v[(i * W + j) / VEC % W].v[(i * W + j) % VEC]) : 0.f; };
#pragma unroll
        for (int i = 0; i < NP; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = f2_pack(weight(2 * i, j), weight(2 * i + 1, j));
            b[i] = bp ? f2_pack(at(bv, 2 * i), at(bv, 2 * i + 1)) : 0;
        }
    }
    __device__ __forceinline__ void set(int j, const Vec<T, VEC>& v) {
#pragma unroll
        for (int i = 0; i < NP; ++i) h[j][i] = f2_pack(at(v, 2 * i), at(v, 2 * i + 1));
    }
    __device__ __forceinline__ Vec<T, VEC> get(int j) const {
        Vec<T, VEC> v;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            float x, y;
            f2_unpack(h[j][i], x, y);
            v.v[2 * i] = from_float<T>(x);
            if (2 * i + 1 < VEC) v.v[2 * i + 1 < VEC ? 2 * i + 1 : 0] = from_float<T>(y);
        }
        return v;
    }
    __device__ __forceinline__ Vec<T, VEC> step(const Vec<T, VEC>& in, int act) {
        Vec<T, VEC> out;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const uint64_t xi = f2_pack(at(in, 2 * i), at(in, 2 * i + 1));
            uint64_t s = b[i];
#pragma unroll
            for (int j = 0; j + 1 < W; ++j) s = f2_fma(w[j][i], h[j][i], s);
            s = f2_fma(w[W - 1][i], xi, s);
#pragma unroll
            for (int j = 0; j + 2 < W; ++j) h[j][i] = h[j + 1][i];
            h[W - 2][i] = xi;
            float x, y;
            f2_unpack(s, x, y);
            out.v[2 * i] = from_float<T>(act ? silu<T>(x) : x);
            if (2 * i + 1 < VEC) out.v[2 * i + 1 < VEC ? 2 * i + 1 : 0] = from_float<T>(act ? silu<T>(y) : y);
        }
        return out;
    }
};

template <typename T, int VEC, int W>
__global__ void __launch_bounds__(CONV_THREADS, 6) conv_prefill_kernel(const ConvArgs a) {
    const int c = (blockIdx.y * CONV_THREADS + threadIdx.x) * VEC;
    if (c >= a.C) return;
    if ((int)blockIdx.x >= a.tiles) {  // final state of one sequence: its last W - 1 inputs
        const int seq = blockIdx.x - a.tiles;
        int64_t begin, end;
        seq_range(a.cu, seq, a.T, begin, end);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            stg<T, VEC>(static_cast<T*>(a.sf) + ((int64_t)seq * (W - 1) + j) * a.C + c,
                        conv_input<T, VEC, W>(a, begin, end - begin - (W - 1) + j, seq, c));
        return;
    }
    Taps<T, VEC, W> taps(a.w, a.bias, c);
    int64_t r = (int64_t)blockIdx.x * a.tile;
    const int64_t stop = min(r + a.tile, a.rows);
    int seq;  // the sequence of row r
    if (a.cu == nullptr) {
        seq = (int)(r / a.T);
    } else {  // the last i with cu[i] <= r
        int lo = 0, hi = a.N;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= r) lo = mid; else hi = mid;
        }
        seq = lo;
    }
    for (; r < stop && seq < a.N; ++seq) {
        int64_t begin, end;
        seq_range(a.cu, seq, a.T, begin, end);
        if (r < begin) r = begin;
        const int64_t e = min(end, stop);
        if (r >= e) continue;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) taps.set(j, conv_input<T, VEC, W>(a, begin, r - begin - (W - 1) + j, seq, c));
        const T* xp = static_cast<const T*>(a.x) + r * a.xs + c;
        T* yp = static_cast<T*>(a.y) + r * a.C + c;
        int64_t left = e - r;
        for (; left >= CONV_UNROLL; left -= CONV_UNROLL) {
            Vec<T, VEC> in[CONV_UNROLL];
#pragma unroll
            for (int u = 0; u < CONV_UNROLL; ++u) in[u] = ldg<T, VEC>(xp + u * a.xs);
#pragma unroll
            for (int u = 0; u < CONV_UNROLL; ++u) stg<T, VEC>(yp + (int64_t)u * a.C, taps.step(in[u], a.silu));
            xp += CONV_UNROLL * a.xs;
            yp += (int64_t)CONV_UNROLL * a.C;
        }
        for (; left > 0; --left) {
            stg<T, VEC>(yp, taps.step(ldg<T, VEC>(xp), a.silu));
            xp += a.xs;
            yp += a.C;
        }
        r = e;
    }
}

// T tokens of B sequences against a state updated in place: a thread owns VEC channels of a sequence.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(CONV_THREADS) conv_decode_kernel(const ConvArgs a) {
    const int c = (blockIdx.y * CONV_THREADS + threadIdx.x) * VEC;
    if (c >= a.C) return;
    Taps<T, VEC, W> taps(a.w, a.bias, c);
    const int64_t b = blockIdx.x;
    T* st = static_cast<T*>(a.sf) + b * (W - 1) * a.C + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        taps.set(j, *reinterpret_cast<const Vec<T, VEC>*>(st + (int64_t)j * a.C));
    }
    for (int t = 0; t < a.T; ++t) {
        const int64_t row = b * a.T + t;
        stg<T, VEC>(static_cast<T*>(a.y) + row * a.C + c,
                    taps.step(ldg<T, VEC>(static_cast<const T*>(a.x) + row * a.xs + c), a.silu));
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        stg<T, VEC>(st + (int64_t)j * a.C, taps.get(j));
    }
}

template <typename T, int VEC, int W>
static cudaError_t conv_launch(ConvArgs& a, bool decode, cudaStream_t stream) {
    const int64_t cblocks = ((int64_t)a.C + CONV_THREADS * VEC - 1) / (CONV_THREADS * VEC);
    if (cblocks > 65535) return cudaErrorInvalidValue;
    if (decode) {
        conv_decode_kernel<T, VEC, W><<<dim3((unsigned)a.N, (unsigned)cblocks), CONV_THREADS, 0, stream>>>(a);
        return cudaGetLastError();
    }
    // Tokens per block: long tiles re-read less (W - 1 rows per tile), short ones fill the GPU. The
    // longest tile that still gives about eight blocks per SM.
    a.tile = 64;
    while (a.tile > CONV_UNROLL && (a.rows + a.tile - 1) / a.tile * cblocks < 148 * 8) a.tile >>= 1;
    const int64_t tiles = (a.rows + a.tile - 1) / a.tile;
    if (tiles + a.N > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.tiles = (int)tiles;
    conv_prefill_kernel<T, VEC, W><<<dim3((unsigned)(tiles + a.N), (unsigned)cblocks), CONV_THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, int VEC>
static cudaError_t conv_width(ConvArgs& a, int W, bool decode, cudaStream_t stream) {
    switch (W) {
        case 2: return conv_launch<T, VEC, 2>(a, decode, stream);
        case 3: return conv_launch<T, VEC, 3>(a, decode, stream);
        default: return conv_launch<T, VEC, 4>(a, decode, stream);
    }
}

template <typename T>
static cudaError_t conv_type(ConvArgs& a, int W, bool decode, cudaStream_t stream) {
    constexpr int VEC = 8 / sizeof(T);
    // 8-byte accesses where every row starts on 8 bytes, else one channel per thread
    const bool wide = a.C % VEC == 0 && a.xs % VEC == 0 && aligned_to(a.x, 8) && aligned_to(a.y, 8) && aligned_to(a.s0, 8) &&
                      aligned_to(a.sf, 8) && aligned_to(a.w, 8) && aligned_to(a.bias, 8);
    return wide ? conv_width<T, VEC>(a, W, decode, stream) : conv_width<T, 1>(a, W, decode, stream);
}

static cudaError_t conv_dtype(ConvArgs& a, int W, int dtype, bool decode, cudaStream_t stream) {
    switch (dtype) {
        case 0: return conv_type<__half>(a, W, decode, stream);
        case 1: return conv_type<__nv_bfloat16>(a, W, decode, stream);
        default: return conv_type<float>(a, W, decode, stream);
    }
}

static bool conv_args_ok(int N, int T, int C, int W, int dtype, int64_t x_stride) {
    return N >= 0 && T >= 0 && C >= 1 && W >= 2 && W <= 4 && dtype >= 0 && dtype <= 2 && x_stride >= C;
}

}  // namespace ssm
}  // namespace gdn

extern "C" cudaError_t causal_conv_prefill(const void* x, int64_t x_stride, const void* w, const void* bias,
                                           const void* s0, void* y, void* sf, const int* cu_seqlens, int N, int T,
                                           int C, int W, int silu, int dtype, cudaStream_t stream) {
    if (!gdn::ssm::conv_args_ok(N, T, C, W, dtype, x_stride)) return cudaErrorInvalidValue;
    if (N == 0) return cudaSuccess;
    const int64_t rows = cu_seqlens ? T : (int64_t)N * T;
    if (!w || !sf || (rows > 0 && (!x || !y))) return cudaErrorInvalidValue;
    gdn::ssm::ConvArgs a{x, w, bias, s0, y, sf, cu_seqlens, x_stride, rows, N, T, C, silu, 0, 0};
    return gdn::ssm::conv_dtype(a, W, dtype, false, stream);
}

extern "C" cudaError_t causal_conv_decode(const void* x, int64_t x_stride, const void* w, const void* bias, void* state,
                                          void* y, int B, int T, int C, int W, int silu, int dtype,
                                          cudaStream_t stream) {
    if (!gdn::ssm::conv_args_ok(B, T, C, W, dtype, x_stride)) return cudaErrorInvalidValue;
    if (B == 0 || T == 0) return cudaSuccess;
    if (!x || !w || !state || !y) return cudaErrorInvalidValue;
    gdn::ssm::ConvArgs a{x, w, bias, nullptr, y, state, nullptr, x_stride, (int64_t)B * T, B, T, C, silu, 0, 0};
    return gdn::ssm::conv_dtype(a, W, dtype, true, stream);
}
