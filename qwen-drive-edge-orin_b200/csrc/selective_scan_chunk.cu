// Selective scan over prompts in 128-token chunks on the tensor cores (tcgen05, TMEM, TMA).
//
// With a_t = d_t A (log decay) and c_i the inclusive sum of a over a chunk, the recurrence
// S <- e^{a_t} S + d_t x_t B_t^T, y_t = S C_t + D x_t is, over one chunk with entry state S,
//   G      = C B^T                                              [128 x 128]  (shared by the heads of a group)
//   y      = diag(e^{c}) (C S^T) + M X + D X,   M_ij = G_ij e^{c_i - c_j} d_j for j <= i, else 0
//   S     <- e^{c_L} S + X'^T B,                X'_j = e^{c_L - c_j} d_j x_j
// all four products with 128 rows.
//
// A CTA owns one segment of a sequence and two "slots" of a group: a slot is one head's tile of up to
// 64 channels (a head of 128 is two slots). The two share the B and C tiles and G, and stand side by
// side in the 128 columns of C S^T and the 128 rows of the state.
//   warps 0-7   M (bf16, both slots) from G in TMEM, in place, the A operand of M X; Y <- e^c Y
//   warps 8-15  the state S (fp32, TMEM-resident): its bf16 copy (operand of C S^T) and its decay; the
//               output tile
//   warps 0-15  X'^T, 32 tokens each warpgroup, into TMEM as the A operand of the state product
//   warp 16     issues the state products, warp 19 the others, per chunk inter (C S^T), intra (M X) and
//               the next chunk's G
//   warp 17     every TMA load and the TMA stores of the output tiles; warp 18 the gates
//
// Precision. G and all sums are fp32. M and the state operand of C S^T are rounded to bf16 once (y is
// a bf16 output, and each of its terms is off by at most one more rounding of that size). The state itself is an fp32 output and carries
// over thousands of tokens: X' is split exactly into three bf16 terms (8 + 8 + 8 bits of an fp32 value),
// so its products are those of fp32 operands; and as the tensor cores truncate their fp32 sums, they only sum
// what is of a chunk's size (output pass: the chunk's sum and the state's remainder beside its bf16 copy; state
// pass: up to four chunks), which joins the rest in rounded fp32 additions. Final states of 65536 tokens of one
// sign with almost no decay are off by 4e-6 of their value in one pass and 6e-6 in segments (7.6e-4 and 4.3e-5 with the whole
// state as the accumulator; the steps that mend it cost 2 to 6%: 8 x 4096 x 64 heads 269 -> 275 us, 8 packed prompts
// 158 -> 168).
//
// Decays are kept as base-2 logarithms, relative to 32-token blocks: e^{c_i - c_j} is a row factor times
// a column factor, one exponential per row and block. Across blocks both are at most 1; inside a block
// the row factor undoes the column factor beyond the row. fp32 holds both where the block decays by less than
// 2^100 and no column factor times its step size is below the normal range; the gate warp marks the other
// blocks, which take an exponential per element. (A third way was tried and left out: the row factors taken out of
// M and applied to the finished row where a chunk decays by less than 2^64; no faster.)
//
// Measured on B200: 7.6 K cycles (4.4 us at 1.73 GHz) per chunk and slot pair with one CTA on every SM, against 1.5 us for
// the pair's 64 KB of x and y at the copy bandwidth; 8 x 4096 tokens of 64 heads of 64 in 275 us at full clocks (256 CTAs in
// two waves; 305 when the power cap holds the SMs at 1.76 GHz), token by token 6.3 ms. No unit is full (on the
// fullest SM: tensor pipe 47%, shared memory 44%; issue slots 68% on its fullest quarter): two loops of dependent steps take about
// the same time, G - M - scaling of y - M X - next G, and state operand - output tile - X'^T - state product. Slots are 64
// channels wide, so P of 80 or 96 takes the time of 128, and P below 64 that of 64. What led here (times of the
// version before the state's remainder):
//   - shared memory feeds the MMAs' operands besides everything else (an MMA of 128 x 128 x 16 with both
//     operands there takes all of its 128 bytes a cycle), so the two operands that the warps form, M and X'^T,
//     are in TMEM;
//   - the kernel is sensitive to instruction fetch: with 90 instead of 63 KB of code the same steps took 315
//     instead of 262 us. So there is one copy of each step and loops stay rolled;
//   - plain pointers into shared memory load through the generic path (304 against 269 us).
// No faster, and left out: twenty-four working warps, M shared by all sixteen, all of X'^T in warps 0-7, three
// x buffers with one B buffer.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <mutex>

#include "gdn_common.cuh"
#include "gdn_ssm.h"
#include "selective_scan.cuh"
#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

constexpr int CH = 128;      // tokens per chunk
constexpr int TILE = 64;     // channels per slot
constexpr int PIECE = 32;    // tokens per piece of X'
constexpr int PIECES = CH / PIECE;
constexpr int WARPS = 20;
constexpr int CHUNK_THREADS = 32 * WARPS;

// ---- shared memory (bytes from a 1024-aligned base); bf16 tiles in the 128-byte swizzle TMA writes:
// panels of 64 columns, rows of 128 bytes
constexpr uint32_t PANEL = CH * 128;                 // 16 KB
constexpr uint32_t OFF_B = 0;                        // 2 buffers x 2 panels [128 tokens][64 state]
constexpr uint32_t OFF_C = OFF_B + 4 * PANEL;        // 2 panels
constexpr uint32_t OFF_X = OFF_C + 2 * PANEL;        // 2 buffers x 2 slots [128 tokens][64 channels]; becomes y
constexpr uint32_t OFF_S = OFF_X + 4 * PANEL;        // 2 panels [128 slot channels][64 state]
constexpr uint32_t OFF_GATE = OFF_S + 2 * PANEL;     // 2 buffers x 2 slots x Gates
constexpr uint32_t GATE_BYTES = 4 * CH * 4;
constexpr uint32_t OFF_MISC = OFF_GATE + 4 * GATE_BYTES;
constexpr uint32_t MISC_SUMS = 0;                    // block sums [2 buffers][2 slots][4]
constexpr uint32_t MISC_BAR = 64;
constexpr uint32_t MISC_TMEM = 344;
constexpr uint32_t MISC_SEG = 348;                   // the CTA's segment and slots:
enum { SEG_SEQ, SEG_J, SEG_COUNT, SEG_ROW, SEG_LEN, SEG_HEAD, SEG_TILE = SEG_HEAD + 2, SEG_SECOND = SEG_TILE + 2,
       SEG_GROUP, SEG_WORDS };
constexpr uint32_t MISC_EXP = 400;                   // [2 buffers][2 slots]: bit b, block b needs an exponential per element
constexpr uint32_t MISC_BYTES = 448;
static_assert(MISC_SEG + 4 * SEG_WORDS <= MISC_EXP && MISC_EXP + 16 <= MISC_BYTES, "segment words overflow");
constexpr uint32_t CHUNK_SMEM = OFF_MISC + MISC_BYTES + 1024;
static_assert(CHUNK_SMEM <= 232448, "exceeds the 227 KB per-block shared memory limit");

// Gates of one slot and chunk (floats): prefix sums of a inside each 32-block, d, h_j = 2^{sum of a
// behind j in its block} d_j, w_j = 2^{sum of a behind j in the chunk} d_j.
constexpr int GT_C = 0, GT_D = CH, GT_H = 2 * CH, GT_W = 3 * CH;

// ---- TMEM columns (all 128 lanes)
constexpr uint32_t TM_G = 0;     // G fp32 [token i][token j]; in place of block b's 32 columns M as bf16
                                 // pairs, 16 columns per slot
constexpr uint32_t TM_Y = 128;   // y fp32 [token][slot, channel]
constexpr uint32_t TM_S = 256;   // S fp32 [slot, channel][state]
constexpr uint32_t TM_X = 384;   // X'^T bf16 pairs [slot, channel][token]: 2 pieces x 3 terms x 16 columns
constexpr uint32_t TM_XP = 48;   // columns per piece
// (state pass: pieces from column 0 on, two accumulators at TM_S and TM_S + 128)
constexpr int GROUP = 4;         // chunks that a state pass accumulates in TMEM before it adds them to its sum

// Barriers. *F full, *E empty. A phase is waited for by its parity, so a waiter may neither skip a
// phase nor let two complete before it looks: every waiter below waits for each phase of its barrier
// in turn (or behind a wait that implies the phase before), and what it does next is needed for the
// phase after.
enum {
    B_XF = 0, B_XE = 2,  // (XE: state pass)
    B_BF = 4,
    B_CF = 6,
    B_GF = 7,   // G in TMEM
    B_ID = 8,   // inter product done (y's columns written, C tile free)
    B_MR = 9,   // M written, y scaled, G read
    B_YD = 10,  // intra product done
    B_YF = 11,  // y's columns read
    B_SC = 12,  // state operand written and state decayed
    B_SD = 13,  // state product done
    B_RF = 14, B_RE = 18,  // pieces of X'^T, one pair of barriers per piece of a chunk: written, read
    B_PF = 22, B_PE = 24,  // gates
    B_YS = 26,             // output tile written, per slot and buffer
    B_DR = 30,             // every MMA of an issuing thread done (exit)
    B_BE = 32,             // B buffers read
    NBARS = 34
};
static_assert(MISC_BAR + 8 * NBARS <= MISC_TMEM, "barriers overlap the TMEM address word");

struct ChunkParams {
    CUtensorMap tm_x, tm_b, tm_c, tm_y;
    ScanArgs a;
    float4* part;      // state pass: final states of segments, [segment][unit][state / 4][slot, channel]
    float* part_log;   // and their log2 decays, [segment][unit][slot]
    unsigned int* status;
    int ptiles;        // slots per head
    int pairs;         // slot pairs per group
    int units;         // G * pairs
    int seg_tokens;    // tokens per segment (a multiple of 128), 0: one segment per sequence
    int segments;      // segments that part and part_log have room for
    int withhold;      // test hook: chunk of each segment whose x tiles are never loaded (-1: none)
};

// The rest of a wait whose first test failed, out of line (the kernel has some thirty waits and is
// sensitive to instruction fetch): false, and bits 0 and 16 of the status word, when it ran out.
__device__ __noinline__ bool scan_wait(uint32_t bar, uint32_t parity, unsigned int* status) {
    if (ptx::mbar_wait_compact(bar, parity, WAIT_ITERS)) return true;
    atomicOr(status, 1u | (1u << 16));
    return false;
}

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// 32 TMEM columns as raw words, so that they can be changed and stored from the same registers.
__device__ __forceinline__ void tmem_ld32u(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void scale32(uint32_t (&r)[32], uint64_t f) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        float x0, x1;
        f2_unpack(f2_mul(f2_pack(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), f), x0, x1);
        r[j] = __float_as_uint(x0);
        r[j + 1] = __float_as_uint(x1);
    }
}
// A bf16 pair as two fp32 values, by the byte selector of its first half, or zeros.
constexpr uint32_t HALF_VALUE = 0x1044, HALF_ZERO = 0x4444;
__device__ __forceinline__ uint64_t halves(uint32_t u, uint32_t first) {
    return f2_pack(__uint_as_float(__byte_perm(u, 0, first)), __uint_as_float(__byte_perm(u, 0, first + 0x2200)));
}
// Address of a row of a 1024-aligned swizzled panel; its 16-byte chunk c is at that address ^ (c << 4).
__device__ __forceinline__ uint32_t row_at(uint32_t panel, int row) { return panel + row * 128 + ((row & 7) << 4); }
// Makes a value opaque here, so that what is derived from it is formed in place and not kept in
// registers over a loop.
__device__ __forceinline__ void keep_local(uint32_t& v) { asm volatile("" : "+r"(v)); }
// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v|, with log(1 + e) = 2 atanh(z), z = e / (2 + e) <= 1/3, by
// its power series (the first term left out is below 2^-27 of the sum). Accurate relative to the result
// for v down to -87 (0 below, where e^v leaves fp32's normal range), in a third of the instructions of log1pf(expf(v)), whose eight copies a chunk the one gate
// warp has no time for.
__device__ __forceinline__ float softplus_series(float v) {
    float x = -fabsf(v);
    x = x < -200.f ? -200.f : x;  // (NaN stays)
    const float t = x * LOG2E;
    const float rest = fmaf(x, 1.9259630e-8f, fmaf(x, LOG2E, -t));  // what the product's and the constant's rounding left out
    const float e = ex2f(t) * fmaf(rest, 0.69314718f, 1.f);
    const float z = __fdividef(e, 2.f + e), q = z * z;
    float s = fmaf(q, 1.f / 15.f, 1.f / 13.f);
    s = fmaf(q, s, 1.f / 11.f);
    s = fmaf(q, s, 1.f / 9.f);
    s = fmaf(q, s, 1.f / 7.f);
    s = fmaf(q, s, 1.f / 5.f);
    s = fmaf(q, s, 1.f / 3.f);
    s = fmaf(q, s, 1.f);
    return (v > 0.f ? v : 0.f) + 2.f * z * s;
}
__device__ __forceinline__ float lds1(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ void sts1(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void sts4(uint32_t addr, float4 v) {
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
// o <- bf16 pairs of v[j] h[j] f, in a diagonal block only where bit j of `keep` is set, else 0 (a
// select, not a product with zero: rows behind a sequence may hold anything). h: a shared-memory address.
template <bool kDiagonal>
__device__ __forceinline__ void form_m(const uint32_t (&v)[32], uint32_t (&o)[16], uint32_t h, float f, uint32_t keep) {
    const uint64_t ff = f2_pack(f, f);
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 h4 = lds4(h + 4 * j);
        float x0, x1, x2, x3;
        f2_unpack(f2_mul(f2_mul(f2_pack(h4.x, h4.y), ff), f2_pack(__uint_as_float(v[j]), __uint_as_float(v[j + 1]))), x0, x1);
        f2_unpack(f2_mul(f2_mul(f2_pack(h4.z, h4.w), ff), f2_pack(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]))), x2, x3);
        if (kDiagonal) {
            x0 = keep & (1u << j) ? x0 : 0.f;
            x1 = keep & (2u << j) ? x1 : 0.f;
            x2 = keep & (4u << j) ? x2 : 0.f;
            x3 = keep & (8u << j) ? x3 : 0.f;
        }
        o[j / 2] = pack_bf16(x0, x1);
        o[j / 2 + 1] = pack_bf16(x2, x3);
    }
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
    return v;
}
// One thread of a converged warp. Issuing threads are chosen by this and not by lane index: the compiler
// then keeps an MMA's descriptors in uniform registers, without which an issue takes 80 cycles and more
// (measured: 128 x 128 x 16 every 66 cycles against 89, 128 x 64 with A in TMEM 32 against 79).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ uint32_t top_halves(float a, float b) {  // bf16 pair of the leading halves
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
__device__ __forceinline__ float head(float a) { return __uint_as_float(__float_as_uint(a) & 0xFFFF0000u); }

// Segment sid of the call: sequence (a.N: there is none), segment j of `count` in it. One warp.
__device__ __forceinline__ void find_segment(const ScanArgs& a, int seg_tokens, int sid, int lane, int& seq, int& j, int& count) {
    seq = sid, j = 0, count = 1;
    if (seg_tokens > 0 && a.cu == nullptr) {
        count = (a.T - 1) / seg_tokens + 1;  // (no sum: T may be near 2^31; a call that is cut has tokens)
        seq = sid / count;
        j = sid - seq * count;
    } else if (seg_tokens == 0 && a.cu != nullptr && a.N <= 32) {  // packed: the longest sequences first
        int64_t b = 0, e = -1;
        if (lane < a.N) seq_range(a.cu, lane, a.T, b, e);
        const int n = (int)(e - b);
        int rank = 0;
#pragma unroll 1
        for (int o = 0; o < 32; ++o) {
            const int other = __shfl_sync(0xffffffffu, n, o);
            rank += other > n || (other == n && o < lane);
        }
        const unsigned hit = __ballot_sync(0xffffffffu, lane < a.N && rank == sid);
        seq = hit ? __ffs(hit) - 1 : a.N;
    } else if (seg_tokens > 0) {  // packed: segments in the order of the sequences
        int base = 0;
        seq = a.N;
        for (int s0 = 0; s0 < a.N; s0 += 32) {
            int n = 0;
            if (s0 + lane < a.N) {
                int64_t b, e;
                seq_range(a.cu, s0 + lane, a.T, b, e);
                n = max(1, (int)((e - b + seg_tokens - 1) / seg_tokens));
            }
            int inc = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, inc, off);
                if (lane >= off) inc += t;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, base + inc > sid);
            if (hit) {
                const int src = __ffs(hit) - 1;
                seq = s0 + src;
                count = __shfl_sync(0xffffffffu, n, src);
                j = sid - (base + __shfl_sync(0xffffffffu, inc, src) - count);
                break;
            }
            base += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}

// kState: the state pass of a segmented call: every segment but a sequence's last from a zero state. With
// weights that decay to the segment's end (chunks in reverse order, the later chunks' decay carried along)
// the state is one long product: no decay of the state, no chain between chunks, four pieces in flight. Groups
// of GROUP chunks take turns in two accumulators; warps 8-15 add each finished one to a sum in shared memory.
// The segment's final state and log decay go to part / part_log, no output.
template <bool kState>
__global__ void __launch_bounds__(CHUNK_THREADS, 1) scan_chunk_kernel(const __grid_constant__ ChunkParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sb = ptx::smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const ScanArgs& a = p.a;
    volatile int* seg = reinterpret_cast<volatile int*>(smem + OFF_MISC + MISC_SEG);
    const uint32_t bar0 = sb + OFF_MISC + MISC_BAR;
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };

    if (kState) ptx::grid_launch_dependents();
    // ---- this CTA's segment ----
    if (warp == 0) {
        const int unit = blockIdx.x % p.units, sid = blockIdx.x / p.units;
        int seq, j, count;
        find_segment(a, p.seg_tokens, sid, lane, seq, j, count);
        if (lane == 0) {
            int64_t b = 0, e = 0;
            if (seq < a.N) seq_range(a.cu, seq, a.T, b, e);
            // rows fit 31 bits (checked by the launcher)
            const int begin = (int)b + j * p.seg_tokens;
            seg[SEG_SEQ] = seq;
            seg[SEG_J] = j;
            seg[SEG_COUNT] = count;
            seg[SEG_ROW] = begin;
            seg[SEG_LEN] = (p.seg_tokens > 0) ? min(p.seg_tokens, (int)e - begin) : (int)(e - b);
            // slots: head and channel tile; an odd one out runs its slot twice and stores it once
            const int g = unit / p.pairs, r_heads = a.H / a.G, first_slot = 2 * (unit - g * p.pairs);
            const bool second = first_slot + 1 < r_heads * p.ptiles;
            for (int s = 0; s < 2; ++s) {
                const int slot = first_slot + (second ? s : 0);
                seg[SEG_HEAD + s] = g * r_heads + slot / p.ptiles;
                seg[SEG_TILE + s] = slot % p.ptiles * TILE;
            }
            seg[SEG_SECOND] = second;
            seg[SEG_GROUP] = g;
        }
    }
    if (tid == 32) {
        for (int i = 0; i < NBARS; ++i) {
            int n = 1;
            if (i == B_MR || i == B_YF || i == B_SC) n = 8;
            if (i >= B_RF && i < B_RF + PIECES) n = 4;
            if (i == B_PE || i == B_PE + 1) n = 16;
            if (i == B_XE || i == B_XE + 1) n = 16;
            if (i >= B_YS && i < B_YS + 4) n = 4;
            ptx::mbar_init(bar(i), n);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 16) {
        ptx::tmem_alloc(sb + OFF_MISC + MISC_TMEM, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + OFF_MISC + MISC_TMEM);
    // What a role needs of these it reads where it needs it: kept in registers over the roles' loops they
    // cost spills.
    const int len = seg[SEG_LEN];
    // no such segment (the grid covers the most there can be); the state pass skips last segments
    const bool idle = seg[SEG_SEQ] >= a.N || (kState && seg[SEG_J] == seg[SEG_COUNT] - 1);
    const int nc = idle ? 0 : (len + CH - 1) / CH;
    auto slot_head = [&](int s) { return (int)seg[SEG_HEAD + s]; };
    auto slot_tile = [&](int s) { return (int)seg[SEG_TILE + s]; };
    const int npanel = a.NS > 64 ? 2 : 1;

    // Waits are bounded. After one ran out a thread waits for nothing more: warps finish their loops on
    // whatever is there (every access stays in its buffer), issuing threads stop.
    bool dead = false;
    auto wait = [&](int b, uint32_t parity) {
        if (!dead && !ptx::mbar_test_wait(bar(b), parity & 1u)) dead = !scan_wait(bar(b), parity & 1u, p.status);
    };
    auto warp_wait = [&](int b, uint32_t parity) {
        wait(b, parity);
        __syncwarp();
    };
    // first token row of chunk k of the walk
    auto chunk_row = [&](int row0, int k) { return row0 + CH * (kState ? nc - 1 - k : k); };
    auto b_off = [](int k) { return OFF_B + (uint32_t)(k & 1) * 2 * PANEL; };
    // Warps 0-15: one warp of a warpgroup polls (`f` waits), the others sleep in a named barrier until it has
    // seen all: twenty polling warps took a third of the issue slots.
    auto team_wait = [&](auto&& f) {
        if ((warp & 3) == 0) f();
        ptx::named_sync(1 + (warp >> 2), 128);
    };
    auto warp_arrive = [&](int b) {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(b));
    };
    // gates and block sums as shared-memory addresses (plain pointers would load through the generic path)
    auto gates = [&](int buf, int s) { return sb + OFF_GATE + (uint32_t)(2 * buf + s) * GATE_BYTES; };
    auto sums = [&](int buf, int s) { return sb + OFF_MISC + MISC_SUMS + (uint32_t)(2 * buf + s) * 16; };
    auto exps = [&](int buf, int s) { return sb + OFF_MISC + MISC_EXP + (uint32_t)(2 * buf + s) * 4; };
    const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16);  // this warp's TMEM lane quarter
    // State pass, group g of its chunks: accumulated (each accumulator has barriers of its own, so that no phase
    // of one can pass unseen behind the other's) and read by the warps that add it up.
    auto sum_done = [](int g) { return g & 1 ? B_YD : B_SD; };
    auto sum_read = [](int g) { return g & 1 ? B_MR : B_SC; };

    // ---- X'^T (warps 0-15): warpgroup i forms piece i of a chunk, 32 tokens; a thread one slot channel
    // (TMEM lane), whose tokens it reads down a column of the x tile (64 contiguous bytes a warp).
    const int wg = warp >> 2, quarter = warp & 3, row = 32 * quarter + lane;
    auto piece = [&](int k) {
        const int s = quarter >> 1, p = row & 63;
        uint32_t gt = gates(k & 1, s) + 4 * (GT_W + PIECE * wg);
        // token t of the piece: rows of 128 bytes whose 16-byte chunks are swizzled by t & 7
        uint32_t at = sb + OFF_X + (2 * (k & 1) + s) * PANEL + PIECE * wg * 128 + ((p >> 3) << 4) + ((p & 7) << 1);
        uint32_t to = tl + (kState ? TM_G + TM_XP * wg : TM_X + TM_XP * (wg & 1));
        ptx::tc_fence_after();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            uint32_t hi[8], mid[8], lo[8];
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const float4 w4 = lds4(gt + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const int t = j + e;
                    const uint32_t x0 = ld_shared_u16((at ^ ((t & 7) << 4)) + t * 128), x1 = ld_shared_u16((at ^ (((t + 1) & 7) << 4)) + (t + 1) * 128);
                    const uint64_t v = f2_mul(f2_pack(__uint_as_float(x0 << 16), __uint_as_float(x1 << 16)),
                                              e ? f2_pack(w4.z, w4.w) : f2_pack(w4.x, w4.y));
                    float v0, v1, r0, r1, l0, l1;
                    f2_unpack(v, v0, v1);
                    hi[(j + e) / 2] = top_halves(v0, v1);
                    const uint64_t r = f2_sub(v, f2_pack(head(v0), head(v1)));
                    f2_unpack(r, r0, r1);
                    mid[(j + e) / 2] = top_halves(r0, r1);
                    f2_unpack(f2_sub(r, f2_pack(head(r0), head(r1))), l0, l1);
                    lo[(j + e) / 2] = top_halves(l0, l1);
                }
            }
            ptx::tmem_st8(to, hi);
            ptx::tmem_st8(to + 16, mid);
            ptx::tmem_st8(to + 32, lo);
            at += 16 * 128;
            to += 8;
            gt += 64;
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        warp_arrive(B_RF + wg);
    };
    // The rows behind the sequence in its last tiles belong to others and may hold anything: zeros, as
    // their products would otherwise reach valid rows as 0 x NaN. Rows [lo, hi) of a panel, by one warpgroup.
    auto zero_rows = [&](uint32_t panel, int lo, int hi) {
#pragma unroll 1
        for (int e = tid & 127; e < (hi - lo) * 8; e += 128) st_shared_v4(row_at(panel, lo + (e >> 3)) ^ ((e & 7) << 4), 0, 0, 0, 0);
        ptx::fence_proxy_async_smem();
    };
    auto zero_x = [&](int k, int valid) {  // this warpgroup's tokens, both slots
        if (valid >= PIECE * (wg + 1)) return;
#pragma unroll 1
        for (int s = 0; s < 2; ++s) zero_rows(sb + OFF_X + (2 * (k & 1) + s) * PANEL, max(valid, PIECE * wg), PIECE * (wg + 1));
    };
    // Both slots of one head (a head of more than 64 channels, or an odd slot run twice): one M for both.
    const bool twin = seg[SEG_HEAD] == seg[SEG_HEAD + 1];

    if (warp < 16) {
        // Warps 0-7: M and the scaling of y of chunk k, then pieces 0 and 1 of chunk k + 1.
        // Warps 8-15: the state at chunk k, the output tile of chunk k - 1, then pieces 2 and 3 of chunk k.
        // One loop and one copy of each part: the kernel is sensitive to instruction fetch.
        const bool second_half = warp >= 8;
        const int cols = wg & 1;  // y: slot; state: 64-column panel
        const uint32_t tm_s = tl + TM_S + 64 * cols, tm_y = tl + TM_Y + 64 * cols;
        // S = decay x (its bf16 copy in shared memory) + (TMEM): see the state's step below
        float decay = 0.f;
        uint32_t half = HALF_VALUE;
        auto copy_row = [&]() {
            uint32_t at = row_at(sb + OFF_S + cols * PANEL, row);
            keep_local(at);
            return at;
        };
        const uint32_t kept = sb + (cols ? OFF_S : OFF_C) + 16 * row;  // state pass: the sum, [state / 4][row] of this panel
        float D = 0.f;
        if (!kState && second_half && a.D != nullptr) D = a.D[slot_head(cols)];
        if (!kState && second_half && !idle) {  // entry state: the initial state, or the one that scan_entry_kernel left
            const int s = quarter >> 1, ch = slot_tile(s) + (row & 63);
            const bool later = seg[SEG_J] > 0;
            if (later) ptx::grid_dependency_wait();
            const size_t sbase = (((size_t)seg[SEG_SEQ] * a.H + slot_head(s)) * a.P + ch) * a.NS + 64 * cols;
            const bool inside = !kState && a.s0 != nullptr && ch < a.P;
            const uint32_t copy = copy_row();
            bool wild = false;
#pragma unroll 1
            for (int q4 = 0; q4 < 4; ++q4) {
                float v[16];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (64 * cols + 16 * q4 + 4 * c < a.NS) {
                        if (later) f = p.part[((size_t)blockIdx.x * 32 + 16 * cols + 4 * q4 + c) * CH + row];
                        else if (inside) f = *reinterpret_cast<const float4*>(a.s0 + sbase + 16 * q4 + 4 * c);
                    }
                    v[4 * c] = f.x, v[4 * c + 1] = f.y, v[4 * c + 2] = f.z, v[4 * c + 3] = f.w;
                    wild |= !(fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))) < 3.38e38f);
                    if (c & 1) st_shared_v4(copy ^ ((2 * q4 + (c >> 1)) << 4), 0, 0, 0, 0);
                }
                uint32_t o[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(v[c]);
                ptx::tmem_st16(tm_s + 16 * q4, o);
            }
            ptx::tmem_wait_st();
            // infinities (and what bf16 rounds to them) have no remainder: such a state stays whole in TMEM
            if (__any_sync(0xffffffffu, wild)) half = HALF_ZERO;
        }
        auto output = [&](int k) {  // y = Y + D x, in place of x
            const int buf = k & 1, valid = min(CH, len - CH * k), s = cols;
            team_wait([&] { wait(B_YD, k); });
            ptx::tc_fence_after();
            uint32_t xt = row_at(sb + OFF_X + (2 * buf + s) * PANEL, row);
            keep_local(xt);
            const uint64_t dd = f2_pack(D, D);
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
                float v[32];
                uint32_t x[16];
                ptx::tmem_ld32(tm_y + 32 * hf, v);
#pragma unroll
                for (int c = 0; c < 4; ++c) ld_shared_v4(xt ^ ((4 * hf + c) << 4), x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
                ptx::tmem_wait_ld();
                if (hf == 1) {
                    ptx::tc_fence_before();
                    warp_arrive(B_YF);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t at = xt ^ ((4 * hf + c) << 4);
                    uint32_t u[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        float x0, x1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(x[4 * c + t] << 16), __uint_as_float(x[4 * c + t] & 0xFFFF0000u)), dd,
                                         f2_pack(v[8 * c + 2 * t], v[8 * c + 2 * t + 1])),
                                  x0, x1);
                        u[t] = pack_bf16(x0, x1);
                    }
                    st_shared_v4(at, u[0], u[1], u[2], u[3]);
                }
            }
            if (valid == CH) {
                ptx::fence_proxy_async_smem();
                warp_arrive(B_YS + 2 * s + buf);
            } else if (row < valid && (s == 0 || seg[SEG_SECOND])) {  // the rows of a partial tile, each by its thread
                const int c0 = slot_tile(s);
                __nv_bfloat16* yr = a.y + (((int64_t)seg[SEG_ROW] + CH * k + row) * a.H + slot_head(s)) * a.P + c0;
                for (int c = 0; c < 8 && c0 + 8 * c < a.P; ++c) {
                    uint32_t u[4];
                    ld_shared_v4(xt ^ (c << 4), u[0], u[1], u[2], u[3]);
                    *reinterpret_cast<uint4*>(yr + 8 * c) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
        };
        if constexpr (kState) {  // (segments of the state pass are whole chunks)
#pragma unroll 1
            for (int k = 0; k < nc; ++k) {
                const int buf = k & 1;
                team_wait([&] {
                    wait(B_PF + buf, (uint32_t)k >> 1);
                    wait(B_XF + buf, (uint32_t)k >> 1);
                    if (k > 0) wait(B_RE + wg, k - 1);
                });
                piece(k);
                if (lane == 0) {
                    ptx::mbar_arrive(bar(B_PE + buf));
                    ptx::mbar_arrive(bar(B_XE + buf));
                }
                if (second_half && k > 0 && k % GROUP == 0) {  // the group before this chunk's, onto the sum
                    const int g = k / GROUP - 1;
                    team_wait([&] { wait(sum_done(g), (uint32_t)g >> 1); });
                    ptx::tc_fence_after();
#pragma unroll 1
                    for (int q4 = 0; q4 < 4; ++q4) {
                        float v[16];
                        ptx::tmem_ld16(tm_s + 128 * (g & 1) + 16 * q4, v);
                        ptx::tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t at = kept + (4 * q4 + c) * (CH * 16);
                            float4 f = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                            if (g > 0) f = add4(f, lds4(at));
                            sts4(at, f);
                        }
                    }
                    ptx::tc_fence_before();
                    warp_arrive(sum_read(g));
                }
            }
            if (second_half && nc > 0) {
                team_wait([&] { wait(sum_done((nc - 1) / GROUP), (uint32_t)((nc - 1) / GROUP) >> 1); });
                ptx::tc_fence_after();
            }
        } else {
#pragma unroll 1
        for (int k = second_half ? 0 : -1; k < nc + (second_half ? 1 : 0); ++k) {
            const int buf = k & 1;
            if (second_half) {
                const int valid = min(CH, len - CH * k);
                if (k < nc) {
                    // The state S: a bf16 copy as the operand of C S^T, and the decay of the rest over this chunk.
                    // The tensor cores cut off the bits of a sum below its last place, 24 times a chunk: with
                    // the whole state as the accumulator its error grew by 1.5e-6 of it a chunk, all one way
                    // (7.6e-4 after 65536 tokens of inputs of one sign). So TMEM holds only what the copy's
                    // rounding left out, and takes the chunk's sum onto that; S is put together again here, in
                    // fp32 with one rounding.
                    team_wait([&] {
                        wait(B_PF + buf, (uint32_t)k >> 1);
                        if (k > 0) wait(B_SD, k - 1);
                        if (k > 0) wait(B_ID, k - 1);  // the last operand has been read
                    });
                    ptx::tc_fence_after();
                    if (cols < npanel) {
                        const float4 R = lds4(sums(buf, quarter >> 1));
                        const float total = (R.x + R.y) + (R.z + R.w);
                        const uint64_t before = f2_pack(decay, decay);
                        decay = ex2f(total);
                        const uint64_t dd = f2_pack(decay, decay);
#pragma unroll 1
                        for (int hf = 0; hf < 2; ++hf) {
                            uint32_t v[32];
                            tmem_ld32u(tm_s + 32 * hf, v);
                            ptx::tmem_wait_ld();
                            const uint32_t at = copy_row();
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t u[4];
                                ld_shared_v4(at ^ ((4 * hf + c) << 4), u[0], u[1], u[2], u[3]);
#pragma unroll
                                for (int t = 0; t < 4; ++t) {
                                    uint32_t &v0 = v[8 * c + 2 * t], &v1 = v[8 * c + 2 * t + 1];
                                    const uint64_t S = f2_fma(halves(u[t], half), before, f2_pack(__uint_as_float(v0), __uint_as_float(v1)));
                                    float x0, x1;
                                    f2_unpack(S, x0, x1);
                                    u[t] = pack_bf16(x0, x1);
                                    f2_unpack(f2_mul(f2_sub(S, halves(u[t], half)), dd), x0, x1);
                                    v0 = __float_as_uint(x0), v1 = __float_as_uint(x1);
                                }
                                st_shared_v4(at ^ ((4 * hf + c) << 4), u[0], u[1], u[2], u[3]);
                            }
                            ptx::tmem_st32(tm_s + 32 * hf, v);
                        }
                        ptx::tmem_wait_st();
                    }
                    if (valid < CH) {  // before any product of this chunk's state (and of its M X)
                        team_wait([&] {
                            wait(B_BF + buf, (uint32_t)k >> 1);
                            wait(B_XF + buf, (uint32_t)k >> 1);
                        });
                        if (cols < npanel) zero_rows(sb + b_off(k) + cols * PANEL, valid, CH);
                        zero_x(k, valid);
                    }
                    ptx::fence_proxy_async_smem();
                    ptx::tc_fence_before();
                    warp_arrive(B_SC);
                } else if (nc > 0) {
                    team_wait([&] { wait(B_SD, nc - 1); });
                    ptx::tc_fence_after();
                }
                if (k > 0) output(k - 1);
            } else if (k >= 0) {
                const int q = quarter;
                {
                    team_wait([&] { wait(B_GF, k); });
                    ptx::tc_fence_after();
                    // M_ij = G_ij h_j 2^{c_i + (sum of a over the blocks between)}: blocks 0, 2 of this warp's
                    // rows here, 1, 3 in the warp of the other group on the same TMEM lanes
#pragma unroll 1
                    for (int b = wg; b < 4; b += 2) {
                        uint32_t v[32];
                        const uint32_t at = tl + TM_G + 32 * b;
                        if (b > q) {  // right of the diagonal
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0;
                            ptx::tmem_st32(at, v);
                            continue;
                        }
                        tmem_ld32u(at, v);
                        ptx::tmem_wait_ld();
#pragma unroll 1
                        for (int s = 0; s < (twin ? 1 : 2); ++s) {
                            const uint32_t gt = gates(buf, s), R = sums(buf, s);
                            const float ci = lds1(gt + 4 * (GT_C + row));
                            uint32_t o[16];
                            if (b < q) {
                                float e = ci;
#pragma unroll 1
                                for (int m = b + 1; m < q; ++m) e += lds1(R + 4 * m);
                                form_m<false>(v, o, gt + 4 * (GT_H + 32 * b), ex2f(e), 0);
                            } else if (!(__float_as_uint(lds1(exps(buf, s))) >> q & 1)) {  // the row factor undoes h_j's 2^{R - c_j} beyond i
                                form_m<true>(v, o, gt + 4 * (GT_H + 32 * b), ex2f(ci - lds1(R + 4 * q)), (2u << lane) - 1u);
                            } else {  // factors beyond fp32's range inside the block: an exponential per element
#pragma unroll
                                for (int j = 0; j < 32; j += 4) {
                                    const float4 c4 = lds4(gt + 4 * (GT_C + 32 * q + j)), d4 = lds4(gt + 4 * (GT_D + 32 * q + j));
                                    const float x0 = j <= lane ? __uint_as_float(v[j]) * (ex2f(ci - c4.x) * d4.x) : 0.f;
                                    const float x1 = j + 1 <= lane ? __uint_as_float(v[j + 1]) * (ex2f(ci - c4.y) * d4.y) : 0.f;
                                    const float x2 = j + 2 <= lane ? __uint_as_float(v[j + 2]) * (ex2f(ci - c4.z) * d4.z) : 0.f;
                                    const float x3 = j + 3 <= lane ? __uint_as_float(v[j + 3]) * (ex2f(ci - c4.w) * d4.w) : 0.f;
                                    o[j / 2] = pack_bf16(x0, x1);
                                    o[j / 2 + 1] = pack_bf16(x2, x3);
                                }
                            }
                            ptx::tmem_st16(at + 16 * s, o);
                        }
                    }
                    // Y <- e^{c_i} (C S^T), so that M X accumulates onto it
                    float e = lds1(gates(buf, wg) + 4 * (GT_C + row));
#pragma unroll 1
                    for (int m = 0; m < q; ++m) e += lds1(sums(buf, wg) + 4 * m);
                    e = ex2f(e);
                    const uint64_t ee = f2_pack(e, e);
                    team_wait([&] { wait(B_ID, k); });
                    ptx::tc_fence_after();
#pragma unroll 1
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t v[32];
                        tmem_ld32u(tm_y + 32 * hf, v);
                        ptx::tmem_wait_ld();
                        scale32(v, ee);
                        ptx::tmem_st32(tm_y + 32 * hf, v);
                    }
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    warp_arrive(B_MR);
                }
                if (lane == 0) ptx::mbar_arrive(bar(B_PE + buf));
            }
            const int kp = second_half ? k : k + 1;
            if (kp < nc) {
                team_wait([&] {
                    if (!second_half) wait(B_PF + (kp & 1), (uint32_t)kp >> 1);
                    wait(B_XF + (kp & 1), (uint32_t)kp >> 1);
                    // the piece's columns: read by the products of the piece two before it
                    if (second_half) wait(B_RE + wg - 2, kp);
                    else if (kp > 0) wait(B_RE + wg + 2, kp - 1);
                });
                if (len - CH * kp < CH) {
                    if (!second_half) zero_x(kp, len - CH * kp);
                    ptx::named_sync(1 + wg, 128);
                }
                piece(kp);
                if (second_half) warp_arrive(B_PE + buf);
            }
        }
        }
        if (second_half && !idle && (kState || seg[SEG_J] == seg[SEG_COUNT] - 1)) {
            const int last = kState ? (nc - 1) / GROUP : 0;
            const uint64_t before = f2_pack(decay, decay);
            const uint32_t copy = copy_row();
            const int s = quarter >> 1, ch = slot_tile(s) + (row & 63);
            const size_t sbase = (((size_t)seg[SEG_SEQ] * a.H + slot_head(s)) * a.P + ch) * a.NS + 64 * cols;
            const bool inside = ch < a.P && (s == 0 || seg[SEG_SECOND]);
#pragma unroll 1
            for (int q4 = 0; q4 < 4; ++q4) {
                float v[16];
                ptx::tmem_ld16(tm_s + 128 * (last & 1) + 16 * q4, v);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float4 f = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                    if (kState) {
                        if (last > 0) f = add4(f, lds4(kept + (4 * q4 + c) * (CH * 16)));
                    } else {
                        const uint32_t at = (copy ^ ((2 * q4 + (c >> 1)) << 4)) + 8 * (c & 1);
                        f2_unpack(f2_fma(halves(__float_as_uint(lds1(at)), half), before, f2_pack(f.x, f.y)), f.x, f.y);
                        f2_unpack(f2_fma(halves(__float_as_uint(lds1(at + 4)), half), before, f2_pack(f.z, f.w)), f.z, f.w);
                    }
                    if (kState)
                        p.part[((size_t)blockIdx.x * 32 + 16 * cols + 4 * q4 + c) * CH + row] = f;
                    else if (inside && 64 * cols + 16 * q4 + 4 * c < a.NS)
                        *reinterpret_cast<float4*>(a.sf + sbase + 16 * q4 + 4 * c) = f;
                }
            }
        }
    } else if (warp == 16 || warp == 19) {
        // ================= MMA issue (one thread of each warp) =================
        if (elect_one()) {
            // (inline waits: behind a call the compiler no longer keeps the descriptors uniform)
            auto wait = [&](int b, uint32_t parity) {
                if (!dead && !ptx::mbar_wait_compact(bar(b), parity & 1u, WAIT_ITERS)) {
                    dead = true;
                    atomicOr(p.status, 1u | (1u << 16));
                }
            };
            constexpr uint32_t ID_G = ptx::idesc_bf16(128, 128, 0, 0, 0);      // C B^T, C S^T
            constexpr uint32_t ID_INTRA = ptx::idesc_bf16(128, 64, 0, 1, 0);   // M X         (A in TMEM, B MN-major)
            constexpr uint32_t ID_TWIN = ptx::idesc_bf16(128, 128, 0, 1, 0);   // M X of both slots
            const uint32_t d16 = ptx::sw128_desc_lo(sb, 16), dpanel = ptx::sw128_desc_lo(sb, PANEL);
            auto desc = [](uint32_t base, uint32_t off) { return ptx::desc_pair(base + (off >> 4), ptx::sw128_desc_hi(1024)); };
            auto kmajor = [](int st) { return (uint32_t)(st >> 2) * PANEL + (uint32_t)(st & 3) * 32u; };
            const int ks = (a.NS + 15) / 16;  // 16-column steps of the state dimension
            if (warp == 16) {
                const uint32_t id_state = ptx::idesc_bf16(128, 16 * ks, 0, 1, 0);  // X'^T B  (A in TMEM, B MN-major)
                for (int k = 0; k < nc; ++k) {
                    wait(B_BF + (k & 1), (uint32_t)k >> 1);
                    if (!kState) wait(B_SC, k);
                    const int g = kState ? k / GROUP : 0;
                    if (kState && k % GROUP == 0 && g >= 2) wait(sum_read(g), (uint32_t)(g - 2) >> 1);
#pragma unroll 1
                    for (int i = 0; i < PIECES; ++i) {
                        wait(B_RF + i, k);
                        if (dead) break;
                        ptx::tc_fence_after();
#pragma unroll
                        for (int st = 0; st < PIECE / 16; ++st)
#pragma unroll
                            for (int term = 0; term < 3; ++term)
                                ptx::mma_bf16_ts(tmem + TM_S + 128 * (g & 1),
                                                 tmem + (kState ? TM_G + TM_XP * i : TM_X + TM_XP * (i & 1)) + 16 * term + 8 * st,
                                                 desc(dpanel, b_off(k) + (uint32_t)(PIECE * i + 16 * st) * 128u), id_state,
                                                 !kState || k % GROUP + i + st + term > 0);
                        ptx::mma_commit(bar(B_RE + i));
                    }
                    if (dead) break;
                    if (kState ? k % GROUP == GROUP - 1 || k == nc - 1 : true) ptx::mma_commit(bar(kState ? sum_done(g) : B_SD));
                    ptx::mma_commit(bar(B_BE + (k & 1)));
                }
            } else if (!kState) {
                auto issue_g = [&](int k) {
                    wait(B_BF + (k & 1), (uint32_t)k >> 1);
                    wait(B_CF, k);
                    if (dead) return;
                    ptx::tc_fence_after();
#pragma unroll 2
                    for (int st = 0; st < ks; ++st)
                            ptx::mma_bf16(tmem + TM_G, desc(d16, OFF_C + kmajor(st)), desc(d16, b_off(k) + kmajor(st)), ID_G, st > 0);
                    ptx::mma_commit(bar(B_GF));
                };
                if (nc > 0) issue_g(0);
                for (int k = 0; k < nc; ++k) {
                    wait(B_SC, k);
                    if (k > 0) wait(B_YF, k - 1);
                    if (dead) break;
                    ptx::tc_fence_after();
#pragma unroll 2
                    for (int st = 0; st < ks; ++st)
                            ptx::mma_bf16(tmem + TM_Y, desc(d16, OFF_C + kmajor(st)), desc(d16, OFF_S + kmajor(st)), ID_G, st > 0);
                    ptx::mma_commit(bar(B_ID));
                    wait(B_MR, k);
                    if (dead) break;
                    ptx::tc_fence_after();
                    const uint32_t xo = OFF_X + (uint32_t)(k & 1) * 2 * PANEL;
                    if (twin) {
#pragma unroll 2
                        for (int st = 0; st < CH / 16; ++st)
                            ptx::mma_bf16_ts(tmem + TM_Y, tmem + TM_G + 32 * (st >> 1) + 8 * (st & 1), desc(dpanel, xo + st * 2048u), ID_TWIN, 1);
                    } else {
#pragma unroll 1
                        for (int s = 0; s < 2; ++s)
#pragma unroll 2
                            for (int st = 0; st < CH / 16; ++st)
                                ptx::mma_bf16_ts(tmem + TM_Y + 64 * s, tmem + TM_G + 32 * (st >> 1) + 16 * s + 8 * (st & 1),
                                                 desc(d16, xo + s * PANEL + st * 2048u), ID_INTRA, 1);
                    }
                    ptx::mma_commit(bar(B_YD));
                    wait(B_YD, k);  // M has been read: G takes its place
                    if (k + 1 < nc) issue_g(k + 1);
                    if (dead) break;
                }
            }
            // nothing in flight when the CTA leaves
            const bool failed = dead;
            dead = false;
            ptx::mma_commit(bar(B_DR + (warp == 19)));
            wait(B_DR + (warp == 19), 0);
            dead |= failed;
        }
        __syncwarp();
    } else if (warp == 17) {
        // ================= TMA (one thread) =================
        if (elect_one()) {
            ptx::prefetch_tensormap(&p.tm_x);
            ptx::prefetch_tensormap(&p.tm_b);
            if (!kState) ptx::prefetch_tensormap(&p.tm_c);
            const int h0 = slot_head(0), h1 = slot_head(1), t0 = slot_tile(0), t1 = slot_tile(1), row0 = seg[SEG_ROW], g = seg[SEG_GROUP];
            const bool second = seg[SEG_SECOND];
            int nb = 0, nx = 0, ncl = 0;  // loads issued (nx: up to this chunk)
            auto load_b = [&](int k) {
                if (dead || k >= nc) return;
                ++nb;
                ptx::mbar_arrive_expect_tx(bar(B_BF + (k & 1)), npanel * PANEL);
#pragma unroll 1
                for (int c = 0; c < npanel; ++c)
                    ptx::tma_load_4d(sb + b_off(k) + c * PANEL, &p.tm_b, bar(B_BF + (k & 1)), 64 * c, g, chunk_row(row0, k), 0);
            };
            auto load_c = [&](int k) {
                if (dead || k >= nc) return;
                ++ncl;
                ptx::mbar_arrive_expect_tx(bar(B_CF), npanel * PANEL);
#pragma unroll 1
                for (int c = 0; c < npanel; ++c) ptx::tma_load_4d(sb + OFF_C + c * PANEL, &p.tm_c, bar(B_CF), 64 * c, g, row0 + CH * k, 0);
            };
            auto load_x = [&](int k) {
                if (dead || k >= nc || k == p.withhold) return;
                nx = k + 1;
                const int buf = k & 1;
                ptx::mbar_arrive_expect_tx(bar(B_XF + buf), 2 * PANEL);
                ptx::tma_load_4d(sb + OFF_X + 2 * buf * PANEL, &p.tm_x, bar(B_XF + buf), t0, h0, chunk_row(row0, k), 0);
                ptx::tma_load_4d(sb + OFF_X + (2 * buf + 1) * PANEL, &p.tm_x, bar(B_XF + buf), t1, h1, chunk_row(row0, k), 0);
            };
#pragma unroll 1
            for (int k = -2; k < nc && !dead; ++k) {  // (one copy of each load: the first two rounds only fill the buffers)
                const int buf = k & 1;
                if constexpr (kState) {
                    if (k >= 0) wait(B_XE + buf, (uint32_t)k >> 1);
                    load_x(k + 2);
                    if (k >= 0) wait(B_BE + buf, (uint32_t)k >> 1);
                    load_b(k + 2);
                } else {
                    if (k >= 0 && k + 1 < nc)  // the next C tile on its way to L2 while its buffer is in use
#pragma unroll 1
                        for (int c = 0; c < npanel; ++c) ptx::tma_prefetch_4d(&p.tm_c, 64 * c, g, row0 + CH * (k + 1), 0);
                    if (k >= 0) wait(B_ID, k);  // (behind it, by the same thread, G of this chunk: B is free with the state product)
                    if (k >= -1) load_c(k + 1);
                    if (k >= 0) wait(B_BE + buf, (uint32_t)k >> 1);
                    load_b(k + 2);
                    if (k >= 0 && len - CH * k >= CH) {  // a full tile: out by TMA (the warps store a partial one themselves)
                        const int row = row0 + CH * k;
#pragma unroll 1
                        for (int s = 0; s < 2; ++s) {
                            wait(B_YS + 2 * s + buf, (uint32_t)k >> 1);
                            if (!dead && (s == 0 || second))
                                tma_store_4d(&p.tm_y, sb + OFF_X + (2 * buf + s) * PANEL, s ? t1 : t0, s ? h1 : h0, row, 0);
                        }
                        ptx::bulk_wait_read_all();
                    }
                    load_x(k + 2);  // (chunk k + 2 exists: chunk k was full)
                }
            }
            // nothing in flight when the CTA leaves
            auto landed = [&](int b, uint32_t parity) {  // (each wait by itself, whatever ran out before)
                dead = false;
                wait(b, parity);
            };
            for (int buf = 0; buf < 2; ++buf) {
                if (nb > buf) landed(B_BF + buf, (uint32_t)(nb - 1 - buf) >> 1);
                if (nx > buf) landed(B_XF + buf, (uint32_t)(nx - 1 - buf) >> 1);
            }
            if (ncl > 0) landed(B_CF, (uint32_t)(ncl - 1));
            ptx::bulk_wait_all();
        }
        __syncwarp();
    } else if (warp == 18) {
        // ================= gates of both slots =================
        float A2[2], bias[2], next[2][4], later[2] = {0.f, 0.f};  // (later: log2 decay of the chunks behind, state pass)
        const int h0 = slot_head(0), h1 = slot_head(1);
        const int64_t row0 = seg[SEG_ROW];
        A2[0] = a.A[h0] * LOG2E, A2[1] = a.A[h1] * LOG2E;
        bias[0] = a.dt_bias ? a.dt_bias[h0] : 0.f, bias[1] = a.dt_bias ? a.dt_bias[h1] : 0.f;
#pragma unroll 1
        for (int k = -1; k < nc; ++k) {
            float ahead[2][4];  // the next chunk's steps, four tokens a lane, clamped to the segment's rows
            if (k + 1 < nc) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t at = (row0 + min(chunk_row(0, k + 1) + 4 * lane + i, len - 1)) * a.dts;
                    ahead[0][i] = a.dt_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.dt)[at + h0]) : static_cast<const float*>(a.dt)[at + h0];
                    ahead[1][i] = a.dt_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.dt)[at + h1]) : static_cast<const float*>(a.dt)[at + h1];
                }
            }
            const int buf = k & 1, valid = kState ? CH : len - CH * k;
            if (k >= 2) warp_wait(B_PE + buf, ((uint32_t)k >> 1) - 1);
#pragma unroll 1
            for (int s = 0; k >= 0 && s < 2; ++s) {
            float d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[i] = (s ? next[1][i] : next[0][i]) + (s ? bias[1] : bias[0]);
                if (a.softplus) d[i] = softplus_series(d[i]);
                d[i] = 4 * lane + i < valid ? d[i] : 0.f;
            }
            const uint32_t gt = gates(buf, s) + 16 * lane;
            const float A2s = s ? A2[1] : A2[0];
            // log2 decays, clamped: 2^-256 is zero like any smaller factor, and the distances of the tokens
            // behind such a step are differences of sums that hold it (one step of 256 leaves them 2^-16,
            // a block of 32 of them 2^-11). NaN stays; rows behind the sequence count nothing, whatever A is.
            float t[4], pre[4], suf[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[i] = d[i] * A2s;
                t[i] = t[i] < -256.f ? -256.f : t[i];
                t[i] = 4 * lane + i < valid ? t[i] : 0.f;
            }
            pre[0] = t[0], pre[1] = t[0] + t[1], pre[2] = pre[1] + t[2], pre[3] = pre[2] + t[3];
            suf[3] = 0.f, suf[2] = t[3], suf[1] = t[3] + t[2], suf[0] = suf[1] + t[1];
            // sums over the 8 lanes of a 32-token block, from the left and, for the accuracy of the
            // short distances, from the right
            float inc = pre[3], dec = pre[3];
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) {
                const float u = __shfl_up_sync(0xffffffffu, inc, off, 8), v = __shfl_down_sync(0xffffffffu, dec, off, 8);
                if ((lane & 7) >= off) inc += u;
                if ((lane & 7) + off < 8) dec += v;
            }
            float left = __shfl_up_sync(0xffffffffu, inc, 1, 8), right = __shfl_down_sync(0xffffffffu, dec, 1, 8);
            if ((lane & 7) == 0) left = 0.f;
            if ((lane & 7) == 7) right = 0.f;
            float R[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) R[b] = __shfl_sync(0xffffffffu, inc, 8 * b + 7);
            float behind = 0.f;
#pragma unroll
            for (int b = 3; b > 0; --b)
                if (b > (lane >> 3)) behind += R[b];
            if (kState) {
                behind += s ? later[1] : later[0];
                const float total = (R[0] + R[1]) + (R[2] + R[3]);
                if (s) later[1] += total;
                else later[0] += total;
            }
            const float f = ex2f(behind);
            const float hv[4] = {ex2f(right + suf[0]) * d[0], ex2f(right + suf[1]) * d[1], ex2f(right + suf[2]) * d[2],
                                 ex2f(right + suf[3]) * d[3]};
            sts4(gt + 4 * GT_D, make_float4(d[0], d[1], d[2], d[3]));
            sts4(gt + 4 * GT_C, make_float4(left + pre[0], left + pre[1], left + pre[2], left + pre[3]));
            sts4(gt + 4 * GT_W, make_float4(hv[0] * f, hv[1] * f, hv[2] * f, hv[3] * f));
            sts4(gt + 4 * GT_H, make_float4(hv[0], hv[1], hv[2], hv[3]));
            // (NaN steps and decays count as out of range: the element form keeps them to the tokens behind)
            bool out = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) out |= d[i] != 0.f && !(fabsf(hv[i]) >= 1.17549435e-38f);
            const unsigned outs = __ballot_sync(0xffffffffu, out);
            if (lane == 0) {
                uint32_t e = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) e |= ((outs >> (8 * b) & 0xffu) != 0 || !(R[b] > -100.f)) ? 1u << b : 0u;
                sts4(sums(buf, s), make_float4(R[0], R[1], R[2], R[3]));
                sts1(exps(buf, s), __uint_as_float(e));
            }
            }
            if (k >= 0) warp_arrive(B_PF + buf);
#pragma unroll
            for (int i = 0; i < 4; ++i) next[0][i] = ahead[0][i], next[1][i] = ahead[1][i];
        }
        if (kState && !idle && lane == 0) p.part_log[2 * (size_t)blockIdx.x] = later[0], p.part_log[2 * (size_t)blockIdx.x + 1] = later[1];
    }
    // an output pass ends after the passes before it, whether or not it needed them (the next launch in the
    // stream waits for this one only)
    if (!kState) ptx::grid_dependency_wait();
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == 16) ptx::tmem_dealloc(tmem, 512);
}

// Entry states of the segments of each sequence, in place of their final states in `part`: from the
// sequence's initial state, E_{j+1} = 2^{log_j} E_j + A_j. A thread owns a float4 of one (sequence, unit) and
// walks the segments, eight of them loaded ahead.
__global__ void __launch_bounds__(256) scan_entry_kernel(const __grid_constant__ ChunkParams p) {
    __shared__ int found[2];
    const ScanArgs& a = p.a;
    const int unit = blockIdx.x % p.units, seq = blockIdx.x / p.units, lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        int first = 0, count = 1;
        if (a.cu == nullptr) {
            count = (a.T - 1) / p.seg_tokens + 1;
            first = seq * count;
        } else {
            for (int s0 = 0; s0 <= seq; s0 += 32) {  // segments of the sequences before
                int n = 0;
                if (s0 + lane <= seq) {
                    int64_t b, e;
                    seq_range(a.cu, s0 + lane, a.T, b, e);
                    n = max(1, (int)((e - b + p.seg_tokens - 1) / p.seg_tokens));
                }
                const int own = __shfl_sync(0xffffffffu, n, (seq - s0) & 31);
                if (s0 + 32 > seq) {
                    count = own;
                    if (lane == seq - s0) n = 0;
                }
                first += __reduce_add_sync(0xffffffffu, n);
            }
        }
        if (lane == 0) found[0] = first, found[1] = count;
    }
    __syncthreads();
    // The scratch holds the segments of sequences that do not overlap. Offsets that are out of order can make
    // overlapping ones of the clamped ranges: what lies behind the scratch is no segment of this call. (No
    // overflow: a call is cut only with fewer than 4 x 148 sequences and at most 64 segments of a mean one.)
    const int first = found[0], count = min(found[1], p.segments - first);
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();  // the state pass's results
    if (count < 2) return;
    const int g = unit / p.pairs, r_heads = a.H / a.G, slot0 = 2 * (unit - g * p.pairs);
    const bool second = slot0 + 1 < r_heads * p.ptiles;
    const int el = blockIdx.y * 256 + threadIdx.x, row = el & (CH - 1), n4 = el / CH, s = row >> 6;
    const int slot = slot0 + (second ? s : 0), h = g * r_heads + slot / p.ptiles, ch = slot % p.ptiles * TILE + (row & 63);
    float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.s0 != nullptr && ch < a.P && 4 * n4 < a.NS)
        S = *reinterpret_cast<const float4*>(a.s0 + (((size_t)seq * a.H + h) * a.P + ch) * a.NS + 4 * n4);
    const size_t step = (size_t)p.units * 32 * CH;
    float4* at = p.part + ((size_t)first * p.units + unit) * 32 * CH + el;
    const float* lg = p.part_log + 2 * ((size_t)first * p.units + unit) + s;
    constexpr int AHEAD = 8;
    for (int j0 = 0; j0 + 1 < count; j0 += AHEAD) {  // the state behind segment j is the entry state of j + 1
        float4 A[AHEAD];
        float l[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (j0 + i + 1 < count) A[i] = at[i * step], l[i] = lg[2 * (size_t)p.units * i];
        // the last segment has no final state of its own here: its place only receives
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (j0 + i + 1 < count) {
                if (j0 + i > 0) at[i * step] = S;
                const float d = ex2f(l[i]);
                S = make_float4(fmaf(d, S.x, A[i].x), fmaf(d, S.y, A[i].y), fmaf(d, S.z, A[i].z), fmaf(d, S.w, A[i].w));
                if (j0 + i + 2 == count) at[(i + 1) * step] = S;
            }
        at += AHEAD * step;
        lg += 2 * (size_t)p.units * AHEAD;
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
    static std::once_flag once;
    static EncodeFn fn = nullptr;
    std::call_once(once, []() {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(ptr);
    });
    return fn;
}

// bf16 [rows][units][width] with a row stride; box 64 x 1 x 128 rows, 128-byte swizzle, zeros outside.
static bool row_map(CUtensorMap* m, const void* base, int width, int units, int64_t rows, int64_t stride) {
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)units, (cuuint64_t)rows, 1};
    cuuint64_t strides[3] = {(cuuint64_t)width * 2, (cuuint64_t)stride * 2, (cuuint64_t)stride * 2 * (cuuint64_t)rows};
    cuuint32_t box[4] = {64, 1, CH, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static cudaError_t chunk_smem_attr() {
    static std::atomic<uint64_t> done_mask{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = (dev < 64) ? (1ull << dev) : 0;
    if (bit && (done_mask.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    for (auto fn : {scan_chunk_kernel<false>, scan_chunk_kernel<true>}) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)CHUNK_SMEM);
        if (e != cudaSuccess) return e;
    }
    if (bit) done_mask.fetch_or(bit, std::memory_order_acq_rel);
    return cudaSuccess;
}

ChunkPlan plan_scan_chunks(int N, int T, bool packed, int H, int P, int G, int sms) {
    ChunkPlan pl{};
    const int ptiles = (P + TILE - 1) / TILE;
    pl.pairs = (H / G * ptiles + 1) / 2;
    pl.units = G * pl.pairs;
    pl.segments = N;
    const int64_t rows = packed ? T : (int64_t)N * T;
    const int64_t chunks = N > 0 ? (rows / N + CH - 1) / CH : 0;  // of the mean sequence
    // Wave model, measured on B200: an output pass takes 4.4 us per chunk and pair and 9.5 for a CTA's start
    // and end, a state pass 2 and 5, the entry states 5. Segments pay where the (sequence, pair) units
    // alone leave SMs idle (65536 tokens over 8 slots: 2.2 ms in one pass, 110 us in 37 segments). A
    // packed batch's longest sequence is taken as twice the mean (the longest ones start first); a batch with one much
    // longer prompt is not cut and takes that prompt's time (16384 beside 7 x 512, 64 heads of 64 in 8 groups: 510 us).
    constexpr double OUT = 4.4, OUT_FIXED = 9.5, STATE = 2.0, STATE_FIXED = 5.0, ENTRY = 5.0;
    const int64_t ctas = (int64_t)N * pl.units;
    auto waves = [&](int64_t n) { return (double)((n + sms - 1) / sms); };
    const double one = OUT * chunks + OUT_FIXED;
    double best = waves(ctas) * one;
    if (packed && N > 1) {
        const double spread = ctas * one / sms + OUT * chunks / 2, longest = 2 * OUT * chunks + OUT_FIXED;
        best = spread > longest ? spread : longest;
    }
    for (int64_t s = 2; s <= chunks && s <= 64 && ctas * (s - 1) < 4 * sms; ++s) {
        const int64_t per = (chunks + s - 1) / s, cut = (chunks + per - 1) / per;
        if (cut < 2) continue;
        const double t = waves(ctas * cut) * (OUT * per + OUT_FIXED) + waves(ctas * (cut - 1)) * (STATE * per + STATE_FIXED) + ENTRY;
        if (t < best) {
            best = t;
            pl.seg_tokens = (int)(per * CH);
            pl.segments = packed ? (int64_t)T / pl.seg_tokens + N : (int64_t)N * ((T - 1) / pl.seg_tokens + 1);
        }
    }
    const int64_t parts = pl.seg_tokens > 0 ? pl.segments * pl.units * 2 : 0;
    pl.part_bytes = (size_t)parts * TILE * CH * 4;
    pl.log_bytes = ((size_t)parts * 4 + 255) / 256 * 256;
    return pl;
}

cudaError_t launch_scan_chunks(const ScanArgs& a, const ChunkPlan& pl, int64_t rows, void* workspace, void* scratch,
                               int withhold, cudaStream_t stream) {
    ChunkParams p;
    memset(&p, 0, sizeof(p));
    if (!row_map(&p.tm_x, a.x, a.P, a.H, rows, a.xs) || !row_map(&p.tm_b, a.B, a.NS, a.G, rows, a.bs) ||
        !row_map(&p.tm_c, a.C, a.NS, a.G, rows, a.cs) || !row_map(&p.tm_y, a.y, a.P, a.H, rows, (int64_t)a.H * a.P))
        return cudaErrorInvalidValue;
    cudaError_t e = chunk_smem_attr();
    if (e != cudaSuccess) return e;
    p.a = a;
    p.status = static_cast<unsigned int*>(workspace);
    p.part_log = static_cast<float*>(scratch);
    p.part = reinterpret_cast<float4*>(static_cast<uint8_t*>(scratch) + pl.log_bytes);
    p.ptiles = (a.P + TILE - 1) / TILE;
    p.pairs = pl.pairs;
    p.units = pl.units;
    p.seg_tokens = pl.seg_tokens;
    p.segments = (int)pl.segments;
    p.withhold = withhold;
    const int64_t ctas = pl.segments * pl.units;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (pl.seg_tokens == 0) {
        scan_chunk_kernel<false><<<(unsigned)ctas, CHUNK_THREADS, CHUNK_SMEM, stream>>>(p);
        return cudaGetLastError();
    }
    // State pass, entry states, output pass. The second and third are launched while the one before still
    // runs (programmatic dependent launch) and wait for it where they read what it wrote; the first waits
    // for the stream as usual, so the inputs are ready for all three.
    scan_chunk_kernel<true><<<(unsigned)ctas, CHUNK_THREADS, CHUNK_SMEM, stream>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(a.N * pl.units), 32 * CH / 256, 1);
    cfg.blockDim = dim3(256, 1, 1);
    if ((e = cudaLaunchKernelEx(&cfg, scan_entry_kernel, p)) != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)ctas, 1, 1);
    cfg.blockDim = dim3(CHUNK_THREADS, 1, 1);
    cfg.dynamicSmemBytes = CHUNK_SMEM;
    return cudaLaunchKernelEx(&cfg, scan_chunk_kernel<false>, p);
}

}  // namespace ssm
}  // namespace gdn
