// A linear layer with everything that follows it in the epilogue, for sm_100a: y = act(x W^T + b) + r, and the products and
// the element-wise pass of its gradient.
//
//   forward          y [rows, out]  = act(x [rows, dim] W[out, dim]^T + b) + r,   optionally 2^15 act'(x W^T + b) in fp16
//   dz = dy act'     element-wise, with the column sums that are the gradient of b
//   dx [rows, dim] = dz W           the contraction runs over W's rows: W is an MN-major operand
//   dW [out, dim]  = dz^T x         both operands MN-major
//
// All products are D[i, j] = sum_k A[i, k] B[j, k] on tcgen05 with fp32 accumulators in tensor memory, operands brought by
// TMA into 128-byte-swizzled tiles: K-major tiles of [rows x 64 k], or MN-major ones of two panels [64 k x 64 rows], so
// that no operand is ever transposed in memory.  The forms:
//
//   linear_pair_kernel    many rows.  Persistent pairs of CTAs (cta_group::2), output tiles of 256 rows x 64 .. 256 columns, two
//                         accumulators in turn so that the epilogue of one tile runs under the products of the next; bound by
//                         the tensor pipe (and, in long runs, by the power cap).  Measured: 4096 x 4096 -> 14336 bf16 with
//                         GELU and bias 306 us = 1573 TFLOP/s alone, tensor pipe 91 % busy; 1999 x 1408 -> 2048 fp16 with SiLU,
//                         bias and residual 17.7 us (one tile a pair: its parts follow one another).
//   linear_shared_pair_kernel  the same for few tiles: two or four pairs share a tile along K (dW of 512 x 512 over 16384 rows
//                         17.9 us; 43.8 with a pair a tile).
//   linear_split_kernel   few rows.  The weight is the 128-row operand and the tokens are the columns (16 .. 128 of them): a
//                         block streams a [128 x K / split] slab of the weight through a ring of TMA tiles, one or two blocks
//                         per SM; the blocks of a cluster share an output tile along K and add their fp32 partial sums over
//                         distributed shared memory, in rank order (no atomics, no workspace, one launch).  Bound by the
//                         weight's bytes: 1 row of 4096 -> 14336 bf16 21.7 us = 5.4 TB/s, 48 rows of 14336 -> 4096 24.6 us.
//   linear_grad_act_kernel  6 bytes a value: 4096 x 4096 bf16 18.1 us = 5.6 TB/s, with the column sums 20.5.
//
// Rounding: the epilogue works on the fp32 accumulators and rounds once.  The slope act' is kept in fp16 also beside bf16
// data, times 2^15: it lies in about [-0.13, 1.14], so 2^15 keeps it below fp16's largest value, and down to 2^-29 it has eight
// times the resolution of bf16 (half a step is 2^-11 of it; below that 2^-40 whatever its size): the backward pass adds no
// error of bf16's size by it (z itself in bf16 would).  dz is rounded to the data type before the two products, which take
// 16-bit operands; its column sums are taken before that rounding.
// The polynomial forms (degree 3 .. 6) run the packed 16-bit programs of fpt_unary on z rounded to the data type: what a
// separate product followed by fpt_unary gives, bit for bit.
// Every mbarrier wait is bounded; a wait that runs out writes a word the host can read without a copy and unwinds.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "fpt_common.h"
#include "fpt_programs.h"
#include "fpt_sm100.cuh"

namespace fpt {
namespace {

using namespace sm100;

constexpr int kBlockK = 64;
constexpr uint32_t kTileBytes = 128 * 128;          // 128 rows x 64 values
constexpr uint32_t kPanelBytes = kTileBytes / 2;    // MN-major: 64 k x 64 rows
constexpr int kMaxRing = 12;                        // stages of a ring
constexpr int kBandTiles = 16;                      // 256-row tiles per band: 4096 rows, see fpt_gate_up_swiglu.cu

enum : uint32_t { kWaitEmpty = 0x51, kWaitFull, kWaitAccEmpty, kWaitAccFull };
enum Act : int { kNone, kSigmoid, kTanh, kSwishAct, kGelu, kProgram };   // compile-time: one straight piece of code each

constexpr float kSlopeScale = 32768.0f;             // of act' as it is stored

struct Programs {                      // of kProgram
    int fwd_shape, fwd_degree, bwd_shape, bwd_degree;
    ProgramWords fwd, bwd;
};

struct LinearParams {
    void* out;                      // [m, n] rows of out_ld
    const void* residual;           // [m, n] or null
    const void* bias;               // [n] or null
    uint16_t* slope;                // [m, n] fp16, kSlopeScale act', or null
    int64_t out_ld, res_ld, slope_ld;
    int m, n, k_blocks;             // k_blocks: of 64 (split form), of 64 chunks (pair form)
    int m_tiles, n_tiles;
    int split;                      // blocks (few-row form) or pairs (pair form) of a cluster, which share a tile along K
    int columns;                    // columns of an output tile (pair form), a multiple of 32
    int ring;                       // stages of the ring
    uint32_t stage_bytes;           // their size, and the K blocks of 64 in one (pair form)
    int chunks;
    bool a_whole, b_whole;          // one copy brings an operand's share of a stage
    int bias_dtype;
    bool vec_out, vec_res, vec_slope, vec_bias;
    bool staged;                    // out, residual and slope rows all start on 16-byte boundaries (pair form)
    Programs act;
    uint32_t* status;
};

// ---- waits --------------------------------------------------------------------------------------------------------

// Launched while the kernel before it drains (launch_early below): barriers and tensor memory are set up by then, and nothing of
// global memory is touched before this.  What that kernel writes changes during this one's life, so nothing is read as constant
// (no __ldg, no __restrict__: such a load may be moved ahead of the wait).
__device__ __forceinline__ void wait_for_inputs() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __noinline__ void report(uint32_t* status, uint32_t where) {
    volatile uint32_t* s = status;
    if (s && *s == 0u) *s = 0x80000000u | where;
    __threadfence_system();
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status, uint32_t where) {
    if (mbar_wait(bar, parity, abort_flag, nullptr, where)) return true;
    report(status, where);
    return false;
}

// ---- epilogue arithmetic ------------------------------------------------------------------------------------------

template <int DT>
__device__ __forceinline__ float value16(uint16_t v) {
    return DT == kBf16 ? __uint_as_float(uint32_t(v) << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
    if (dtype == FPT_FP32) return static_cast<const float*>(p)[i];
    const uint16_t v = static_cast<const uint16_t*>(p)[i];
    return dtype == FPT_BF16 ? value16<kBf16>(v) : value16<kFp16>(v);
}

// One program on two lanes with its shape and degree known at run time (the same instructions in the same order as
// eval_program; the branches are uniform).
template <int DT>
__device__ __forceinline__ uint32_t run_program(uint32_t x, const ProgramWords& p, int shape, int degree) {
    using P = Pk<DT>;
    const uint32_t sign = x & kSignMask;
    const uint32_t t = P::min_abs(x, p.clamp);
    const int top = shape == kEven ? degree : degree - 1;
    uint32_t h = p.c[top];
    for (int k = top - 1; k >= 0; --k) h = P::fma(t, h, p.c[k]);
    if (shape == kEven) return h;
    h = P::mul(t, h);
    if (shape == kOdd) return h ^ sign;
    if (shape == kOddSat) return P::min(h, Consts<DT>::one) ^ sign;
    if (shape == kOddHalf) return P::add(Consts<DT>::half, h ^ sign);
    if (shape == kXmulHalf) return P::mul(x, P::add(Consts<DT>::half, h ^ sign));
    return P::fma(x & ~kSignMask, h, P::mul(Consts<DT>::half, x));       // kSwish
}

// P(Z > a) for a standard normal Z and a >= 0, with e = exp(-a^2 / 2): e times a polynomial in t = 1 / (1 + 0.265 a), fitted here to
// erfcx(a / sqrt 2) / 2 by least squares with the weights moved to the largest relative errors: 6.3e-7 of the tail up to
// a = 13.5, where it leaves fp32 (1e-6 with the fp32 steps), so that the tail of GELU is good to a rounding of fp16 as well.
__device__ __forceinline__ float normal_tail(float a, float e) {
    const float t = mufu_rcp(fmaf(a, 0.265f, 1.0f));
    float q = fmaf(t, -0.067787036f, 0.195273099f);
    q = fmaf(t, q, -0.066362908f);
    q = fmaf(t, q, 0.142493326f);
    q = fmaf(t, q, 0.082946594f);
    q = fmaf(t, q, 0.107836780f);
    q = fmaf(t, q, 0.105599835f);
    return q * t * e;
}
// tanh: the quotient of exponentials, and where that cancels (|z| < 0.3) its series to z^9 (next term < 2^-24 of z).  Its slope
// (times kSlopeScale) is 4 r (1 - r) with r = 1 / (1 + e^2z), and 1 - r is e^2z r where r is near 1: 1 - tanh^2 would cancel.
template <bool SLOPE>
__device__ __forceinline__ float tanh_of(float z, float& slope) {
    const float e = mufu_ex2(2.8853900817779268f * z), r = mufu_rcp(1.0f + e);
    if constexpr (SLOPE) slope = 4.0f * kSlopeScale * r * (z < 0.0f ? e * r : 1.0f - r);
    const float far = fmaf(-2.0f, r, 1.0f);
    const float q = z * z;
    float s = fmaf(q, 2.1869488536e-2f, -5.3968253968e-2f);
    s = fmaf(q, s, 1.3333333333e-1f);
    s = fmaf(q, s, -3.3333333333e-1f);
    return fabsf(z) < 0.3f ? fmaf(z * q, s, z) : far;
}
// q = logistic(z), and 1 - q without cancelling
__device__ __forceinline__ float logistic(float z, float& rest) {
    const float e = mufu_ex2(-1.4426950408889634f * z), q = mufu_rcp(1.0f + e);
    rest = z > 0.0f ? e * q : 1.0f - q;
    return q;
}

// z -> act(z), d -> act'(z) kSlopeScale where wanted
template <int DT, int ACT, bool SLOPE, int N>
__device__ __forceinline__ void activate(const Programs& a, float (&z)[N], float (&d)[N]) {
    if constexpr (ACT == kProgram) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint32_t x = Sfu<DT>::pack(z[i], z[i + 1]);
            const uint32_t y = run_program<DT>(x, a.fwd, a.fwd_shape, a.fwd_degree);
            z[i] = Sfu<DT>::lo(y);
            z[i + 1] = Sfu<DT>::hi(y);
            if constexpr (SLOPE) {
                const uint32_t s = run_program<DT>(x, a.bwd, a.bwd_shape, a.bwd_degree);
                d[i] = Sfu<DT>::lo(s) * kSlopeScale;
                d[i + 1] = Sfu<DT>::hi(s) * kSlopeScale;
            }
        }
    } else if constexpr (ACT != kNone) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = z[i];
            if constexpr (ACT == kGelu) {
                const float e = mufu_ex2(-0.72134752044448170368f * x * x), tail = normal_tail(fabsf(x), e);
                const float phi = x < 0.0f ? tail : 1.0f - tail;
                z[i] = x * phi;
                if constexpr (SLOPE) d[i] = fmaf(x * 0.3989422804014327f, e, phi) * kSlopeScale;
            } else if constexpr (ACT == kTanh) {
                z[i] = tanh_of<SLOPE>(x, d[i]);
            } else {
                float rest;
                const float q = logistic(x, rest);
                z[i] = ACT == kSwishAct ? x * q : q;
                if constexpr (SLOPE) d[i] = q * kSlopeScale * (ACT == kSwishAct ? fmaf(x, rest, 1.0f) : rest);
            }
        }
    }
}

// N consecutive columns of one row: bias, activation, residual, stores.  N is a multiple of 4; column a multiple of N.
template <int DT, int ACT, bool SLOPE, int N>
__device__ __forceinline__ void finish(const LinearParams& p, float (&z)[N], int row, int column) {
    constexpr int kWords = N / 2, kVec = kWords >= 4 ? 4 : 2;            // 16-byte accesses, 8-byte ones for N = 4
    using V = std::conditional_t<kVec == 4, uint4, uint2>;
    const bool whole = column + N <= p.n;
    if (p.bias) {
        if (whole && p.vec_bias && p.bias_dtype != FPT_FP32) {
            const V* b = reinterpret_cast<const V*>(static_cast<const uint16_t*>(p.bias) + column);
#pragma unroll
            for (int v = 0; v < kWords / kVec; ++v) {
                const V w = b[v];
                const uint32_t* words = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const uint32_t x = words[i];
                    if (p.bias_dtype == FPT_BF16) {
                        z[2 * (v * kVec + i)] += Sfu<kBf16>::lo(x);
                        z[2 * (v * kVec + i) + 1] += Sfu<kBf16>::hi(x);
                    } else {
                        z[2 * (v * kVec + i)] += Sfu<kFp16>::lo(x);
                        z[2 * (v * kVec + i) + 1] += Sfu<kFp16>::hi(x);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (column + i < p.n) z[i] += load_any(p.bias, p.bias_dtype, column + i);
        }
    }
    float d[N];
    activate<DT, ACT, SLOPE>(p.act, z, d);
    if constexpr (SLOPE) {
        uint16_t* to = p.slope + int64_t(row) * p.slope_ld + column;
        if (whole && p.vec_slope) {
#pragma unroll
            for (int v = 0; v < kWords / kVec; ++v) {
                V w;
                uint32_t* words = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) words[i] = Sfu<kFp16>::pack(d[2 * (v * kVec + i)], d[2 * (v * kVec + i) + 1]);
                reinterpret_cast<V*>(to)[v] = w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (column + i < p.n) to[i] = __half_as_ushort(__float2half_rn(d[i]));
        }
    }
    if (p.residual) {
        const uint16_t* from = static_cast<const uint16_t*>(p.residual) + int64_t(row) * p.res_ld + column;
        if (whole && p.vec_res) {
#pragma unroll
            for (int v = 0; v < kWords / kVec; ++v) {
                const V w = reinterpret_cast<const V*>(from)[v];
                const uint32_t* words = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    z[2 * (v * kVec + i)] += Sfu<DT>::lo(words[i]);
                    z[2 * (v * kVec + i) + 1] += Sfu<DT>::hi(words[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (column + i < p.n) z[i] += value16<DT>(from[i]);
        }
    }
    uint16_t* to = static_cast<uint16_t*>(p.out) + int64_t(row) * p.out_ld + column;
    if (whole && p.vec_out) {
#pragma unroll
        for (int v = 0; v < kWords / kVec; ++v) {
            V w;
            uint32_t* words = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) words[i] = Sfu<DT>::pack(z[2 * (v * kVec + i)], z[2 * (v * kVec + i) + 1]);
            reinterpret_cast<V*>(to)[v] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (column + i < p.n) to[i] = uint16_t(Sfu<DT>::pack(z[i], 0.0f));
    }
}

// ---- the same for a warp that holds 32 rows x 32 columns, a row per lane -------------------------------------------------
//
// A lane's row is 64 contiguous bytes; read or written from registers, a warp's accesses would touch 32 lines with 16 bytes
// each.  The chunk goes through 2 KB of shared memory instead, four lanes to a row: eight rows of 64 bytes per access.  The
// 16-byte piece q of row r lies at piece q ^ (r / 2 % 4): no bank conflicts on either side.

struct Stage {
    alignas(16) uint4 piece[32 * 4];
};
__device__ __forceinline__ int stage_at(int row, int piece) { return row * 4 + (piece ^ ((row >> 1) & 3)); }

// rows `row0 + 8 i + lane / 4`, i = 0 .. 3; `valid` rows exist
__device__ __forceinline__ void load_rows(uint4 (&v)[4], const uint16_t* base, int64_t ld, int lane, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        v[i] = make_uint4(0, 0, 0, 0);
        if (r < valid) v[i] = *reinterpret_cast<const uint4*>(base + int64_t(r) * ld + 8 * (lane & 3));
    }
}
__device__ __forceinline__ void rows_to_stage(Stage& s, const uint4 (&v)[4], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s.piece[stage_at(8 * i + (lane >> 2), lane & 3)] = v[i];
}
__device__ __forceinline__ void stage_to_rows(const Stage& s, uint16_t* base, int64_t ld, int lane, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        const uint4 v = s.piece[stage_at(r, lane & 3)];
        if (r < valid) *reinterpret_cast<uint4*>(base + int64_t(r) * ld + 8 * (lane & 3)) = v;
    }
}

// All 32 lanes, converged.  `res`: this chunk of the residual as load_rows left it (where p.residual); `bias`: of column
// `column + lane` (where p.bias).
template <int DT, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_staged(const LinearParams& p, float (&z)[32], const uint4 (&res)[4], float bias, Stage& s, int row0, int column, int lane) {
    const int valid = p.m - row0;
    if (p.bias) {                                   // a column per lane, read back by all
        float* shared = reinterpret_cast<float*>(s.piece);
        shared[lane] = bias;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 v = reinterpret_cast<const float4*>(shared)[i];
            z[4 * i] += v.x, z[4 * i + 1] += v.y, z[4 * i + 2] += v.z, z[4 * i + 3] += v.w;
        }
        __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {                   // halves: fewer registers
        float (&half)[16] = *reinterpret_cast<float (*)[16]>(z + 16 * h);
        float d[16];
        activate<DT, ACT, SLOPE>(p.act, half, d);
        if constexpr (SLOPE) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
                s.piece[stage_at(lane, 2 * h + q)] = make_uint4(Sfu<kFp16>::pack(d[8 * q], d[8 * q + 1]), Sfu<kFp16>::pack(d[8 * q + 2], d[8 * q + 3]),
                                                                Sfu<kFp16>::pack(d[8 * q + 4], d[8 * q + 5]), Sfu<kFp16>::pack(d[8 * q + 6], d[8 * q + 7]));
        }
    }
    if constexpr (SLOPE) {
        __syncwarp();
        stage_to_rows(s, p.slope + int64_t(row0) * p.slope_ld + column, p.slope_ld, lane, valid);
        __syncwarp();
    }
    if (p.residual) {
        rows_to_stage(s, res, lane);
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint4 v = s.piece[stage_at(lane, q)];
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[8 * q + 2 * i] += Sfu<DT>::lo(words[i]);
                z[8 * q + 2 * i + 1] += Sfu<DT>::hi(words[i]);
            }
        }
        // each lane overwrites its own row next: nobody else reads it before the barrier below
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        s.piece[stage_at(lane, q)] = make_uint4(Sfu<DT>::pack(z[8 * q], z[8 * q + 1]), Sfu<DT>::pack(z[8 * q + 2], z[8 * q + 3]),
                                                Sfu<DT>::pack(z[8 * q + 4], z[8 * q + 5]), Sfu<DT>::pack(z[8 * q + 6], z[8 * q + 7]));
    __syncwarp();
    stage_to_rows(s, static_cast<uint16_t*>(p.out) + int64_t(row0) * p.out_ld + column, p.out_ld, lane, valid);
    __syncwarp();
}

// kind::f16 instruction descriptor with both operands of this data type (umma_idesc_bf16 is the bf16 one)
template <int DT>
__host__ __device__ constexpr uint32_t instruction(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
    return umma_idesc_bf16(m, n, a_mn, b_mn) & (DT == kBf16 ? ~0u : ~((7u << 7) | (7u << 10)));
}
// low word of a tile's shared-memory descriptor, and what one K step of 16 adds to it
template <bool MN>
__device__ __forceinline__ uint32_t tile_lo(const void* tile) { return umma_smem_desc_lo(smem_u32(tile), MN ? kPanelBytes : 16u); }
template <bool MN>
constexpr uint32_t kStep16 = MN ? 2048u / 16u : 2u;

// 16 bytes of shared memory: of any CTA of the cluster (map_to_cta), into this one's
__device__ __forceinline__ float4 load_cluster(uint32_t address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ float load_cluster1(uint32_t address) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ void store_shared(uint32_t address, uint32_t x) {
    asm volatile("st.shared.b32 [%0], %1;" :: "r"(address), "r"(x) : "memory");
}

// ---- many rows: pairs of CTAs ---------------------------------------------------------------------------------------

constexpr uint32_t kRingBytes = 192 * 1024;
constexpr int kChunks = 2;              // K blocks of 64 in a stage
// TMA, product and allocation warps, one idle, eight epilogue warps.  Measured (1999 x 1408 x 2048 fp16, one tile a pair, SiLU,
// bias and residual): 17.3 us with eight, 17.4 with twelve, 18.4 with sixteen (96 registers a thread, spills); one epilogue for
// all activations, chosen at run time, took 23.4.
constexpr int kEpilogueWarps = 8;
constexpr int kPairThreads = 128 + 32 * kEpilogueWarps;

struct PairSmem {
    alignas(1024) uint8_t ring[kRingBytes];        // stages of an A tile and a B tile, as many as fit
    alignas(8) uint64_t full[kMaxRing];
    uint64_t empty[kMaxRing];
    uint64_t acc_full[2], acc_empty[2];
    Stage stage[kEpilogueWarps];
    uint32_t tmem_base;
    uint32_t abort_flag;
};

struct PairTile {
    int row0, column0;
};
// bands of kBandTiles row tiles; inside a band the column tile is the slow index, so that the pairs at work together share
// a few panels of B while the band's rows of A stay in L2
__device__ __forceinline__ PairTile pair_tile(const LinearParams& p, int tile) {
    const int per_band = kBandTiles * p.n_tiles;
    const int band = tile / per_band, r = tile - band * per_band;
    const int in_band = min(kBandTiles, p.m_tiles - band * kBandTiles);
    const int column = r / in_band;
    return PairTile{(band * kBandTiles + r - column * in_band) * 256, column * p.columns};
}

// An operand's share of a stage: `rows` rows (at most 128) x 64 chunks K.  K-major: a tile [rows x 64] per chunk; MN-major: a
// panel [64 chunks k x 64 rows] per 64 rows.  A copy takes the engine some 200 clocks whatever its size (measured: loads
// alone run at 231-273 ns per K block with two copies in it, 20 or 32 KB alike), so where the sizes allow (`whole`) one copy
// brings all tiles or panels, through a map whose third dimension walks over them.
template <bool MN>
__device__ __forceinline__ void load_pair(uint8_t* to, const CUtensorMap* map, uint32_t bar, int kb, int row, int rows, int chunks, bool whole) {
    if constexpr (MN) {
        if (whole) {
            tma_load_4d_pair(to, map, bar, 0, kb * chunks * kBlockK, row / 64, 0);
        } else {
            tma_load_4d_pair(to, map, bar, row, kb * chunks * kBlockK, 0, 0);
            if (rows > 64) tma_load_4d_pair(to + uint32_t(chunks) * kPanelBytes, map, bar, row + 64, kb * chunks * kBlockK, 0, 0);
        }
    } else {
        if (whole) {
            tma_load_4d_pair(to, map, bar, 0, row, kb * chunks, 0);
        } else {
            for (int c = 0; c < chunks; ++c) tma_load_4d_pair(to + uint32_t(c * rows) * 128u, map, bar, (kb * chunks + c) * kBlockK, row, 0, 0);
        }
    }
}
// shared memory of that share
template <bool MN>
__host__ __device__ constexpr uint32_t share_bytes(int rows, int chunks) {
    return MN ? uint32_t((rows + 63) / 64) * uint32_t(chunks) * kPanelBytes : uint32_t(rows * chunks) * 128u;
}
// low word of its descriptor at K step k of 16
template <bool MN>
__device__ __forceinline__ uint32_t share_lo(uint32_t first, uint32_t k, uint32_t rows) {
    return MN ? first + k * (2048u / 16u) : first + k / 4 * (rows * 8u) + k % 4 * 2u;
}

// Each CTA of the pair holds 128 rows of A and half the tile's columns' rows of B and receives 128 rows x p.columns columns of
// D; the hand-overs are those of gate_up_swiglu_pair_kernel.  The host picks the number of columns so that the tiles come
// out even over the pairs.  Where there are only a few tiles (SHARED), the p.split pairs of a cluster share a tile along K, one tile
// a cluster: every CTA finishes a share of the tile's columns and lays the fp32 sums of the others' shares where its ring was,
// a column's 128 rows together (a lane per row: with a row's columns together every lane's read from another CTA is a transfer
// of its own, and the exchange of 256 columns took 4 us more).  The order of the additions is fixed.
template <int DT, int ACT, bool SLOPE, bool A_MN, bool B_MN, bool SHARED>
__device__ __forceinline__ void pair_tiles(const CUtensorMap& map_a, const CUtensorMap& map_b, const LinearParams& p) {
    extern __shared__ uint8_t smem_raw[];
    PairSmem& sm = *reinterpret_cast<PairSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = cluster_cta_rank(), rank = SHARED ? cta & 1u : cta, lead = SHARED ? cta & ~1u : 0u;   // rank in the pair; its first CTA
    const int split = SHARED ? p.split : 1;
    volatile uint32_t* abort_flag = &sm.abort_flag;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.ring; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&sm.acc_full[a], 1);
            mbar_init(&sm.acc_empty[a], 2 * kEpilogueWarps);   // of both CTAs
        }
        sm.abort_flag = 0u;
        mbar_fence_init();
        tma_prefetch_descriptor(&map_a);
        tma_prefetch_descriptor(&map_b);
    }
    if (warp == 2) {
        tmem_alloc_pair(&sm.tmem_base, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    wait_for_inputs();
    const int tiles = p.m_tiles * p.n_tiles;
    const int first_tile = int(blockIdx.x / uint32_t(2 * split)), tile_step = int(gridDim.x / uint32_t(2 * split));
    const int part = SHARED ? int(cta >> 1) : 0;    // of the K blocks
    const int kb0 = SHARED ? int(int64_t(p.k_blocks) * part / split) : 0, kb1 = SHARED ? int(int64_t(p.k_blocks) * (part + 1) / split) : p.k_blocks;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, turn = 0;                       // stage, and how often the ring has gone round
            bool ok = true;
            const int b_rows = p.columns / 2;
            const uint32_t a_bytes = share_bytes<A_MN>(128, p.chunks), bytes = 2 * (a_bytes + share_bytes<B_MN>(b_rows, p.chunks));
            for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
                const PairTile t = pair_tile(p, tile);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (turn > 0) ok = wait(&sm.empty[s], (turn - 1u) & 1u, abort_flag, p.status, kWaitEmpty);
                    if (!ok) break;
                    const uint32_t bar = map_to_cta(smem_u32(&sm.full[s]), lead);
                    uint8_t* stage = sm.ring + s * p.stage_bytes;
                    if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], bytes);
                    load_pair<A_MN>(stage, &map_a, bar, kb, t.row0 + int(rank) * 128, 128, p.chunks, p.a_whole);
                    load_pair<B_MN>(stage + a_bytes, &map_b, bar, kb, t.column0 + int(rank) * b_rows, b_rows, p.chunks, p.b_whole);
                    if (++s == uint32_t(p.ring)) s = 0, ++turn;
                }
            }
        }
    } else if (warp == 1 && rank == 0) {
        const bool elected = elect_one();
        const uint32_t idesc = instruction<DT>(256, uint32_t(p.columns), A_MN, B_MN);
        constexpr uint32_t desc_hi = umma_smem_desc_hi(1024);
        const uint32_t panel = uint32_t(p.chunks) * kPanelBytes, b_rows = uint32_t(p.columns / 2);
        const uint32_t a_first = umma_smem_desc_lo(smem_u32(sm.ring), A_MN ? panel : 16u);
        const uint32_t b_first = umma_smem_desc_lo(smem_u32(sm.ring) + share_bytes<A_MN>(128, p.chunks), B_MN ? panel : 16u);
        uint32_t s = 0, turn = 0, local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step, ++local) {
            const uint32_t a = local & 1u, use = local >> 1;
            if (use > 0) {
                ok = mbar_wait_cluster(&sm.acc_empty[a], (use - 1u) & 1u, abort_flag, nullptr, kWaitAccEmpty);
                if (!ok) {
                    report(p.status, kWaitAccEmpty);
                    break;
                }
                tc_fence_after_sync();
            }
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = wait(&sm.full[s], turn & 1u, abort_flag, p.status, kWaitFull);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t a_lo = a_first + s * (p.stage_bytes / 16u), b_lo = b_first + s * (p.stage_bytes / 16u);
#pragma unroll 4
                for (uint32_t k = 0; k < uint32_t(p.chunks) * (kBlockK / 16); ++k)
                    if (elected) umma_ss_words_pair(tmem + a * 256u, share_lo<A_MN>(a_lo, k, 128), share_lo<B_MN>(b_lo, k, b_rows), desc_hi, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                if (elected) umma_commit_pair(&sm.empty[s], uint16_t(3u << lead));
                if (++s == uint32_t(p.ring)) s = 0, ++turn;
            }
            if (ok && elected) umma_commit_pair(&sm.acc_full[a], uint16_t(3u << lead));
        }
    } else if (warp >= 4) {
        // four warps hold the 128 rows (a warp reads the 32 lanes of its number modulo 4); such sets take the 32-column chunks in
        // turn
        const uint32_t lane_base = uint32_t(32 * (warp & 3)) << 16;
        const int set = (warp - 4) >> 2;
        Stage& stage = sm.stage[warp - 4];
        const int share = SHARED ? p.columns / split : p.columns, c_first = part * share;  // the columns this CTA finishes
        const uint32_t sums = smem_u32(sm.ring) + uint32_t(32 * (warp & 3) + lane) * 4u;       // [column][row of 128]
        uint32_t local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step, ++local) {
            const PairTile t = pair_tile(p, tile);
            const uint32_t a = local & 1u;
            const int row0 = t.row0 + int(rank) * 128 + 32 * (warp & 3), valid = p.m - row0;
            const int column_end = min(p.n, t.column0 + p.columns);
            uint4 res[4];
            float bias = 0.0f;
            const auto prefetch = [&](int column) {                     // residual and bias of a chunk, ahead of its turn
                if (!p.staged || column + 32 > column_end || valid <= 0) return;
                if (p.residual) load_rows(res, static_cast<const uint16_t*>(p.residual) + int64_t(row0) * p.res_ld + column, p.res_ld, lane, valid);
                if (p.bias) bias = load_any(p.bias, p.bias_dtype, column + lane);
            };
            prefetch(t.column0 + c_first + set * 32);
            ok = wait(&sm.acc_full[a], (local >> 1) & 1u, abort_flag, p.status, kWaitAccFull);
            tc_fence_after_sync();
            if constexpr (SHARED) {                 // one tile a cluster: the ring is done with
                if (ok) {
#pragma unroll 1
                    for (int c = set * 32; c < p.columns; c += kEpilogueWarps * 8) {
                        if (c >= c_first && c < c_first + share) continue;      // stays in tensor memory
                        uint32_t acc[32];
                        tmem_ld_32x32b_x32(tmem + lane_base + a * 256u + uint32_t(c), acc);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) store_shared(sums + uint32_t(c + i) * 512u, acc[i]);
                    }
                }
                __syncwarp();
                cluster_sync_all();                 // the other warps' is behind their part
            }
            if (!ok) break;
#pragma unroll 1
            for (int c = c_first + set * 32; c < c_first + share; c += kEpilogueWarps * 8) {
                const int column = t.column0 + c;
                if (column >= p.n || valid <= 0) break;
                uint32_t acc[32];
                tmem_ld_32x32b_x32(tmem + lane_base + a * 256u + uint32_t(c), acc);
                tmem_ld_wait();
                float z[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = __uint_as_float(acc[i]);
                if constexpr (SHARED) {
#pragma unroll 1
                    for (int q = 1; q < split; ++q) {                   // the other pairs' sums, from the next pair round
                        const uint32_t other = (cta + 2u * uint32_t(q)) & uint32_t(2 * split - 1);      // split: a power of two
                        const uint32_t from = map_to_cta(sums + uint32_t(c) * 512u, other);
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = load_cluster1(from + 512u * uint32_t(i));
#pragma unroll
                        for (int i = 0; i < 32; ++i) z[i] += v[i];
                    }
                }
                if (p.staged && column + 32 <= p.n) {
                    const uint4 mine[4] = {res[0], res[1], res[2], res[3]};
                    const float mine_bias = bias;
                    if (!SHARED || c + kEpilogueWarps * 8 < c_first + share) prefetch(column + kEpilogueWarps * 8);
                    finish_staged<DT, ACT, SLOPE>(p, z, mine, mine_bias, stage, row0, column, lane);
                } else {
                    if (lane < valid) finish<DT, ACT, SLOPE>(p, z, row0 + lane, column);
                    __syncwarp();
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(&sm.acc_empty[a]);
                else mbar_arrive_cluster(map_to_cta(smem_u32(&sm.acc_empty[a]), lead));
            }
        }
    }
    if (SHARED && warp < 4) {                       // the barrier between the sums of the cluster and their readers
        __syncwarp();
        cluster_sync_all();
    }
    // no CTA may leave while another can still reach its barriers, its tensor memory or its sums
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync_all();
    if (warp == 2) tmem_dealloc_pair(tmem, 512);
}
template <int DT, int ACT, bool SLOPE, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ LinearParams p) {
    pair_tiles<DT, ACT, SLOPE, A_MN, B_MN, false>(map_a, map_b, p);
}
template <int DT, int ACT, bool SLOPE, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kPairThreads, 1)         // clusters of 2 p.split
linear_shared_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ LinearParams p) {
    pair_tiles<DT, ACT, SLOPE, A_MN, B_MN, true>(map_a, map_b, p);
}

// ---- few rows: the weight streams, the tokens are columns ---------------------------------------------------------------

constexpr int kSplitThreads = 256;
constexpr int kMaxSplit = 8;

// Barriers, then (1024-byte aligned) the ring of weight and token tiles, as many stages as the launch has memory for; after
// the last product its first 512 TOKENS bytes hold this block's sums, [token][output].
struct SplitSmem {
    uint64_t full[kMaxRing], empty[kMaxRing];
    uint64_t acc_full;
    uint32_t tmem_base;
    uint32_t abort_flag;
};
constexpr uint32_t kSplitRingOffset = 1024;
static_assert(sizeof(SplitSmem) <= kSplitRingOffset, "barriers before the ring");

// D is [tokens, outputs] (p.m tokens, p.n outputs); A = the weight, B = the tokens.  The p.split blocks of a cluster take
// equal runs of K blocks.
template <int DT, int ACT, bool SLOPE, int TOKENS, bool W_MN>
__global__ void __launch_bounds__(kSplitThreads, 2)
linear_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearParams p) {
    constexpr uint32_t kXBytes = TOKENS * 128, kStageBytes = kTileBytes + kXBytes;
    constexpr uint32_t kColumns = TOKENS < 32 ? 32 : TOKENS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    SplitSmem& sm = *reinterpret_cast<SplitSmem*>(base);
    uint8_t* ring = base + kSplitRingOffset;
    float (*partial)[128] = reinterpret_cast<float (*)[128]>(ring);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? int(cluster_cta_rank()) : 0;
    volatile uint32_t* abort_flag = &sm.abort_flag;
    const int tile = blockIdx.x / p.split;
    const int output0 = tile / p.m_tiles * 128, token0 = tile % p.m_tiles * TOKENS;
    const int kb0 = int(int64_t(p.k_blocks) * rank / p.split), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / p.split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.ring; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        mbar_init(&sm.acc_full, 1);
        sm.abort_flag = 0u;
        mbar_fence_init();
    }
    if (warp == 2) {
        tmem_alloc(&sm.tmem_base, kColumns);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    wait_for_inputs();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, turn = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (turn > 0 && !wait(&sm.empty[s], (turn - 1u) & 1u, abort_flag, p.status, kWaitEmpty)) break;
                uint8_t* stage = ring + s * kStageBytes;
                mbar_arrive_expect_tx(&sm.full[s], kStageBytes);
                if (W_MN && p.b_whole) {
                    tma_load_4d(stage, &map_w, &sm.full[s], 0, kb * kBlockK, output0 / 64, 0);
                } else if (W_MN) {
                    tma_load_4d(stage, &map_w, &sm.full[s], output0, kb * kBlockK, 0, 0);
                    tma_load_4d(stage + kPanelBytes, &map_w, &sm.full[s], output0 + 64, kb * kBlockK, 0, 0);
                } else if (p.b_whole) {
                    tma_load_4d(stage, &map_w, &sm.full[s], 0, output0, kb, 0);
                } else {
                    tma_load_4d(stage, &map_w, &sm.full[s], kb * kBlockK, output0, 0, 0);
                }
                tma_load_4d(stage + kTileBytes, &map_x, &sm.full[s], kb * kBlockK, token0, 0, 0);
                if (++s == uint32_t(p.ring)) s = 0, ++turn;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool elected = elect_one();
        constexpr uint32_t idesc = instruction<DT>(128, TOKENS, W_MN, false);
        constexpr uint32_t desc_hi = umma_smem_desc_hi(1024);
        const uint32_t w_first = tile_lo<W_MN>(ring), x_first = tile_lo<false>(ring + kTileBytes);
        uint32_t s = 0, turn = 0;
        bool ok = true;
        for (int i = 0; i < kb1 - kb0; ++i) {
            ok = wait(&sm.full[s], turn & 1u, abort_flag, p.status, kWaitFull);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t w_lo = w_first + s * (kStageBytes / 16u), x_lo = x_first + s * (kStageBytes / 16u);
#pragma unroll
            for (uint32_t k = 0; k < kBlockK / 16; ++k)
                if (elected) umma_ss_words(tmem, w_lo + k * kStep16<W_MN>, x_lo + k * kStep16<false>, desc_hi, idesc, (i > 0 || k > 0) ? 1u : 0u);
            if (elected) umma_commit(&sm.empty[s]);
            if (++s == uint32_t(p.ring)) s = 0, ++turn;
        }
        if (ok && elected) umma_commit(&sm.acc_full);
        __syncwarp();
    }
    // every warp: accumulator -> shared memory, transposed to [token][output]
    bool ok = wait(&sm.acc_full, 0u, abort_flag, p.status, kWaitAccFull);
    tc_fence_after_sync();
    __syncwarp();
    if (ok) {
        const uint32_t lane_base = uint32_t(32 * (warp & 3)) << 16;
#pragma unroll 1
        for (int c = (warp >> 2) * 16; c < TOKENS; c += 32) {
            uint32_t acc[16];
            tmem_ld_32x32b_x16(tmem + lane_base + uint32_t(c), acc);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) partial[c + i][32 * (warp & 3) + lane] = __uint_as_float(acc[i]);
        }
    }
    tc_fence_before_sync();
    if (p.split > 1) {
        __syncwarp();
        cluster_sync_all();
    } else {
        __syncthreads();
    }
    if (warp == 2) tmem_dealloc(tmem, kColumns);
    // a warp finishes a row of 128 outputs, four per lane; the rows are dealt out over the cluster
    if (ok) {
        const int output = output0 + 4 * lane;
        const int warps = kSplitThreads / 32 * p.split;
        constexpr int kRows = TOKENS >= 64 ? 2 : 1;            // rows in hand: their reads overlap
#pragma unroll 1
        for (int first = rank * (kSplitThreads / 32) + warp; first < TOKENS && token0 + first < p.m; first += kRows * warps) {
            float z[kRows][4];
            if (p.split > 1) {
                float4 part[kRows][kMaxSplit];
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const uint32_t mine = smem_u32(&partial[min(first + i * warps, TOKENS - 1)][4 * lane]);
#pragma unroll
                    for (int r = 0; r < kMaxSplit; ++r)
                        if (r < p.split) part[i][r] = load_cluster(map_to_cta(mine, uint32_t(r)));
                }
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    z[i][0] = part[i][0].x, z[i][1] = part[i][0].y, z[i][2] = part[i][0].z, z[i][3] = part[i][0].w;
#pragma unroll
                    for (int r = 1; r < kMaxSplit; ++r)
                        if (r < p.split) z[i][0] += part[i][r].x, z[i][1] += part[i][r].y, z[i][2] += part[i][r].z, z[i][3] += part[i][r].w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const float4 v = *reinterpret_cast<const float4*>(&partial[min(first + i * warps, TOKENS - 1)][4 * lane]);
                    z[i][0] = v.x, z[i][1] = v.y, z[i][2] = v.z, z[i][3] = v.w;
                }
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int t = first + i * warps;
                if (t < TOKENS && token0 + t < p.m && output < p.n) finish<DT, ACT, SLOPE>(p, z[i], token0 + t, output);
            }
        }
    }
    if (p.split > 1) {                            // the partial sums stay until the whole cluster has read them
        __syncwarp();
        cluster_sync_all();
    }
}

// ---- the element-wise pass of the gradient ------------------------------------------------------------------------------

constexpr int kActThreads = 256;
constexpr int kActColumns = 256;       // columns a block covers: 32 lanes of 8
constexpr int kActRowLanes = kActThreads / 32;
constexpr int kActBlocks = 5;           // resident on an SM, at 48 registers (asked for of the compiler: 22.4 us instead of 20.5)

struct GradActParams {
    const uint16_t* dy;
    const uint16_t* slope;              // fp16, kSlopeScale act', or null for 1
    uint16_t* dz;                       // or null
    float* partial;                     // [chunks, out] column sums, or null
    int64_t dy_ld, slope_ld, dz_ld;
    int rows, out, chunk_rows;
    bool vec_dy;
};

// dz = dy * act'(z) and the column sums of dz over chunk_rows rows a block
template <int DT>
__global__ void __launch_bounds__(kActThreads) linear_grad_act_kernel(const GradActParams p) {
    __shared__ float sums[kActRowLanes][kActColumns + 1];
    const int lane = threadIdx.x & 31, row_lane = threadIdx.x >> 5;
    const int column = blockIdx.x * kActColumns + 8 * lane;
    const int row_first = int(blockIdx.y) * p.chunk_rows, row_end = row_first + min(p.chunk_rows, p.rows - row_first);   // not past 2^31
    const int live = min(8, p.out - column);                    // columns of this lane that exist
    wait_for_inputs();
    float sum[8] = {};
    if (live > 0) {
#pragma unroll 2
        for (int row = row_first + row_lane; row < row_end; row += kActRowLanes) {
            const uint16_t* dy = p.dy + int64_t(row) * p.dy_ld + column;
            uint32_t g[4] = {0, 0, 0, 0}, s[4] = {0, 0, 0, 0};
            if (p.vec_dy && live == 8) {
                const uint4 v = *reinterpret_cast<const uint4*>(dy);
                g[0] = v.x, g[1] = v.y, g[2] = v.z, g[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < live) g[i / 2] |= uint32_t(dy[i]) << (16 * (i & 1));
            }
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = Sfu<DT>::lo(g[i]);
                v[2 * i + 1] = Sfu<DT>::hi(g[i]);
            }
            if (p.slope) {                                      // rows padded to 16 bytes: whole words may be read
                const uint4 w = *reinterpret_cast<const uint4*>(p.slope + int64_t(row) * p.slope_ld + column);
                s[0] = w.x, s[1] = w.y, s[2] = w.z, s[3] = w.w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = 2 * i < live ? v[2 * i] * (Sfu<kFp16>::lo(s[i]) * (1.0f / kSlopeScale)) : 0.0f;
                    v[2 * i + 1] = 2 * i + 1 < live ? v[2 * i + 1] * (Sfu<kFp16>::hi(s[i]) * (1.0f / kSlopeScale)) : 0.0f;
                }
            }
            if (p.dz) {
                uint4 w;
                w.x = Sfu<DT>::pack(v[0], v[1]), w.y = Sfu<DT>::pack(v[2], v[3]);
                w.z = Sfu<DT>::pack(v[4], v[5]), w.w = Sfu<DT>::pack(v[6], v[7]);
                *reinterpret_cast<uint4*>(p.dz + int64_t(row) * p.dz_ld + column) = w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[i];
        }
    }
    if (!p.partial) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[row_lane][8 * lane + i] = sum[i];
    __syncthreads();
    const int c = blockIdx.x * kActColumns + threadIdx.x;
    if (c < p.out) {
        float total = 0.0f;
#pragma unroll
        for (int r = 0; r < kActRowLanes; ++r) total += sums[r][threadIdx.x];
        p.partial[int64_t(blockIdx.y) * p.out + c] = total;
    }
}

// the chunks' sums, always in the same order
__global__ void __launch_bounds__(256) linear_bias_grad_kernel(const float* partial, void* out, int chunks, int n, int dtype) {
    __shared__ float part[8][33];
    wait_for_inputs();
    const int column = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
    float sum = 0.0f;
    if (column < n)
#pragma unroll 4
        for (int c = lane; c < chunks; c += 8) sum += partial[int64_t(c) * n + column];
    part[lane][threadIdx.x & 31] = sum;
    __syncthreads();
    if (lane == 0 && column < n) {
#pragma unroll
        for (int i = 1; i < 8; ++i) sum += part[i][threadIdx.x];
        if (dtype == FPT_FP32) static_cast<float*>(out)[column] = sum;
        else if (dtype == FPT_BF16) static_cast<__nv_bfloat16*>(out)[column] = __float2bfloat16_rn(sum);
        else static_cast<__half*>(out)[column] = __float2half_rn(sum);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------

// [rows, columns] of 16-bit values, rows of `ld`: boxes of 64 columns x box_rows
int operand_map(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, int64_t ld, int box_rows) {
    const uint64_t dims[4] = {uint64_t(columns), uint64_t(rows), 1, 1};
    const uint64_t plane = uint64_t(ld) * 2 * uint64_t(rows);
    const uint64_t strides[3] = {uint64_t(ld) * 2, plane, plane};
    return make_tensor_map_bf16_4d(map, base, dims, strides, uint32_t(box_rows));
}
// the same with the columns as columns / 64 slices: boxes of 64 columns x box_rows x box_slices.  Only for whole slices: a
// slice that reached past the row's end would read the next row's values, and past the last row's end other memory.
int sliced_map(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, int64_t ld, int box_rows, int box_slices) {
    const uint64_t dims[4] = {64, uint64_t(rows), uint64_t(columns / 64), 1};
    const uint64_t strides[3] = {uint64_t(ld) * 2, 128, uint64_t(ld) * 2 * uint64_t(rows)};
    return make_tensor_map_bf16_4d(map, base, dims, strides, uint32_t(box_rows), uint32_t(box_slices));
}
// one operand, `size` of its rows per CTA and tile
// (an MN-major operand in slices starts its tiles on slices)
int tile_map(CUtensorMap* map, bool* whole, const void* base, int64_t rows, int64_t k, int64_t ld, bool mn, int size, int chunks) {
    *whole = mn ? rows % 64 == 0 && size % 64 == 0 : k % 64 == 0;
    if (mn) return *whole ? sliced_map(map, base, k, rows, ld, chunks * kBlockK, size > 64 ? 2 : 1) : operand_map(map, base, k, rows, ld, chunks * kBlockK);
    return *whole ? sliced_map(map, base, rows, k, ld, size, chunks) : operand_map(map, base, rows, k, ld, size);
}

struct Product {
    const void *a, *b;                 // D[i, j] = sum_k A[i, k] B[j, k], i < m, j < n
    int64_t a_ld, b_ld, m, n, k;
    bool a_mn, b_mn;                   // operand stored [k, rows] instead of [rows, k]
};

// A launch that may begin while the kernel before it in the stream drains; `cluster` 0: the kernel's own attribute, or none.  The
// kernel's limit of shared memory belongs to all threads of the process: it is set to `smem_most`, which is the same in every
// call of a kernel, so that no thread lowers it between another's setting and launch.
template <class... P, class... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, size_t smem_most, unsigned cluster, cudaStream_t stream, const A&... args) {
    if (smem_most > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_most));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, P(args)...);
}

// Columns of an output tile.  A tile's time goes with its width and some 64 columns more (measured, 4096 x 4096 x 14336, us per
// tile at widths 96, 128 .. 256: 16.6, 17.2, 19.3, 21.7, 24.3, 27.6); the launch takes as many of them as the busiest pair has,
// but where power is the limit pairs that run dry early leave clock to the others, so that the mean counts half.
// Measured at 4096 x 4096 x 4096, us at widths 128, 160 .. 256: 123, 113, 101, 100, 96 (3.46 tiles a pair at the last).
int pair_columns(const Product& q, int pairs) {
    const int key = fpt::tuning_linear_columns();
    if (key > 0) return key;
    const int64_t row_tiles = (q.m + 255) / 256;
    int best = 256;
    int64_t least = INT64_MAX;
    for (int c = 256; c >= 64; c -= 32) {
        if (q.b_mn && c % 128) continue;            // whole slices of 64 columns for either CTA of the pair
        const int64_t tiles = row_tiles * ((q.n + c - 1) / c), rounds = (tiles + pairs - 1) / pairs;
        const int64_t time = (rounds * pairs + tiles) * (c + 64);
        if (time < least) {
            least = time;
            best = c;
        }
    }
    return best;
}

// Tile width and pairs per tile, and the time it should take in nanoseconds: 3600 + 9.5 per column to start, read out and end; per
// K block and round 1.25 per column (products), 165 + 0.36 per column (a pair's loads) or what all tiles at work draw at 14 TB/s;
// no less than both operands at 6 TB/s.  Tiles shared along K take 1200 + 8 per column more, and all their clusters have to be
// resident at once (32 of four CTAs, 14 of eight; 16 of eight take two rounds).
// Measured, us on one pair a tile, the best width, and on two or four: 256 rows of 4096 -> 4096 15.8 and 14.0, 512 rows of
// 4096 -> 4096 17.7 and 19.3, of 14336 -> 4096 53.5 and 49.1; dW of 512 x 512 over 16384 rows 43.8 and 17.9.
struct PairForm {
    int columns, split;
    int64_t time;
};
PairForm pair_form(const Product& q, int sm_count) {
    const int64_t stages = (q.k + kChunks * kBlockK - 1) / (kChunks * kBlockK), row_tiles = (q.m + 255) / 256;
    const auto tiles = [&](int columns) { return row_tiles * ((q.n + columns - 1) / columns); };
    const int64_t operands = (q.m + q.n) * q.k * 2 / 6000;
    const auto stream = [&](int columns, int split) {                 // the K blocks of the busiest pair
        const int64_t count = tiles(columns) * split, resident = std::min<int64_t>(count, sm_count / 2), rounds = (count + resident - 1) / resident;
        const int64_t block = std::max<int64_t>({125 * columns / 100, 165 + 36 * columns / 100, (16384 + 64 * columns) * 2 * resident / 14000});
        return std::max(operands, rounds * ((stages + split - 1) / split) * kChunks * block);
    };
    const int columns = pair_columns(q, sm_count / 2);
    const int key = fpt::tuning_linear_tokens() == 0 ? fpt::tuning_linear_split() : 0, width = fpt::tuning_linear_columns();
    PairForm best{columns, 1, 3600 + 95 * columns / 10 + stream(columns, 1)};
    for (int split = 2; split <= 4; split *= 2) {
        if (split > stages || (key > 0 && key != split)) continue;
        for (int c = 256; c >= 64; c /= 2) {
            if ((width > 0 && c != width) || c % (32 * split) || (q.b_mn && c % 128)) continue;
            if (key <= 0 && tiles(c) > (split == 2 ? 32 : 14) * sm_count / 148) continue;
            const int64_t time = 4800 + 175 * c / 10 + stream(c, split);
            if (key > 0 || time < best.time) best = PairForm{c, split, time};
            if (key > 0) return best;
        }
    }
    return best;
}

template <int DT, int ACT, bool SLOPE, bool A_MN, bool B_MN>
int launch_pair(const Product& q, LinearParams& p, const DeviceInfo& dev, PairForm form, cudaStream_t stream) {
    CUtensorMap map_a, map_b;
    p.columns = form.columns;
    p.split = form.split;
    p.chunks = kChunks;
    p.k_blocks = int((q.k + p.chunks * kBlockK - 1) / (p.chunks * kBlockK));
    if (int rc = tile_map(&map_a, &p.a_whole, q.a, q.m, q.k, q.a_ld, A_MN, 128, p.chunks)) return rc;
    if (int rc = tile_map(&map_b, &p.b_whole, q.b, q.n, q.k, q.b_ld, B_MN, p.columns / 2, p.chunks)) return rc;
    p.m_tiles = int((q.m + 255) / 256);
    p.n_tiles = int((q.n + p.columns - 1) / p.columns);
    p.stage_bytes = share_bytes<A_MN>(128, p.chunks) + share_bytes<B_MN>(p.columns / 2, p.chunks);
    p.ring = int(std::min<uint32_t>(kMaxRing, kRingBytes / p.stage_bytes));
    p.staged = p.vec_out && (!p.residual || p.vec_res) && (!p.slope || p.vec_slope);
    static_assert(sizeof(PairSmem) + 1024 <= 227 * 1024, "shared memory budget");
    static_assert(128 * 256 * 4 <= kRingBytes, "a CTA's sums fit its ring");
    const size_t smem = sizeof(PairSmem) + 1024;
    const int64_t tiles = int64_t(p.m_tiles) * p.n_tiles;
    const int64_t pairs = p.split > 1 ? tiles * p.split : std::min<int64_t>(tiles, dev.sm_count / 2);
    if (pairs > 0x3fffffff) return FPT_ERR_BAD_SIZE;
    if (p.split > 1)
        return cuda_status(launch_early(linear_shared_pair_kernel<DT, ACT, SLOPE, A_MN, B_MN>, unsigned(2 * pairs), kPairThreads, smem, smem, unsigned(2 * p.split), stream, map_a, map_b, p));
    return cuda_status(launch_early(linear_pair_kernel<DT, ACT, SLOPE, A_MN, B_MN>, unsigned(2 * pairs), kPairThreads, smem, smem, 0u, stream, map_a, map_b, p));
}

// Whether a block of the few-row form takes all of an SM's shared memory: where every block can have an SM to itself (clusters do
// not pack into every last one: 16 clusters of 8 or 48 of 3 took two rounds); else it takes half.
bool alone_on_sm(int64_t blocks, int split, int sm_count) {
    return split == 1 ? blocks <= sm_count : split <= 4 && blocks <= sm_count * 7 / 8;
}

// B, the tokens' operand, becomes the column side: D is written row by row as [tokens, outputs] all the same
template <int DT, int ACT, bool SLOPE, int TOKENS, bool W_MN>
int launch_split(const Product& q, LinearParams& p, const DeviceInfo& dev, int split, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (int rc = tile_map(&map_w, &p.b_whole, q.b, q.n, q.k, q.b_ld, W_MN, 128, 1)) return rc;
    if (int rc = operand_map(&map_x, q.a, q.m, q.k, q.a_ld, TOKENS)) return rc;
    p.m_tiles = int((q.m + TOKENS - 1) / TOKENS);
    p.n_tiles = int((q.n + 127) / 128);
    p.split = split;
    const int64_t blocks = int64_t(p.m_tiles) * p.n_tiles * split;
    if (blocks > 0x7fffffff) return FPT_ERR_BAD_SIZE;
    const uint32_t stage = kTileBytes + TOKENS * 128;
    constexpr uint32_t kRingMost = 216 * 1024, kRingHalf = 108 * 1024;     // of a block alone on its SM, of one of two
    constexpr size_t kSmemMost = 1024 + kSplitRingOffset + kRingMost;
    static_assert(TOKENS * 512 <= kRingHalf && kSmemMost <= 227 * 1024, "shared memory budget");
    const uint32_t budget = alone_on_sm(blocks, split, dev.sm_count) ? kRingMost : kRingHalf;
    p.ring = int(std::min<uint32_t>(kMaxRing, budget / stage));
    const size_t smem = 1024 + kSplitRingOffset + std::max<size_t>(size_t(p.ring) * stage, size_t(TOKENS) * 512);
    return cuda_status(launch_early(linear_split_kernel<DT, ACT, SLOPE, TOKENS, W_MN>, unsigned(blocks), kSplitThreads, smem, kSmemMost,
                                      split > 1 ? unsigned(split) : 0u, stream, map_w, map_x, p));
}

// Which form, by the time it should take, in nanoseconds.  The terms were fitted to a sweep of both forms over six layers (512 x
// 512 to 14336 x 4096, 1 to 1024 rows); the picks lie within some 5 % of the best measured, in a few places 20 % (256 rows of
// 8192 -> 1024 16.5 us, on shared tiles 13.6).
//   few rows   3000 to start and end, 20 per token of a tile (read-out), 300 + 40 a block for a cluster; the stream takes the
//              longest of 210 per K block and block on an SM (alone: and a third per token), of 1800 per turn of the ring where
//              a block has half the memory, of the weight at 6 TB/s and of the tiles at 14 TB/s
//   pairs      as pair_form
// Clusters of five and seven are left out: seven blocks do not pack into a processing cluster of the chip (twice the time).
struct Form {
    int tokens, split;                 // tokens 0: pairs
};
Form choose_form(const Product& q, const PairForm& pairs, int k_blocks, int sm_count) {
    const int64_t kb = k_blocks;
    int64_t least = pairs.time;
    Form best{0, 1};
    const int key = fpt::tuning_linear_tokens(), split_key = fpt::tuning_linear_split();
    if (key > 0) least = INT64_MAX;
    if (q.a_mn || key == 0) return best;
    for (int tokens = 16; tokens <= 128; tokens *= 2) {
        if (key > 0 && tokens != key) continue;
        if (key < 0 && q.m > 8 * tokens) continue;
        const int64_t tiles = (q.m + tokens - 1) / tokens * ((q.n + 127) / 128);
        for (int split = 1; split <= kMaxSplit && (split == 1 || split <= kb / 2); ++split) {
            if (split_key > 0 && split != std::max<int64_t>(1, std::min<int64_t>(split_key, kb / 2))) continue;
            const int64_t blocks = tiles * split, per_sm = (blocks + sm_count - 1) / sm_count;
            if (split_key <= 0 && (split == 5 || split == 7)) continue;
            // one round of blocks, with room for the larger clusters to find their place
            if (split > 1 && blocks > (split > 2 ? 256 * sm_count / 148 : 2 * sm_count) && split_key <= 0) break;
            const int64_t turn = 1800 / std::min<int64_t>(kMaxRing, 108 * 1024 / (kTileBytes + tokens * 128));
            const int64_t block = alone_on_sm(blocks, split, sm_count) ? 210 + tokens / 3 : std::max(210 * per_sm, turn);
            const int64_t issue = block * ((kb + split - 1) / split);
            const int64_t weight = q.n * q.k * 2 / 6000, traffic = tiles * kb * (16384 + 128 * tokens) / 14000;
            const int64_t time = 3000 + 20 * tokens + (split > 1 ? 300 + 40 * split : 0) + std::max(issue, std::max(weight, traffic));
            if (time < least) {
                least = time;
                best = Form{tokens, split};
            }
        }
    }
    return best;
}

template <int DT, int ACT, bool SLOPE, bool A_MN, bool B_MN>
int launch_product(const Product& q, LinearParams& p, const DeviceInfo& dev, cudaStream_t stream) {
    p.m = int(q.m);
    p.n = int(q.n);
    p.k_blocks = int((q.k + kBlockK - 1) / kBlockK);
    const PairForm pairs = pair_form(q, dev.sm_count);
    if constexpr (!A_MN) {
        const Form form = choose_form(q, pairs, p.k_blocks, dev.sm_count);
        switch (form.tokens) {
        case 16: return launch_split<DT, ACT, SLOPE, 16, B_MN>(q, p, dev, form.split, stream);
        case 32: return launch_split<DT, ACT, SLOPE, 32, B_MN>(q, p, dev, form.split, stream);
        case 64: return launch_split<DT, ACT, SLOPE, 64, B_MN>(q, p, dev, form.split, stream);
        case 128: return launch_split<DT, ACT, SLOPE, 128, B_MN>(q, p, dev, form.split, stream);
        default: break;
        }
    }
    return launch_pair<DT, ACT, SLOPE, A_MN, B_MN>(q, p, dev, pairs, stream);
}

bool aligned16(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

int check_sizes(int64_t rows, int64_t dim, int64_t out, int dtype) {
    if (rows < 0 || dim <= 0 || out <= 0) return FPT_ERR_BAD_SIZE;
    if (rows > 0x7fffffff - 256 || dim > 0x7fffffff - 256 || out > 0x7fffffff - 256) return FPT_ERR_BAD_SIZE;
    if ((rows + 255) / 256 * ((out + 255) / 256) > 0x3fffffff || (out + 255) / 256 * ((dim + 255) / 256) > 0x3fffffff ||
        (rows + 255) / 256 * ((dim + 255) / 256) > 0x3fffffff)
        return FPT_ERR_BAD_SIZE;
    if (dim % 8) return FPT_ERR_UNSUPPORTED_SHAPE;
    if (dtype != FPT_FP16 && dtype != FPT_BF16) return FPT_ERR_BAD_ENUM;
    return FPT_OK;
}

template <int ACT, bool SLOPE, bool A_MN, bool B_MN>
int run_product(const Product& q, LinearParams& p, int dtype, cudaStream_t stream) {
    DeviceInfo dev;
    if (int rc = current_device_info(&dev)) return rc;
    return dtype == FPT_BF16 ? launch_product<kBf16, ACT, SLOPE, A_MN, B_MN>(q, p, dev, stream)
                             : launch_product<kFp16, ACT, SLOPE, A_MN, B_MN>(q, p, dev, stream);
}
template <int ACT>
int run_forward(const Product& q, LinearParams& p, int dtype, cudaStream_t stream) {
    if constexpr (ACT != kNone)
        if (p.slope) return run_product<ACT, true, false, false>(q, p, dtype, stream);
    return run_product<ACT, false, false, false>(q, p, dtype, stream);
}

}  // namespace
}  // namespace fpt

using namespace fpt;

extern "C" int fpt_linear(void* out, void* slope, const void* x, const void* weight, const void* bias, const void* residual,
                          int64_t rows, int64_t dim, int64_t out_features, int64_t x_ld, int64_t w_ld, int64_t out_ld,
                          int64_t residual_ld, int64_t slope_ld, int dtype, int bias_dtype, int function, int degree, int source,
                          void* status, fpt_stream_t stream) {
    if (int rc = check_sizes(rows, dim, out_features, dtype)) return rc;
    if (bias && (bias_dtype < FPT_FP16 || bias_dtype > FPT_FP32)) return FPT_ERR_BAD_ENUM;
    if (function != FPT_FN_NONE && function != FPT_FN_SIGMOID && function != FPT_FN_TANH && function != FPT_FN_SWISH && function != FPT_FN_GELU)
        return FPT_ERR_BAD_ENUM;
    if (source != FPT_SRC_CURRENT && source != FPT_SRC_SOLLYA) return FPT_ERR_BAD_ENUM;
    LinearParams p{};
    if (function == FPT_FN_NONE && (degree != 0 || slope)) return FPT_ERR_UNKNOWN_PROGRAM;
    if (degree != 0) {
        const ProgramRow* fwd = find_program(function, FPT_FWD, degree, dtype, source);
        const ProgramRow* bwd = find_program(function, FPT_BWD, degree, dtype, source);
        if (!fwd || (slope && !bwd)) return FPT_ERR_UNKNOWN_PROGRAM;
        if (fwd->shape > kEven || (bwd && bwd->shape > kEven)) return FPT_ERR_UNSUPPORTED_SHAPE;
        p.act.fwd = program_words(*fwd);
        p.act.fwd_shape = fwd->shape;
        p.act.fwd_degree = fwd->degree;
        if (bwd) {
            p.act.bwd = program_words(*bwd);
            p.act.bwd_shape = bwd->shape;
            p.act.bwd_degree = bwd->degree;
        }
    }
    if (rows == 0) return FPT_OK;
    if (!out || !x || !weight) return FPT_ERR_NULL_POINTER;
    if (x_ld < dim || w_ld < dim || out_ld < out_features || (residual && residual_ld < out_features) || (slope && slope_ld < out_features))
        return FPT_ERR_BAD_SIZE;
    if (!aligned16(x, x_ld) || !aligned16(weight, w_ld)) return FPT_ERR_MISALIGNED;
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(slope)) & 1u) return FPT_ERR_MISALIGNED;
    if (bias && reinterpret_cast<uintptr_t>(bias) % (bias_dtype == FPT_FP32 ? 4u : 2u)) return FPT_ERR_MISALIGNED;
    p.out = out;
    p.out_ld = out_ld;
    p.residual = residual;
    p.res_ld = residual_ld;
    p.slope = static_cast<uint16_t*>(slope);
    p.slope_ld = slope_ld;
    p.bias = bias;
    p.bias_dtype = bias_dtype;
    p.vec_out = aligned16(out, out_ld);
    p.vec_res = aligned16(residual, residual_ld);
    p.vec_slope = aligned16(slope, slope_ld);
    p.vec_bias = reinterpret_cast<uintptr_t>(bias) % 16 == 0;
    p.status = static_cast<uint32_t*>(status);
    const Product q{x, weight, x_ld, w_ld, rows, out_features, dim, false, false};
    if (degree != 0) return run_forward<kProgram>(q, p, dtype, stream);
    switch (function) {
    case FPT_FN_SIGMOID: return run_forward<kSigmoid>(q, p, dtype, stream);
    case FPT_FN_TANH: return run_forward<kTanh>(q, p, dtype, stream);
    case FPT_FN_SWISH: return run_forward<kSwishAct>(q, p, dtype, stream);
    case FPT_FN_GELU: return run_forward<kGelu>(q, p, dtype, stream);
    default: return run_forward<kNone>(q, p, dtype, stream);
    }
}

extern "C" int fpt_linear_grad_input(void* dx, const void* dz, const void* weight, int64_t rows, int64_t dim, int64_t out_features,
                                     int64_t dx_ld, int64_t dz_ld, int64_t w_ld, int dtype, void* status, fpt_stream_t stream) {
    if (int rc = check_sizes(rows, dim, out_features, dtype)) return rc;
    if (rows == 0) return FPT_OK;
    if (!dx || !dz || !weight) return FPT_ERR_NULL_POINTER;
    if (dx_ld < dim || dz_ld < out_features || w_ld < dim) return FPT_ERR_BAD_SIZE;
    if (!aligned16(dz, dz_ld) || !aligned16(weight, w_ld) || (reinterpret_cast<uintptr_t>(dx) & 1u)) return FPT_ERR_MISALIGNED;
    LinearParams p{};
    p.out = dx;
    p.out_ld = dx_ld;
    p.vec_out = aligned16(dx, dx_ld);
    p.status = static_cast<uint32_t*>(status);
    const Product q{dz, weight, dz_ld, w_ld, rows, dim, out_features, false, true};
    return run_product<kNone, false, false, true>(q, p, dtype, stream);
}

extern "C" int fpt_linear_grad_weight(void* dw, const void* dz, const void* x, int64_t rows, int64_t dim, int64_t out_features,
                                      int64_t dw_ld, int64_t dz_ld, int64_t x_ld, int dtype, void* status, fpt_stream_t stream) {
    if (int rc = check_sizes(rows, dim, out_features, dtype)) return rc;
    if (!dw) return FPT_ERR_NULL_POINTER;
    if (dw_ld < dim) return FPT_ERR_BAD_SIZE;
    if (reinterpret_cast<uintptr_t>(dw) & 1u) return FPT_ERR_MISALIGNED;
    if (rows == 0) {                    // the sum over no rows
        DeviceInfo dev;
        if (int rc = current_device_info(&dev)) return rc;
        return cuda_status(cudaMemset2DAsync(dw, size_t(dw_ld) * 2, 0, size_t(dim) * 2, size_t(out_features), stream));
    }
    if (!dz || !x) return FPT_ERR_NULL_POINTER;
    if (dz_ld < out_features || x_ld < dim) return FPT_ERR_BAD_SIZE;
    if (!aligned16(dz, dz_ld) || !aligned16(x, x_ld)) return FPT_ERR_MISALIGNED;
    LinearParams p{};
    p.out = dw;
    p.out_ld = dw_ld;
    p.vec_out = aligned16(dw, dw_ld);
    p.status = static_cast<uint32_t*>(status);
    const Product q{dz, x, dz_ld, x_ld, out_features, dim, rows, true, true};
    return run_product<kNone, false, true, true>(q, p, dtype, stream);
}

namespace {
// rows one block sums, at least 32: as many blocks as 148 SMs hold at once (a constant: the size of the workspace does not ask for a
// device).  Measured with the column sums, 4096 x 4096 and 2048 x 14336 bf16, us at 3, 4, 5 and 6 blocks an SM: 23.3, 20.8, 20.5, 25.0
// and 39.4, 34.2, 31.8, 39.4 (the sixth is a second round).
int grad_act_chunk(int64_t rows, int64_t out) {
    const int64_t column_blocks = (out + kActColumns - 1) / kActColumns;
    const int64_t chunks = std::max<int64_t>(1, 148 * kActBlocks / column_blocks);
    return int(std::min<int64_t>(rows, std::max<int64_t>((rows + chunks - 1) / chunks, std::max<int64_t>(32, (rows + 65534) / 65535))));
}
}  // namespace

extern "C" int64_t fpt_linear_grad_act_workspace_bytes(int64_t rows, int64_t out_features) {
    if (rows <= 0 || out_features <= 0) return 0;
    const int64_t chunk = grad_act_chunk(rows, out_features);
    return (rows + chunk - 1) / chunk * out_features * int64_t(sizeof(float));
}

extern "C" int fpt_linear_grad_act(void* dz, void* dbias, const void* dy, const void* slope, void* workspace, int64_t workspace_bytes,
                                   int64_t rows, int64_t out_features, int64_t dz_ld, int64_t dy_ld, int64_t slope_ld, int dtype,
                                   int bias_dtype, fpt_stream_t stream) {
    if (int rc = check_sizes(rows, 8, out_features, dtype)) return rc;
    if (dbias && (bias_dtype < FPT_FP16 || bias_dtype > FPT_FP32)) return FPT_ERR_BAD_ENUM;
    if (dbias && reinterpret_cast<uintptr_t>(dbias) % (bias_dtype == FPT_FP32 ? 4u : 2u)) return FPT_ERR_MISALIGNED;
    const int64_t padded = (out_features + 7) / 8 * 8;
    if (rows > 0) {
        if (!dy) return FPT_ERR_NULL_POINTER;
        if (dy_ld < out_features || (dz && dz_ld < padded) || (slope && slope_ld < padded)) return FPT_ERR_BAD_SIZE;
        if (reinterpret_cast<uintptr_t>(dy) & 1u) return FPT_ERR_MISALIGNED;
        if ((dz && !aligned16(dz, dz_ld)) || (slope && !aligned16(slope, slope_ld))) return FPT_ERR_MISALIGNED;
        if (dbias && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 4)) return workspace ? FPT_ERR_MISALIGNED : FPT_ERR_NULL_POINTER;
        if (dbias && workspace_bytes < fpt_linear_grad_act_workspace_bytes(rows, out_features)) return FPT_ERR_SCRATCH_TOO_SMALL;
    }
    DeviceInfo dev;
    if (int rc = current_device_info(&dev)) return rc;
    int chunks = 0;
    if (rows > 0 && (dz || dbias)) {
        GradActParams p{};
        p.dy = static_cast<const uint16_t*>(dy);
        p.slope = static_cast<const uint16_t*>(slope);
        p.dz = static_cast<uint16_t*>(dz);
        p.partial = dbias ? static_cast<float*>(workspace) : nullptr;
        p.dy_ld = dy_ld;
        p.slope_ld = slope_ld;
        p.dz_ld = dz_ld;
        p.rows = int(rows);
        p.out = int(out_features);
        p.chunk_rows = grad_act_chunk(rows, out_features);
        p.vec_dy = aligned16(dy, dy_ld);
        chunks = int((rows + p.chunk_rows - 1) / p.chunk_rows);
        const dim3 grid(unsigned((out_features + kActColumns - 1) / kActColumns), unsigned(chunks));
        if (int rc = cuda_status(launch_early(dtype == FPT_BF16 ? linear_grad_act_kernel<kBf16> : linear_grad_act_kernel<kFp16>, grid, kActThreads, 0, 0, 0u, stream, p))) return rc;
    }
    if (dbias) {
        return cuda_status(launch_early(linear_bias_grad_kernel, unsigned((out_features + 31) / 32), 256u, 0, 0, 0u, stream,
                                        static_cast<const float*>(workspace), dbias, chunks, int(out_features), bias_dtype));
    }
    return FPT_OK;
}
