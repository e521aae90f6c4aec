// A linear layer with everything that follows it in the epilogue, for sm_100a: y = act(x W^T + b) + r, and the products and
// the element-wise pass of its gradient.
//
//   forward          y [rows, out]  = act(x [rows, dim] W[out, dim]^T + b) + r,   optionally act'(x W^T + b) in fp16
//   dz = dy act'     element-wise, with the column sums that are the gradient of b
//   dx [rows, dim] = dz W           the contraction runs over W's rows: W is an MN-major operand
//   dW [out, dim]  = dz^T x         both operands MN-major
//
// All products are D[i, j] = sum_k A[i, k] B[j, k] on tcgen05 with fp32 accumulators in tensor memory, operands brought by
// TMA into 128-byte-swizzled tiles: K-major tiles of [rows x 64 k], or MN-major ones of two panels [64 k x 64 rows], so
// that no operand is ever transposed in memory.  Two forms:
//
//   linear_pair_kernel    many rows.  Persistent pairs of CTAs (cta_group::2), 256 x 256 output tiles, two accumulators in
//                         turn so that the epilogue of one tile runs under the products of the next; bound by the tensor
//                         pipe (and, in long runs, by the power cap).
//   linear_split_kernel   few rows.  The weight is the 128-row operand and the tokens are the columns (16 .. 128 of them): a
//                         block streams a [128 x K / split] slab of the weight through a ring of TMA tiles, two blocks per
//                         SM; the blocks of a cluster share an output tile along K and add their fp32 partial sums over
//                         distributed shared memory, in rank order (no atomics, no workspace, one launch).  Bound by the
//                         weight's bytes.
//
// Rounding: the epilogue works on the fp32 accumulators and rounds once.  The slope act' is kept in fp16 also beside bf16
// data: it lies in about [-0.13, 1.13], where fp16 has eight times the resolution of bf16 at the same size, so the backward
// pass adds no error of bf16's size by it (z itself in bf16 would).  dz is rounded to the data type before the two
// products, which take 16-bit operands; its column sums are taken before that rounding.
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
constexpr int kBandTiles = 16;                      // 256-row tiles per band: 4096 rows, see fpt_gate_up_swiglu.cu

enum : uint32_t { kWaitEmpty = 0x51, kWaitFull, kWaitAccEmpty, kWaitAccFull };
enum ActKind : int { kActNone, kActNative, kActProgram };

struct Activation {
    int kind, fn;
    int fwd_shape, fwd_degree, bwd_shape, bwd_degree;
    ProgramWords fwd, bwd;
};

struct LinearParams {
    void* out;                      // [m, n] rows of out_ld
    const void* residual;           // [m, n] or null
    const void* bias;               // [n] or null
    uint16_t* slope;                // [m, n] fp16 or null
    int64_t out_ld, res_ld, slope_ld;
    int m, n, k_blocks;
    int m_tiles, n_tiles;
    int split;                      // blocks per cluster (split form)
    int bias_dtype;
    bool vec_out, vec_res, vec_slope, vec_bias;
    Activation act;
    uint32_t* status;
};

// ---- waits --------------------------------------------------------------------------------------------------------

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

__device__ __forceinline__ float logistic(float z) { return mufu_rcp(1.0f + mufu_ex2(-1.4426950408889634f * z)); }

// z -> act(z), d -> act'(z) where wanted
template <int DT, int N>
__device__ __forceinline__ void activate(const Activation& a, float (&z)[N], float (&d)[N], bool want) {
    if (a.kind == kActNone) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = 1.0f;
    } else if (a.kind == kActProgram) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint32_t x = Sfu<DT>::pack(z[i], z[i + 1]);
            const uint32_t y = run_program<DT>(x, a.fwd, a.fwd_shape, a.fwd_degree);
            z[i] = Sfu<DT>::lo(y);
            z[i + 1] = Sfu<DT>::hi(y);
            if (want) {
                const uint32_t s = run_program<DT>(x, a.bwd, a.bwd_shape, a.bwd_degree);
                d[i] = Sfu<DT>::lo(s);
                d[i + 1] = Sfu<DT>::hi(s);
            }
        }
    } else if (a.fn == FPT_FN_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = z[i], phi = 0.5f * (1.0f + erff(x * 0.70710678118654752440f));
            z[i] = x * phi;
            if (want) d[i] = fmaf(x * 0.3989422804014327f, mufu_ex2(-0.72134752044448170368f * x * x), phi);
        }
    } else if (a.fn == FPT_FN_SWISH) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = z[i], p = logistic(x);
            z[i] = x * p;
            if (want) d[i] = p * fmaf(x, 1.0f - p, 1.0f);
        }
    } else if (a.fn == FPT_FN_SIGMOID) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float p = logistic(z[i]);
            z[i] = p;
            if (want) d[i] = p * (1.0f - p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float y = tanhf(z[i]);
            z[i] = y;
            if (want) d[i] = fmaf(-y, y, 1.0f);
        }
    }
}

// N consecutive columns of one row: bias, activation, residual, stores.  N is a multiple of 4; column a multiple of N.
template <int DT, int N>
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
    activate<DT, N>(p.act, z, d, p.slope != nullptr);
    if (p.slope) {
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

// ---- many rows: pairs of CTAs ---------------------------------------------------------------------------------------

constexpr int kPairRing = 6;
constexpr int kPairThreads = 384;       // TMA, product and allocation warps, one idle, eight epilogue warps

struct PairSmem {
    alignas(1024) uint8_t a[kPairRing][kTileBytes];
    alignas(1024) uint8_t b[kPairRing][kTileBytes];
    alignas(8) uint64_t full[kPairRing];
    uint64_t empty[kPairRing];
    uint64_t acc_full[2], acc_empty[2];
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
    return PairTile{(band * kBandTiles + r - column * in_band) * 256, column * 256};
}

template <bool MN>
__device__ __forceinline__ void load_pair(uint8_t* tile, const CUtensorMap* map, uint32_t bar, int kb, int row) {
    if constexpr (MN) {
        tma_load_4d_pair(tile, map, bar, row, kb * kBlockK, 0, 0);
        tma_load_4d_pair(tile + kPanelBytes, map, bar, row + 64, kb * kBlockK, 0, 0);
    } else {
        tma_load_4d_pair(tile, map, bar, kb * kBlockK, row, 0, 0);
    }
}

// Each CTA of the pair holds 128 rows of A and of B and receives 128 rows x 256 columns of D; the hand-overs are those of
// gate_up_swiglu_pair_kernel.
template <int DT, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ LinearParams p) {
    extern __shared__ uint8_t smem_raw[];
    PairSmem& sm = *reinterpret_cast<PairSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    volatile uint32_t* abort_flag = &sm.abort_flag;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairRing; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&sm.acc_full[a], 1);
            mbar_init(&sm.acc_empty[a], 16);            // eight epilogue warps in each CTA
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
    const int tiles = p.m_tiles * p.n_tiles;
    const int first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
                const PairTile t = pair_tile(p, tile);
                for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
                    const uint32_t s = it % kPairRing, use = it / kPairRing;
                    if (use > 0) ok = wait(&sm.empty[s], (use - 1u) & 1u, abort_flag, p.status, kWaitEmpty);
                    if (!ok) break;
                    const uint32_t bar = map_to_cta(smem_u32(&sm.full[s]), 0);
                    if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], 4 * kTileBytes);
                    load_pair<A_MN>(sm.a[s], &map_a, bar, kb, t.row0 + int(rank) * 128);
                    load_pair<B_MN>(sm.b[s], &map_b, bar, kb, t.column0 + int(rank) * 128);
                }
            }
        }
    } else if (warp == 1 && rank == 0) {
        const bool elected = elect_one();
        constexpr uint32_t idesc = instruction<DT>(256, 256, A_MN, B_MN);
        constexpr uint32_t desc_hi = umma_smem_desc_hi(1024);
        uint32_t it = 0, local = 0;
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
            for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
                const uint32_t s = it % kPairRing;
                ok = wait(&sm.full[s], (it / kPairRing) & 1u, abort_flag, p.status, kWaitFull);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t a_lo = tile_lo<A_MN>(sm.a[s]), b_lo = tile_lo<B_MN>(sm.b[s]);
#pragma unroll
                for (uint32_t k = 0; k < kBlockK / 16; ++k)
                    if (elected) umma_ss_words_pair(tmem + a * 256u, a_lo + k * kStep16<A_MN>, b_lo + k * kStep16<B_MN>, desc_hi, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                if (elected) umma_commit_pair(&sm.empty[s], 3);
            }
            if (ok && elected) umma_commit_pair(&sm.acc_full[a], 3);
        }
    } else if (warp >= 4) {
        // four warps hold the 128 rows (a warp reads the 32 lanes of its number modulo 4); two such sets take 128 columns each
        const uint32_t lane_base = uint32_t(32 * (warp & 3)) << 16;
        const int half = (warp - 4) >> 2;
        uint32_t local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step, ++local) {
            const PairTile t = pair_tile(p, tile);
            const uint32_t a = local & 1u;
            ok = wait(&sm.acc_full[a], (local >> 1) & 1u, abort_flag, p.status, kWaitAccFull);
            if (!ok) break;
            tc_fence_after_sync();
            const int row = t.row0 + int(rank) * 128 + 32 * (warp & 3) + lane;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                const int column = t.column0 + half * 128 + c * 32;
                if (column >= p.n) break;
                uint32_t acc[32];
                tmem_ld_32x32b_x32(tmem + lane_base + a * 256u + uint32_t(half * 128 + c * 32), acc);
                tmem_ld_wait();
                if (row < p.m) {
                    float z[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) z[i] = __uint_as_float(acc[i]);
                    finish<DT, 32>(p, z, row, column);
                }
                __syncwarp();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(&sm.acc_empty[a]);
                else mbar_arrive_cluster(map_to_cta(smem_u32(&sm.acc_empty[a]), 0));
            }
        }
    }
    // neither CTA may leave while the other can still reach its barriers or tensor memory
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync_all();
    if (warp == 2) tmem_dealloc_pair(tmem, 512);
}

// ---- few rows: the weight streams, the tokens are columns ---------------------------------------------------------------

constexpr int kSplitThreads = 256;
constexpr int kMaxSplit = 8;

template <int TOKENS>
struct SplitSmem {
    static constexpr uint32_t kXBytes = TOKENS * 128;
    static constexpr int kRing = 108 * 1024 / int(kTileBytes + kXBytes);       // two blocks an SM
    struct Ring {
        alignas(1024) uint8_t w[kRing][kTileBytes];
        alignas(1024) uint8_t x[kRing][kXBytes];
    };
    union {
        Ring ring;
        float partial[TOKENS][128];               // after the last product: this block's sums, [token][output]
    };
    alignas(8) uint64_t full[kRing];
    uint64_t empty[kRing];
    uint64_t acc_full;
    uint32_t tmem_base;
    uint32_t abort_flag;
};

__device__ __forceinline__ float4 load_cluster(uint32_t address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}

// D is [tokens, outputs] (p.m tokens, p.n outputs); A = the weight, B = the tokens.  The p.split blocks of a cluster take
// equal runs of K blocks.
template <int DT, int TOKENS, bool W_MN>
__global__ void __launch_bounds__(kSplitThreads, 2)
linear_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearParams p) {
    using Smem = SplitSmem<TOKENS>;
    constexpr int kRing = Smem::kRing;
    constexpr uint32_t kColumns = TOKENS < 32 ? 32 : TOKENS;
    extern __shared__ uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? int(cluster_cta_rank()) : 0;
    volatile uint32_t* abort_flag = &sm.abort_flag;
    const int tile = blockIdx.x / p.split;
    const int output0 = tile / p.m_tiles * 128, token0 = tile % p.m_tiles * TOKENS;
    const int kb0 = int(int64_t(p.k_blocks) * rank / p.split), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / p.split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kRing; ++s) {
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

    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < kb1 - kb0; ++i) {
                const int s = i % kRing, kb = kb0 + i;
                if (i >= kRing && !wait(&sm.empty[s], uint32_t(i / kRing - 1) & 1u, abort_flag, p.status, kWaitEmpty)) break;
                mbar_arrive_expect_tx(&sm.full[s], kTileBytes + Smem::kXBytes);
                if constexpr (W_MN) {
                    tma_load_4d(sm.ring.w[s], &map_w, &sm.full[s], output0, kb * kBlockK, 0, 0);
                    tma_load_4d(sm.ring.w[s] + kPanelBytes, &map_w, &sm.full[s], output0 + 64, kb * kBlockK, 0, 0);
                } else {
                    tma_load_4d(sm.ring.w[s], &map_w, &sm.full[s], kb * kBlockK, output0, 0, 0);
                }
                tma_load_4d(sm.ring.x[s], &map_x, &sm.full[s], kb * kBlockK, token0, 0, 0);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool elected = elect_one();
        constexpr uint32_t idesc = instruction<DT>(128, TOKENS, W_MN, false);
        constexpr uint32_t desc_hi = umma_smem_desc_hi(1024);
        bool ok = true;
        for (int i = 0; i < kb1 - kb0; ++i) {
            const int s = i % kRing;
            ok = wait(&sm.full[s], uint32_t(i / kRing) & 1u, abort_flag, p.status, kWaitFull);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t w_lo = tile_lo<W_MN>(sm.ring.w[s]), x_lo = tile_lo<false>(sm.ring.x[s]);
#pragma unroll
            for (uint32_t k = 0; k < kBlockK / 16; ++k)
                if (elected) umma_ss_words(tmem, w_lo + k * kStep16<W_MN>, x_lo + k * kStep16<false>, desc_hi, idesc, (i > 0 || k > 0) ? 1u : 0u);
            if (elected) umma_commit(&sm.empty[s]);
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
            for (int i = 0; i < 16; ++i) sm.partial[c + i][32 * (warp & 3) + lane] = __uint_as_float(acc[i]);
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
        for (int t = rank * (kSplitThreads / 32) + warp; t < TOKENS && token0 + t < p.m; t += warps) {
            float z[4];
            if (p.split > 1) {
                const uint32_t mine = smem_u32(&sm.partial[t][4 * lane]);
                float4 part[kMaxSplit];
#pragma unroll
                for (int r = 0; r < kMaxSplit; ++r)
                    if (r < p.split) part[r] = load_cluster(map_to_cta(mine, uint32_t(r)));
                z[0] = part[0].x, z[1] = part[0].y, z[2] = part[0].z, z[3] = part[0].w;
#pragma unroll
                for (int r = 1; r < kMaxSplit; ++r)
                    if (r < p.split) z[0] += part[r].x, z[1] += part[r].y, z[2] += part[r].z, z[3] += part[r].w;
            } else {
                const float4 v = *reinterpret_cast<const float4*>(&sm.partial[t][4 * lane]);
                z[0] = v.x, z[1] = v.y, z[2] = v.z, z[3] = v.w;
            }
            if (output < p.n) finish<DT, 4>(p, z, token0 + t, output);
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

struct GradActParams {
    const uint16_t* dy;
    const uint16_t* slope;              // fp16, or null for 1
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
    const int row_end = min(p.rows, (int(blockIdx.y) + 1) * p.chunk_rows);
    const int live = min(8, p.out - column);                    // columns of this lane that exist
    float sum[8] = {};
    if (live > 0) {
#pragma unroll 2
        for (int row = int(blockIdx.y) * p.chunk_rows + row_lane; row < row_end; row += kActRowLanes) {
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
                    v[2 * i] = 2 * i < live ? v[2 * i] * Sfu<kFp16>::lo(s[i]) : 0.0f;
                    v[2 * i + 1] = 2 * i + 1 < live ? v[2 * i + 1] * Sfu<kFp16>::hi(s[i]) : 0.0f;
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
__global__ void __launch_bounds__(256) linear_bias_grad_kernel(const float* __restrict__ partial, void* out, int chunks, int n, int dtype) {
    __shared__ float part[8][33];
    const int column = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
    float sum = 0.0f;
    if (column < n)
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

struct Product {
    const void *a, *b;                 // D[i, j] = sum_k A[i, k] B[j, k], i < m, j < n
    int64_t a_ld, b_ld, m, n, k;
    bool a_mn, b_mn;                   // operand stored [k, rows] instead of [rows, k]
};

template <class K>
cudaError_t launch_cluster(K kernel, unsigned grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream,
                           const CUtensorMap& a, const CUtensorMap& b, const LinearParams& p) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = cluster ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, a, b, p);
}

template <int DT, bool A_MN, bool B_MN>
int launch_pair(const Product& q, LinearParams& p, const DeviceInfo& dev, cudaStream_t stream) {
    CUtensorMap map_a, map_b;
    if (int rc = A_MN ? operand_map(&map_a, q.a, q.k, q.m, q.a_ld, kBlockK) : operand_map(&map_a, q.a, q.m, q.k, q.a_ld, 128)) return rc;
    if (int rc = B_MN ? operand_map(&map_b, q.b, q.k, q.n, q.b_ld, kBlockK) : operand_map(&map_b, q.b, q.n, q.k, q.b_ld, 128)) return rc;
    p.m_tiles = int((q.m + 255) / 256);
    p.n_tiles = int((q.n + 255) / 256);
    static_assert(sizeof(PairSmem) + 1024 <= 227 * 1024, "shared memory budget");
    const size_t smem = sizeof(PairSmem) + 1024;
    const int64_t pairs = std::min<int64_t>(int64_t(p.m_tiles) * p.n_tiles, dev.sm_count / 2);
    auto kernel = linear_pair_kernel<DT, A_MN, B_MN>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return int(e);
    kernel<<<unsigned(2 * pairs), kPairThreads, smem, stream>>>(map_a, map_b, p);
    return cuda_status(cudaGetLastError());
}

// B, the tokens' operand, becomes the column side: D is written row by row as [tokens, outputs] all the same
template <int DT, int TOKENS, bool W_MN>
int launch_split(const Product& q, LinearParams& p, const DeviceInfo& dev, int split, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (int rc = W_MN ? operand_map(&map_w, q.b, q.k, q.n, q.b_ld, kBlockK) : operand_map(&map_w, q.b, q.n, q.k, q.b_ld, 128)) return rc;
    if (int rc = operand_map(&map_x, q.a, q.m, q.k, q.a_ld, TOKENS)) return rc;
    using Smem = SplitSmem<TOKENS>;
    static_assert(2 * (sizeof(Smem) + 2048) <= 228 * 1024, "two blocks an SM");
    p.m_tiles = int((q.m + TOKENS - 1) / TOKENS);
    p.n_tiles = int((q.n + 127) / 128);
    p.split = split;
    const int64_t blocks = int64_t(p.m_tiles) * p.n_tiles * split;
    if (blocks > 0x7fffffff) return FPT_ERR_BAD_SIZE;
    return cuda_status(launch_cluster(linear_split_kernel<DT, TOKENS, W_MN>, unsigned(blocks), kSplitThreads, sizeof(Smem) + 1024,
                                      split > 1 ? unsigned(split) : 0u, stream, map_w, map_x, p));
}

template <int DT>
int launch_product(const Product& q, LinearParams& p, const DeviceInfo& dev, cudaStream_t stream) {
    p.m = int(q.m);
    p.n = int(q.n);
    p.k_blocks = int((q.k + kBlockK - 1) / kBlockK);
    const int key = fpt::tuning_linear_tokens();
    int tokens = key >= 0 ? key : q.m <= 16 ? 16 : q.m <= 32 ? 32 : q.m <= 64 ? 64 : q.m <= 256 ? 128 : 0;
    if (q.a_mn) tokens = 0;
    if (tokens) {
        // as many blocks as are resident together (two an SM), at least two K blocks each
        const int64_t tiles = (q.m + tokens - 1) / tokens * ((q.n + 127) / 128);
        int split = int(std::max<int64_t>(1, std::min<int64_t>(kMaxSplit, 2 * dev.sm_count / tiles)));
        if (fpt::tuning_linear_split() > 0) split = fpt::tuning_linear_split();
        split = std::max(1, std::min(split, p.k_blocks / 2));
        auto by_weight = [&](auto t) {
            constexpr int T = decltype(t)::value;
            return q.b_mn ? launch_split<DT, T, true>(q, p, dev, split, stream) : launch_split<DT, T, false>(q, p, dev, split, stream);
        };
        if (tokens == 16) return by_weight(IC<16>{});
        if (tokens == 32) return by_weight(IC<32>{});
        if (tokens == 64) return by_weight(IC<64>{});
        return by_weight(IC<128>{});
    }
    if (q.a_mn) return q.b_mn ? launch_pair<DT, true, true>(q, p, dev, stream) : FPT_ERR_UNSUPPORTED_SHAPE;
    return q.b_mn ? launch_pair<DT, false, true>(q, p, dev, stream) : launch_pair<DT, false, false>(q, p, dev, stream);
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

int run_product(const Product& q, LinearParams& p, int dtype, cudaStream_t stream) {
    DeviceInfo dev;
    if (int rc = current_device_info(&dev)) return rc;
    return dtype == FPT_BF16 ? launch_product<kBf16>(q, p, dev, stream) : launch_product<kFp16>(q, p, dev, stream);
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
    p.act.kind = function == FPT_FN_NONE ? kActNone : degree == 0 ? kActNative : kActProgram;
    p.act.fn = function;
    if (function == FPT_FN_NONE && degree != 0) return FPT_ERR_UNKNOWN_PROGRAM;
    if (p.act.kind == kActProgram) {
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
    return run_product(q, p, dtype, stream);
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
    return run_product(q, p, dtype, stream);
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
    return run_product(q, p, dtype, stream);
}

namespace {
// rows one block sums: enough blocks for every SM several times over, at least 32 rows each
int grad_act_chunk(int64_t rows, int64_t out) {
    const int64_t column_blocks = (out + kActColumns - 1) / kActColumns;
    const int64_t chunks = std::max<int64_t>(1, 148 * 6 / column_blocks);
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
        if (dtype == FPT_BF16) linear_grad_act_kernel<kBf16><<<grid, kActThreads, 0, stream>>>(p);
        else linear_grad_act_kernel<kFp16><<<grid, kActThreads, 0, stream>>>(p);
        if (int rc = cuda_status(cudaGetLastError())) return rc;
    }
    if (dbias) {
        linear_bias_grad_kernel<<<unsigned((out_features + 31) / 32), 256, 0, stream>>>(static_cast<const float*>(workspace), dbias, chunks, int(out_features), bias_dtype);
        return cuda_status(cudaGetLastError());
    }
    return FPT_OK;
}
