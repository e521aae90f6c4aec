// Queries and keys on their way into the attention, for sm_100a: the root-mean-square norm of every head with a learned
// weight and the position rotation in one pass (fpt_qk_rope with norm), the rotation alone with positions on several axes
// (fpt_qk_rope without), and the backward pass of the first (fpt_qk_norm_rope_bwd; the rotation's own is fpt_qk_rope with
// inverse set).
//
//   r = rsqrt(mean(x^2) + eps),  u = r x,  v = w u,  y = R v            (R: rotation of every pair by its angle)
//   g = R^T dy,  h = w g,  dx = r (h - u mean(h u)),  dw = sum over rows of g u
//
// Angles: the phase of pair i is position * increment_i in 32-bit integers, where one turn is 2^32.  The product wraps as
// the angle does, so the reduction to one turn costs nothing and is exact at every position, and of a 64-bit position only
// the low word is needed.  sine and cosine come from sincospif on phase / 2^31.  All arithmetic is fp32; values are
// rounded once, when they are stored.
//
// Work split: a head of D dimensions is held by a group of G = 8, 16 or 32 lanes, 8 dimensions (4 pairs) a lane whatever
// the pairing, so that the mean is a shuffle reduction inside the group and no pair leaves its lane.  A block of 256
// threads takes a few tokens and some of their heads, computes the sines and cosines of those tokens once into shared
// memory and rotates every head with them.  The passes are bound by memory traffic: 2 (forward), 3 (backward) values per
// value of q and k.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "fpt_common.h"

namespace fpt {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;
constexpr int kMaxTileTokens = 8;
constexpr int kMaxAxes = 4;
constexpr int kLane = 8;              // dimensions one lane holds

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, division by invariant integers): with l = ceil(log2 d)
// and m = ceil(2^(31 + l) / d), floor(n m / 2^(31 + l)) is exact because n (m d - 2^(31 + l)) < 2^31 2^l.
struct Divider {
    uint32_t d, m;
    int shift;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return shift < 0 ? n : __umulhi(n, m) >> shift; }
};
Divider divider(uint32_t d) {
    int l = 0;
    while ((uint64_t(1) << l) < d) ++l;
    return Divider{d, l ? uint32_t(((uint64_t(1) << (31 + l)) + d - 1) / d) : 0u, l - 1};
}

struct Rows {                          // [batch, seq, heads, dim] by strides in elements, dim contiguous
    int64_t b, s, h;
};
struct Side {                          // queries or keys
    const void* x;
    const void* grad;                  // backward: gradient of the output
    void* out;                         // contiguous [batch, seq, heads, dim]
    const void* weight;                // [dim] or null
    float* partial;                    // backward: [blocks, dim] partial weight gradients, or null
    Rows xs, gs;
    uint32_t heads;
    Divider per_block, chunks;         // heads one block takes; blocks over the heads of one token
    uint32_t blocks;
};
struct QkRopeArgs {
    Side side[2];                      // 0 queries, 1 keys
    const uint32_t* increments;
    const void* positions;             // null: 0 .. seq - 1
    int64_t pos_axis, pos_b, pos_s;    // in elements
    int pos_words;                     // 1: 32-bit positions, 2: 64-bit
    Divider seq, pairs;
    uint32_t tokens, tile_tokens, tiles;
    int dim, units, rotary_units;      // units of kLane dimensions; those below rotary_units are rotated
    float eps;
    int weight_dtype;
    uint32_t sin_sign;                 // 0x80000000: rotate backwards
    bool vec_x[2], vec_g[2];           // rows and strides of x / grad allow 16-byte accesses
    uint8_t axis[kMaxPairs];
};

template <class T>
struct Raw;                            // 8 values of one lane as they are stored
template <>
struct Raw<float> {
    uint4 w[2];
};
template <>
struct Raw<__half> {
    uint4 w[1];
};
template <>
struct Raw<__nv_bfloat16> {
    uint4 w[1];
};

template <class T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&f)[kLane]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <class T>
__device__ __forceinline__ Raw<T> pack(const float (&f)[kLane]) {
    Raw<T> r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    return r;
}

// Where a lane's 8 dimensions lie in its head: two runs of four, `lo` and `hi` (adjacent pairs and the dimensions behind
// the last pair: one run of eight, hi = lo + 4).
struct Place {
    int lo, hi;
};
template <bool HALVES>
__device__ __forceinline__ Place place(int unit, int rotary_units) {
    if (HALVES && unit < rotary_units) return Place{4 * unit, 4 * (rotary_units + unit)};
    return Place{8 * unit, 8 * unit + 4};
}

template <class T, bool HALVES>
__device__ __forceinline__ Raw<T> load_lane(const T* head, Place p, bool vec) {
    Raw<T> r;
    if (vec) {
        if constexpr (std::is_same<T, float>::value) {
            r.w[0] = *reinterpret_cast<const uint4*>(head + p.lo);
            r.w[1] = *reinterpret_cast<const uint4*>(head + p.hi);
        } else if constexpr (HALVES) {
            const uint2 a = *reinterpret_cast<const uint2*>(head + p.lo), b = *reinterpret_cast<const uint2*>(head + p.hi);
            r.w[0] = make_uint4(a.x, a.y, b.x, b.y);
        } else {
            r.w[0] = *reinterpret_cast<const uint4*>(head + p.lo);
        }
    } else {                           // any alignment: one value at a time
        T v[kLane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = head[p.lo + i];
            v[4 + i] = head[p.hi + i];
        }
        r = *reinterpret_cast<const Raw<T>*>(v);
    }
    return r;
}
template <class T, bool HALVES>
__device__ __forceinline__ void store_lane(T* head, Place p, const Raw<T>& r) {
    if constexpr (std::is_same<T, float>::value) {
        *reinterpret_cast<uint4*>(head + p.lo) = r.w[0];
        *reinterpret_cast<uint4*>(head + p.hi) = r.w[1];
    } else if constexpr (HALVES) {
        *reinterpret_cast<uint2*>(head + p.lo) = make_uint2(r.w[0].x, r.w[0].y);
        *reinterpret_cast<uint2*>(head + p.hi) = make_uint2(r.w[0].z, r.w[0].w);
    } else {
        *reinterpret_cast<uint4*>(head + p.lo) = r.w[0];
    }
}

// The 4 pairs of a lane: adjacent (0,1) (2,3) .. or halves (0,4) (1,5) ..
template <bool HALVES>
__device__ __forceinline__ void rotate(float (&f)[kLane], const float4& c, const float4& s) {
    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float& a = f[HALVES ? i : 2 * i];
        float& b = f[HALVES ? i + 4 : 2 * i + 1];
        const float y = a * cs[i] - b * sn[i], z = b * cs[i] + a * sn[i];
        a = y;
        b = z;
    }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int m = G / 2; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
    if (dtype == FPT_FP32) return static_cast<const float*>(w)[i];
    if (dtype == FPT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
    return __half2float(static_cast<const __half*>(w)[i]);
}

struct Trig {
    alignas(16) float cos[kMaxTileTokens * kMaxPairs], sin[kMaxTileTokens * kMaxPairs];
};
// sines and cosines of `count` tokens from token0 on, by the whole block
__device__ __forceinline__ void fill_trig(Trig& trig, const QkRopeArgs& a, uint32_t token0, uint32_t count) {
    const uint32_t n = count * a.pairs.d;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t t = a.pairs.div(i), pair = i - t * a.pairs.d;
        const uint32_t token = token0 + t, b = a.seq.div(token), s = token - b * a.seq.d;
        uint32_t position = s;
        if (a.positions) {
            const int64_t at = int64_t(a.axis[pair]) * a.pos_axis + int64_t(b) * a.pos_b + int64_t(s) * a.pos_s;
            position = static_cast<const uint32_t*>(a.positions)[at * a.pos_words];      // low word
        }
        float sn, cs;
        sincospif(float(int32_t(position * a.increments[pair])) * 0x1p-31f, &sn, &cs);
        trig.cos[i] = cs;
        trig.sin[i] = __uint_as_float(__float_as_uint(sn) ^ a.sin_sign);
    }
}

template <class T, int G, bool HALVES, bool NORM>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(const __grid_constant__ QkRopeArgs a) {
    constexpr uint32_t kGroups = kThreads / G;
    constexpr int kUnroll = 4;
    __shared__ Trig trig;
    const bool keys = blockIdx.x >= a.side[0].blocks;
    const Side& side = a.side[keys];
    const uint32_t block = keys ? blockIdx.x - a.side[0].blocks : blockIdx.x;
    const uint32_t tile = side.chunks.div(block), chunk = block - tile * side.chunks.d;
    const uint32_t token0 = tile * a.tile_tokens, count = min(a.tile_tokens, a.tokens - token0);
    const uint32_t head0 = chunk * side.per_block.d;
    const uint32_t items = count * side.per_block.d;
    const int unit = threadIdx.x & (G - 1);
    const uint32_t group = threadIdx.x / G;
    const bool live = unit < a.units, turns = unit < a.rotary_units;
    const Place at = place<HALVES>(unit, a.rotary_units);
    const T* x = static_cast<const T*>(side.x);
    T* out = static_cast<T*>(side.out);
    const bool vec = a.vec_x[keys];

    float w[kLane];
    if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < kLane; ++i)
            w[i] = live && side.weight ? load_weight(side.weight, a.weight_dtype, (i < 4 ? at.lo : at.hi - 4) + i) : 1.0f;
    }
    bool filled = false;
    const float inv_dim = 1.0f / float(a.dim);
    for (uint32_t first = 0; first < items; first += kGroups * kUnroll) {
        Raw<T> raw[kUnroll];
        uint32_t slot[kUnroll];
        int64_t to[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = first + uint32_t(k) * kGroups + group;
            slot[k] = side.per_block.div(i);
            const uint32_t head = head0 + i - slot[k] * side.per_block.d, token = token0 + slot[k];
            to[k] = -1;
            raw[k] = Raw<T>{};
            if (i < items && head < side.heads && live) {
                const uint32_t b = a.seq.div(token), s = token - b * a.seq.d;
                to[k] = (int64_t(token) * side.heads + head) * a.dim;
                raw[k] = load_lane<T, HALVES>(x + (int64_t(b) * side.xs.b + int64_t(s) * side.xs.s + int64_t(head) * side.xs.h), at, vec);
            }
        }
        if (!filled) {                 // under the first loads
            fill_trig(trig, a, token0, count);
            __syncthreads();
            filled = true;
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            float f[kLane];
            unpack<T>(raw[k], f);
            if constexpr (NORM) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < kLane; ++i) ss = fmaf(f[i], f[i], ss);
                const float r = rsqrtf(fmaf(group_sum<G>(ss), inv_dim, a.eps));
#pragma unroll
                for (int i = 0; i < kLane; ++i) f[i] = f[i] * r * w[i];
            }
            if (to[k] < 0) continue;
            if (turns) {
                const uint32_t e = slot[k] * a.pairs.d + 4u * uint32_t(unit);
                rotate<HALVES>(f, *reinterpret_cast<const float4*>(&trig.cos[e]), *reinterpret_cast<const float4*>(&trig.sin[e]));
            }
            store_lane<T, HALVES>(out + to[k], at, pack<T>(f));
        }
    }
}

// Persistent blocks, each on one side; every thread keeps the weight gradient of its 8 dimensions over all heads it meets.
template <class T, int G, bool HALVES>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_bwd_kernel(const __grid_constant__ QkRopeArgs a) {
    constexpr uint32_t kGroups = kThreads / G;
    constexpr int kUnroll = 2;
    __shared__ union {
        Trig trig;
        float dw[kThreads * kLane];
    } sm;
    const bool keys = blockIdx.x >= a.side[0].blocks;
    const Side& side = a.side[keys];
    const uint32_t block = keys ? blockIdx.x - a.side[0].blocks : blockIdx.x;
    const int unit = threadIdx.x & (G - 1);
    const uint32_t group = threadIdx.x / G;
    const bool live = unit < a.units, turns = unit < a.rotary_units;
    const Place at = place<HALVES>(unit, a.rotary_units);
    const T* x = static_cast<const T*>(side.x);
    const T* grad = static_cast<const T*>(side.grad);
    T* out = static_cast<T*>(side.out);
    const bool vec_x = a.vec_x[keys], vec_g = a.vec_g[keys];
    float w[kLane], dw[kLane];
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
        w[i] = live && side.weight ? load_weight(side.weight, a.weight_dtype, (i < 4 ? at.lo : at.hi - 4) + i) : 1.0f;
        dw[i] = 0.0f;
    }
    const float inv_dim = 1.0f / float(a.dim);
    for (uint32_t tile = block; tile < a.tiles; tile += side.blocks) {
        const uint32_t token0 = tile * a.tile_tokens, count = min(a.tile_tokens, a.tokens - token0);
        const uint32_t items = count * side.heads;
        bool filled = false;
        for (uint32_t first = 0; first < items; first += kGroups * kUnroll) {
            Raw<T> raw[kUnroll], raw_g[kUnroll];
            uint32_t slot[kUnroll];
            int64_t to[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const uint32_t i = first + uint32_t(k) * kGroups + group;
                slot[k] = side.per_block.div(i);
                const uint32_t head = i - slot[k] * side.heads, token = token0 + slot[k];
                to[k] = -1;
                raw[k] = Raw<T>{};
                raw_g[k] = Raw<T>{};
                if (i < items && live) {
                    const uint32_t b = a.seq.div(token), s = token - b * a.seq.d;
                    to[k] = (int64_t(token) * side.heads + head) * a.dim;
                    raw[k] = load_lane<T, HALVES>(x + (int64_t(b) * side.xs.b + int64_t(s) * side.xs.s + int64_t(head) * side.xs.h), at, vec_x);
                    raw_g[k] = load_lane<T, HALVES>(grad + (int64_t(b) * side.gs.b + int64_t(s) * side.gs.s + int64_t(head) * side.gs.h), at, vec_g);
                }
            }
            if (!filled) {
                __syncthreads();       // the previous tile's angles have been read
                fill_trig(sm.trig, a, token0, count);
                __syncthreads();
                filled = true;
            }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                float f[kLane], g[kLane];
                unpack<T>(raw[k], f);
                unpack<T>(raw_g[k], g);
                if (turns && to[k] >= 0) {
                    const uint32_t e = slot[k] * a.pairs.d + 4u * uint32_t(unit);
                    rotate<HALVES>(g, *reinterpret_cast<const float4*>(&sm.trig.cos[e]), *reinterpret_cast<const float4*>(&sm.trig.sin[e]));
                }
                float ss = 0.0f, dot = 0.0f;
#pragma unroll
                for (int i = 0; i < kLane; ++i) {
                    ss = fmaf(f[i], f[i], ss);
                    dot = fmaf(g[i] * w[i], f[i], dot);
                }
                const float r = rsqrtf(fmaf(group_sum<G>(ss), inv_dim, a.eps));
                const float m = group_sum<G>(dot) * r * inv_dim;          // mean(h u)
                if (to[k] < 0) continue;
#pragma unroll
                for (int i = 0; i < kLane; ++i) {
                    const float u = f[i] * r;
                    dw[i] = fmaf(g[i], u, dw[i]);
                    f[i] = r * fmaf(g[i], w[i], -u * m);
                }
                store_lane<T, HALVES>(out + to[k], at, pack<T>(f));
            }
        }
    }
    if (side.partial) {                // sum over the groups of the block, in the order of the groups
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLane; ++i) sm.dw[threadIdx.x * kLane + i] = dw[i];
        __syncthreads();
        for (int e = threadIdx.x; e < a.units * kLane; e += kThreads) {
            const int u = e / kLane, i = e - u * kLane;
            float sum = 0.0f;
            for (uint32_t gr = 0; gr < kGroups; ++gr) sum += sm.dw[(gr * G + u) * kLane + i];
            const Place p = place<HALVES>(u, a.rotary_units);
            side.partial[int64_t(block) * a.dim + (i < 4 ? p.lo : p.hi - 4) + i] = sum;
        }
    }
}

// dw[column] = sum of the blocks' partial gradients, always in the same order
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* __restrict__ q_partial, const float* __restrict__ k_partial,
                                                          void* q_out, void* k_out, int q_blocks, int k_blocks, int dim, int dtype) {
    __shared__ float part[256];
    const float* partial = blockIdx.y ? k_partial : q_partial;
    void* out = blockIdx.y ? k_out : q_out;
    const int blocks = blockIdx.y ? k_blocks : q_blocks;
    if (!out) return;
    const int column = blockIdx.x * 8 + (threadIdx.x & 7), lane = threadIdx.x >> 3;   // 32 threads a column
    float sum = 0.0f;
    for (int b = lane; b < blocks; b += 32) sum += partial[int64_t(b) * dim + column];
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int half = 128; half >= 8; half >>= 1) {
        if (int(threadIdx.x) < half) part[threadIdx.x] += part[threadIdx.x + half];
        __syncthreads();
    }
    if (threadIdx.x < 8) {
        const float v = part[threadIdx.x];
        if (dtype == FPT_FP32) static_cast<float*>(out)[column] = v;
        else if (dtype == FPT_BF16) static_cast<__nv_bfloat16*>(out)[column] = __float2bfloat16_rn(v);
        else static_cast<__half*>(out)[column] = __float2half_rn(v);
    }
}

template <int V>
using IC = std::integral_constant<int, V>;

bool vectors(const void* p, const Rows& r, int64_t batch, int64_t seq, int64_t heads, size_t item) {
    const int64_t step = 16 / int64_t(item);
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (batch < 2 || r.b % step == 0) && (seq < 2 || r.s % step == 0) &&
           (heads < 2 || r.h % step == 0);
}

// what both directions share; returns a status
int prepare(QkRopeArgs& a, const void* q, const void* k, void* q_out, void* k_out, const void* q_weight, const void* k_weight,
            const void* increments, const void* positions, int position_bits, const int64_t* pos_strides,
            const uint8_t* pair_axes, int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads, int64_t head_dim,
            int64_t pairs, const int64_t* q_strides, const int64_t* k_strides, int pairing, int dtype, int weight_dtype) {
    if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0) return FPT_ERR_BAD_SIZE;
    if (head_dim <= 0 || head_dim % 8 || head_dim > 2 * kMaxPairs) return FPT_ERR_UNSUPPORTED_SHAPE;
    if (pairs <= 0 || pairs % 4 || 2 * pairs > head_dim) return FPT_ERR_UNSUPPORTED_SHAPE;
    if (pairing != FPT_PAIRS_ADJACENT && pairing != FPT_PAIRS_HALVES) return FPT_ERR_BAD_ENUM;
    if (dtype < FPT_FP16 || dtype > FPT_FP32 || weight_dtype < FPT_FP16 || weight_dtype > FPT_FP32) return FPT_ERR_BAD_ENUM;
    if (positions && position_bits != 32 && position_bits != 64) return FPT_ERR_BAD_ENUM;
    // token counts and block counts (at most one block a head) stay below 2^31
    if (seq > 0 && batch > (int64_t(1) << 30) / seq) return FPT_ERR_BAD_SIZE;
    const int64_t tokens = batch * seq;
    if (std::max(q_heads, k_heads) > 65535 || tokens * std::max<int64_t>(q_heads + k_heads, 1) > (int64_t(1) << 34)) return FPT_ERR_BAD_SIZE;
    if (tokens == 0 || q_heads + k_heads == 0) return FPT_OK;
    if (!increments || !q_strides || !k_strides || (positions && !pos_strides)) return FPT_ERR_NULL_POINTER;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return FPT_ERR_NULL_POINTER;
    const size_t item = dtype == FPT_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(q_out) % 16 || reinterpret_cast<uintptr_t>(k_out) % 16) return FPT_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(q) % item || reinterpret_cast<uintptr_t>(k) % item) return FPT_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(increments) % 4 || reinterpret_cast<uintptr_t>(positions) % size_t(position_bits ? position_bits / 8 : 4))
        return FPT_ERR_MISALIGNED;
    const size_t weight_item = weight_dtype == FPT_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(q_weight) % weight_item || reinterpret_cast<uintptr_t>(k_weight) % weight_item) return FPT_ERR_MISALIGNED;
    for (int s = 0; s < 2; ++s) {
        Side& d = a.side[s];
        const int64_t* st = s ? k_strides : q_strides;
        d.x = s ? k : q;
        d.out = s ? k_out : q_out;
        d.weight = s ? k_weight : q_weight;
        d.xs = Rows{st[0], st[1], st[2]};
        d.heads = uint32_t(s ? k_heads : q_heads);
        a.vec_x[s] = vectors(d.x, d.xs, batch, seq, d.heads, item);
    }
    a.increments = static_cast<const uint32_t*>(increments);
    a.positions = positions;
    a.pos_words = position_bits == 64 ? 2 : 1;
    if (positions) { a.pos_axis = pos_strides[0]; a.pos_b = pos_strides[1]; a.pos_s = pos_strides[2]; }
    for (int64_t i = 0; i < pairs; ++i) {
        a.axis[i] = pair_axes ? pair_axes[i] : 0;
        if (a.axis[i] >= kMaxAxes) return FPT_ERR_BAD_ENUM;
    }
    a.seq = divider(uint32_t(seq));
    a.pairs = divider(uint32_t(pairs));
    a.tokens = uint32_t(tokens);
    a.dim = int(head_dim);
    a.units = int(head_dim / kLane);
    a.rotary_units = int(pairs / 4);
    a.weight_dtype = weight_dtype;
    return FPT_OK;
}

// f(type, group size, pairing) with compile-time arguments
template <class F>
int dispatch(int dtype, int units, int pairing, F&& f) {
    auto by_pairing = [&](auto type, auto g) {
        return pairing == FPT_PAIRS_HALVES ? f(type, g, std::true_type{}) : f(type, g, std::false_type{});
    };
    auto by_group = [&](auto type) {
        if (units <= 8) return by_pairing(type, IC<8>{});
        if (units <= 16) return by_pairing(type, IC<16>{});
        return by_pairing(type, IC<32>{});
    };
    if (dtype == FPT_FP32) return by_group(float{});
    if (dtype == FPT_BF16) return by_group(__nv_bfloat16{});
    return by_group(__half{});
}
int group_lanes(int units) { return units <= 8 ? 8 : units <= 16 ? 16 : 32; }

}  // namespace
}  // namespace fpt

using namespace fpt;

extern "C" int fpt_qk_rope(void* q_out, void* k_out, const void* q, const void* k, const void* q_weight, const void* k_weight,
                           const void* phase_increments, const void* positions, int position_bits, const int64_t* position_strides,
                           const uint8_t* pair_axes, int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads,
                           int64_t head_dim, int64_t pairs, const int64_t* q_strides, const int64_t* k_strides, int pairing,
                           int norm, float eps, int inverse, int dtype, int weight_dtype, fpt_stream_t stream) {
    QkRopeArgs a{};
    if (int rc = prepare(a, q, k, q_out, k_out, q_weight, k_weight, phase_increments, positions, position_bits, position_strides,
                         pair_axes, batch, seq, q_heads, k_heads, head_dim, pairs, q_strides, k_strides, pairing, dtype, weight_dtype))
        return rc;
    if (norm && !(eps >= 0.0f)) return FPT_ERR_BAD_SIZE;
    if (norm && inverse) return FPT_ERR_BAD_ENUM;
    if (a.tokens == 0) return FPT_OK;
    DeviceInfo dev;
    if (int rc = current_device_info(&dev)) return rc;
    a.eps = eps;
    a.sin_sign = inverse ? 0x80000000u : 0u;
    // One head per group and block while that gives no more than a few blocks per SM (single tokens: the shortest chain
    // of loads); beyond it a block takes all heads of as many tokens as give every group eight heads.
    const uint32_t groups = uint32_t(kThreads / group_lanes(a.units));
    const uint64_t rows = uint64_t(a.tokens) * (a.side[0].heads + a.side[1].heads);
    const bool few = rows <= uint64_t(groups) * uint64_t(dev.sm_count) * 4;
    const uint32_t heads = std::max(a.side[0].heads, a.side[1].heads);
    a.tile_tokens = few ? 1u : std::max(1u, std::min<uint32_t>(kMaxTileTokens, groups * 8 / heads));
    a.tiles = (a.tokens + a.tile_tokens - 1) / a.tile_tokens;
    for (Side& s : a.side) {
        const uint32_t per = std::max(1u, std::min(s.heads, few ? groups : groups * 8));
        s.per_block = divider(per);
        s.chunks = divider(std::max(1u, (s.heads + per - 1) / per));
        s.blocks = s.heads ? a.tiles * s.chunks.d : 0u;
    }
    const unsigned grid = a.side[0].blocks + a.side[1].blocks;
    return dispatch(dtype, a.units, pairing, [&](auto type, auto g, auto halves) {
        using T = decltype(type);
        constexpr int G = decltype(g)::value;
        constexpr bool H = decltype(halves)::value;
        if (norm) qk_rope_kernel<T, G, H, true><<<grid, kThreads, 0, stream>>>(a);
        else qk_rope_kernel<T, G, H, false><<<grid, kThreads, 0, stream>>>(a);
        return cuda_status(cudaGetLastError());
    });
}

namespace {
// blocks of the backward pass on the query side and on the key side: persistent, shared out by the heads
void bwd_blocks(int64_t q_heads, int64_t k_heads, int sm_count, uint32_t (&blocks)[2]) {
    const int64_t total = int64_t(sm_count) * 4, heads = q_heads + k_heads;
    blocks[0] = q_heads ? uint32_t(std::max<int64_t>(1, (total * q_heads + heads / 2) / heads)) : 0u;
    blocks[1] = k_heads ? uint32_t(std::max<int64_t>(1, total - (q_heads ? int64_t(blocks[0]) : 0))) : 0u;
}
}  // namespace

extern "C" int64_t fpt_qk_norm_rope_bwd_workspace_bytes(int64_t q_heads, int64_t k_heads, int64_t head_dim) {
    if (q_heads < 0 || k_heads < 0 || q_heads + k_heads == 0 || head_dim <= 0) return 0;
    DeviceInfo dev;
    if (current_device_info(&dev)) return 0;
    uint32_t blocks[2];
    bwd_blocks(q_heads, k_heads, dev.sm_count, blocks);
    return (int64_t(blocks[0]) + blocks[1]) * head_dim * int64_t(sizeof(float));
}

extern "C" int fpt_qk_norm_rope_bwd(void* dq, void* dk, void* dq_weight, void* dk_weight, const void* dq_out, const void* dk_out,
                                    const void* q, const void* k, const void* q_weight, const void* k_weight,
                                    const void* phase_increments, const void* positions, int position_bits,
                                    const int64_t* position_strides, const uint8_t* pair_axes, void* workspace,
                                    int64_t workspace_bytes, int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads,
                                    int64_t head_dim, int64_t pairs, const int64_t* q_strides, const int64_t* k_strides,
                                    const int64_t* dq_out_strides, const int64_t* dk_out_strides, int pairing, float eps,
                                    int dtype, int weight_dtype, fpt_stream_t stream) {
    QkRopeArgs a{};
    if (int rc = prepare(a, q, k, dq, dk, q_weight, k_weight, phase_increments, positions, position_bits, position_strides,
                         pair_axes, batch, seq, q_heads, k_heads, head_dim, pairs, q_strides, k_strides, pairing, dtype, weight_dtype))
        return rc;
    if (!(eps >= 0.0f)) return FPT_ERR_BAD_SIZE;
    const bool weights = dq_weight || dk_weight;
    const size_t item = dtype == FPT_FP32 ? 4 : 2;
    if (a.tokens) {
        if ((q_heads && (!dq_out || !dq_out_strides)) || (k_heads && (!dk_out || !dk_out_strides))) return FPT_ERR_NULL_POINTER;
        if (reinterpret_cast<uintptr_t>(dq_out) % item || reinterpret_cast<uintptr_t>(dk_out) % item) return FPT_ERR_MISALIGNED;
    }
    if (weights && reinterpret_cast<uintptr_t>(workspace) % 4) return FPT_ERR_MISALIGNED;
    DeviceInfo dev;
    if (int rc = current_device_info(&dev)) return rc;
    uint32_t blocks[2] = {0, 0};
    if (a.tokens) bwd_blocks(q_heads, k_heads, dev.sm_count, blocks);
    if (weights && a.tokens) {
        if (!workspace) return FPT_ERR_NULL_POINTER;
        if (workspace_bytes < (int64_t(blocks[0]) + blocks[1]) * head_dim * int64_t(sizeof(float))) return FPT_ERR_SCRATCH_TOO_SMALL;
    }
    float* partial = static_cast<float*>(workspace);
    if (a.tokens) {
        a.eps = eps;
        a.sin_sign = 0x80000000u;
        const uint32_t groups = uint32_t(kThreads / group_lanes(a.units));
        const uint32_t heads = std::max(a.side[0].heads, a.side[1].heads);
        a.tile_tokens = std::max(1u, std::min<uint32_t>(kMaxTileTokens, groups * 8 / heads));
        // no more tokens a tile than keep every block busy
        while (a.tile_tokens > 1 && a.tokens / a.tile_tokens < std::max(blocks[0], blocks[1])) --a.tile_tokens;
        a.tiles = (a.tokens + a.tile_tokens - 1) / a.tile_tokens;
        for (int s = 0; s < 2; ++s) {
            Side& d = a.side[s];
            const int64_t* st = s ? dk_out_strides : dq_out_strides;
            d.grad = s ? dk_out : dq_out;
            if (d.heads) {
                d.gs = Rows{st[0], st[1], st[2]};
                a.vec_g[s] = vectors(d.grad, d.gs, batch, seq, d.heads, item);
            }
            blocks[s] = std::min(blocks[s], a.tiles);
            d.blocks = blocks[s];
            d.per_block = divider(std::max(1u, d.heads));
            d.partial = (s ? dk_weight : dq_weight) ? partial + (s ? int64_t(blocks[0]) * head_dim : 0) : nullptr;
        }
        const unsigned grid = blocks[0] + blocks[1];
        const int rc = dispatch(dtype, a.units, pairing, [&](auto type, auto g, auto halves) {
            qk_norm_rope_bwd_kernel<decltype(type), decltype(g)::value, decltype(halves)::value><<<grid, kThreads, 0, stream>>>(a);
            return cuda_status(cudaGetLastError());
        });
        if (rc) return rc;
    }
    if (weights) {                     // without tokens: zeros
        weight_grad_kernel<<<dim3{unsigned(head_dim / 8), 2}, 256, 0, stream>>>(partial, partial ? partial + int64_t(blocks[0]) * head_dim : nullptr,
                                                                              dq_weight, dk_weight, int(blocks[0]), int(blocks[1]), int(head_dim), weight_dtype);
        return cuda_status(cudaGetLastError());
    }
    return FPT_OK;
}
