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
// the low word is needed.  Sine and cosine are Taylor series on the exact remainder from the nearest quarter turn.  All
// arithmetic is fp32; values are rounded once, when they are stored.
//
// Work split: a lane holds two runs of C dimensions of a head (C = 8 where the sizes are multiples of it, else 4), placed so
// that whole pairs lie in one lane under either pairing; a group of 4 .. 32 lanes holds a head, and the mean is a shuffle
// reduction inside the group.  A block of 256 threads takes a few tokens and computes their sines and cosines once into
// shared memory; each of its groups keeps to one token, so that a lane reads its sines, cosines and weights into registers
// once and walks over the heads with them.  The passes are bound by memory traffic, 2 (forward) or 3 (backward) values per
// value of q and k, once instructions and shared-memory reads are few enough: pairs are kept as two fp32 vectors (first
// members, second members), which costs nothing to unpack, and handled by the two-wide fp32 instructions.
// Measured, 2 x 4096 tokens x (32 + 8) heads x 128 bf16: forward with the norm 29.2 us = 5.7 TB/s, backward 46 us = 5.4 TB/s
// (next to the memory bound by latencies at 16 warps an SM); rotation alone of 15840 such tokens 50.0 us = 6.5 TB/s.  In fp32 at the
// first size: 77 us = 4.4 TB/s, 135 us = 3.7 TB/s, rotation alone 78 us = 4.3 TB/s.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "fpt_common.h"
#include "fpt_qk_rope_plan.h"

namespace fpt {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;
constexpr int kMaxTrig = 2048;          // tokens x pairs of a tile
constexpr int kMaxAxes = 4;
constexpr int kStages = 3;              // items of a thread in its ring
// Blocks an SM holds, by registers (16-bit data; 2 in fp32).  Measured: the forward pass with the norm 29.5 us at 3 and 33.3 at 4
// (which spills), the rotation alone 51.8 at 3 and 50.8 at 4, forward and backward pass together 121 with the backward
// pass at 3 (spills) and 87 at 2 (before the shares of share_blocks).  The backward pass in fp32 with runs of 8 holds 96 KB of
// rings and 18 KB besides: one block is resident and the second half of them follows.  With the sines' arrays cut to what a
// tile uses two are resident, which is not always faster (us, one and two): 2 x 4096 tokens of 32 + 8 heads of 128 135 and 146, of
// 8 + 1 of 256 89 and 81, of 40 + 8 of 80 134 and 124; the 16-byte copies at a stride of 32 bytes ask the L2 for every sector twice.
template <class T, bool NORM>
constexpr int kFwdBlocks = sizeof(T) == 4 ? 2 : NORM ? 3 : 4;
constexpr int kBwdBlocks = 2;

// Launched while the kernel before it drains; nothing of global memory is touched before this.  What that kernel writes changes
// during this one's life, so nothing is read as constant (no __ldg, no __restrict__: such a load may be moved ahead of the wait).
__device__ __forceinline__ void wait_for_inputs() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

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

struct Rows {                          // [batch, seq, heads, dim] by strides in bytes, dim contiguous
    int64_t b, s;
    uint32_t h;
};
struct Side {                          // queries or keys
    const void* x;
    const void* grad;                  // backward: gradient of the output
    void* out;                         // contiguous [batch, seq, heads, dim]
    const void* weight;                // [dim] or null
    float* partial;                    // backward: [blocks, dim] partial weight gradients, or null
    Rows xs, gs;
    uint32_t heads;
    BwdShare share;                    // backward: its tiles and blocks
};
struct QkRopeArgs {
    Side side[2];                      // 0 queries, 1 keys
    const uint32_t* increments;
    const void* positions;             // null: 0 .. seq - 1
    int64_t pos_axis, pos_b, pos_s;    // in elements
    int pos_words;                     // 1: 32-bit positions, 2: 64-bit
    Divider seq, pairs, parts;         // parts: blocks that share the heads of a token (forward)
    uint32_t tokens, tile_tokens;      // tile_tokens: a power of two
    uint32_t groups;                   // heads a block has in hand at a time (forward)
    uint32_t heads_per_part;
    int dim, units, rotary_units;      // lanes of a head that hold something, that rotate
    float eps;
    int weight_dtype;
    uint32_t sin_sign;                 // 0x80000000: rotate backwards
    uint8_t axis[kMaxPairs];
};

// ---- two-wide fp32 --------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// ---- a lane's share of a head -----------------------------------------------------------------------------------------
//
// Two runs of C dimensions, at C unit and at pairs + C unit (dimensions behind the last pair: one run of 2 C), as they are
// stored, and as C pairs: halves pairs dimension lo + p with hi + p; adjacent finds C / 2 pairs in each run.

template <class T, int C>
struct Raw {
    static constexpr int kWords = C * int(sizeof(T)) / 4;
    uint32_t lo[kWords], hi[kWords];
};
template <int C>
struct Pairs {
    uint64_t a[C / 2], b[C / 2];       // first and second members of pairs (2 j, 2 j + 1)
};

struct Place {
    int lo, hi;
};
template <int C>
__device__ __forceinline__ Place place(int unit, int rotary_units) {
    return unit < rotary_units ? Place{C * unit, C * (rotary_units + unit)} : Place{2 * C * unit, 2 * C * unit + C};
}
// dimension of the first / second member of pair p
template <int C, bool HALVES>
__device__ __forceinline__ int member(const Place& at, int p, bool second) {
    if (HALVES) return (second ? at.hi : at.lo) + p;
    return (p < C / 2 ? at.lo + 2 * p : at.hi + 2 * p - C) + (second ? 1 : 0);
}

// Loads go through a ring in shared memory that every thread has to itself: it fills its own 2 C values of the items ahead by
// asynchronous copies and waits for its own copies only, so that loads are in flight all the time without holding
// registers and without a barrier.  Layout [stage][16-byte piece][thread]: no bank conflicts.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const char* from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int AHEAD>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(AHEAD) : "memory"); }

template <int WORDS>
struct Piece {
    static constexpr int kBytes = WORDS % 4 == 0 ? 16 : 8, kCount = WORDS * 4 / kBytes;
};
// one run from a base (the same for the whole block) and a 32-bit offset into this thread's place of the ring
template <int WORDS>
__device__ __forceinline__ void fetch_run(uint32_t to, const char* base, uint32_t offset) {
    using P = Piece<WORDS>;
#pragma unroll
    for (int i = 0; i < P::kCount; ++i) copy_async<P::kBytes>(to + i * (kThreads * P::kBytes), base + offset + i * P::kBytes);
}
template <int WORDS>
__device__ __forceinline__ void read_run(uint32_t (&w)[WORDS], const char* place) {
    using P = Piece<WORDS>;
#pragma unroll
    for (int i = 0; i < P::kCount; ++i) {
        const char* from = place + i * (kThreads * P::kBytes);
        if constexpr (P::kBytes == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(from);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(from);
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    }
}
// the ring of one tensor: stages of both runs of every thread
template <class T, int C, int STAGES>
struct Ring {
    static constexpr int kWords = Raw<T, C>::kWords, kRunBytes = kThreads * kWords * 4, kStageBytes = 2 * kRunBytes;
    static constexpr int kBytes = STAGES * kStageBytes;
    char* mine;
    uint32_t mine_u32;
    __device__ __forceinline__ explicit Ring(char* base) : mine(base + threadIdx.x * Piece<kWords>::kBytes), mine_u32(uint32_t(__cvta_generic_to_shared(mine))) {}
    __device__ __forceinline__ void fetch(uint32_t stage, const char* base, uint32_t lo, uint32_t hi) const {
        fetch_run<kWords>(mine_u32 + stage * kStageBytes, base, lo);
        fetch_run<kWords>(mine_u32 + stage * kStageBytes + kRunBytes, base, hi);
    }
    __device__ __forceinline__ Raw<T, C> read(uint32_t stage) const {
        Raw<T, C> r;
        read_run<kWords>(r.lo, mine + stage * kStageBytes);
        read_run<kWords>(r.hi, mine + stage * kStageBytes + kRunBytes);
        return r;
    }
};
template <int WORDS>
__device__ __forceinline__ void store_run(char* base, uint32_t offset, const uint32_t (&w)[WORDS]) {
    char* to = base + offset;
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    }
}

template <class T>
__device__ __forceinline__ float2 values(uint32_t w) {     // the two 16-bit values of a word
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ uint32_t word(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <class T, int C, bool HALVES>
__device__ __forceinline__ Pairs<C> unpack(const Raw<T, C>& r) {
    Pairs<C> v;
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
        if constexpr (sizeof(T) == 4) {
            const uint32_t* run = HALVES || j < C / 4 ? r.lo : r.hi;
            const int i = HALVES ? 2 * j : 4 * (j % (C / 4));
            const auto f = [](uint32_t w) { return __uint_as_float(w); };
            v.a[j] = HALVES ? two(f(run[i]), f(run[i + 1])) : two(f(run[i]), f(run[i + 2]));
            v.b[j] = HALVES ? two(f(r.hi[i]), f(r.hi[i + 1])) : two(f(run[i + 1]), f(run[i + 3]));
        } else if constexpr (HALVES) {
            const float2 a = values<T>(r.lo[j]), b = values<T>(r.hi[j]);
            v.a[j] = two(a.x, a.y);
            v.b[j] = two(b.x, b.y);
        } else {
            const uint32_t* run = j < C / 4 ? r.lo : r.hi;
            const float2 p = values<T>(run[2 * (j % (C / 4))]), q = values<T>(run[2 * (j % (C / 4)) + 1]);
            v.a[j] = two(p.x, q.x);
            v.b[j] = two(p.y, q.y);
        }
    }
    return v;
}
template <class T, int C, bool HALVES>
__device__ __forceinline__ Raw<T, C> pack(const Pairs<C>& v) {
    Raw<T, C> r;
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
        const float2 a = split(v.a[j]), b = split(v.b[j]);
        if constexpr (sizeof(T) == 4) {
            const auto w = [](float f) { return __float_as_uint(f); };
            if constexpr (HALVES) {
                r.lo[2 * j] = w(a.x), r.lo[2 * j + 1] = w(a.y);
                r.hi[2 * j] = w(b.x), r.hi[2 * j + 1] = w(b.y);
            } else {
                uint32_t* run = j < C / 4 ? r.lo : r.hi;
                const int i = 4 * (j % (C / 4));
                run[i] = w(a.x), run[i + 1] = w(b.x), run[i + 2] = w(a.y), run[i + 3] = w(b.y);
            }
        } else if constexpr (HALVES) {
            r.lo[j] = word<T>(a.x, a.y);
            r.hi[j] = word<T>(b.x, b.y);
        } else {
            uint32_t* run = j < C / 4 ? r.lo : r.hi;
            run[2 * (j % (C / 4))] = word<T>(a.x, b.x);
            run[2 * (j % (C / 4)) + 1] = word<T>(a.y, b.y);
        }
    }
    return r;
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

// sin and cos of 2 pi phase / 2^32.  The phase is reduced to the nearest quarter turn in integers, exactly, and the rest,
// at most pi / 4, goes through the Taylor series (remainders x^11 / 11! < 2^-29 and x^12 / 12! < 2^-33).
__device__ __forceinline__ float2 phase_sincos(uint32_t phase) {
    const uint32_t quarter = (phase + 0x20000000u) >> 30;
    const float x = float(int32_t(phase - (quarter << 30))) * 1.4629180792671596e-9f;       // 2 pi / 2^32
    const float q = x * x;
    float s = fmaf(q, 2.7557319224e-6f, -1.9841269841e-4f);
    s = fmaf(q, s, 8.3333333333e-3f);
    s = fmaf(q, s, -1.6666666667e-1f);
    s = fmaf(x * q, s, x);
    float c = fmaf(q, -2.7557319224e-7f, 2.4801587302e-5f);
    c = fmaf(q, c, -1.3888888889e-3f);
    c = fmaf(q, c, 4.1666666667e-2f);
    c = fmaf(q, c, -0.5f);
    c = fmaf(q, c, 1.0f);
    const float sn = quarter & 1u ? c : s, cs = quarter & 1u ? s : c;
    return make_float2(__uint_as_float(__float_as_uint(sn) ^ (quarter << 30 & 0x80000000u)),
                       __uint_as_float(__float_as_uint(cs) ^ ((quarter + 1u) << 30 & 0x80000000u)));
}

// What the lanes of a block share.  Sines, cosines and weights lie in the order of the lanes, C pairs each; the second four
// of eight lie behind all the first fours, so that neighbouring lanes read neighbouring 16-byte pieces.
struct Shared {
    alignas(16) float cos[kMaxTrig], sin[kMaxTrig];
    alignas(16) float weight[2][2][kMaxPairs];     // [queries / keys][first / second members]
};
// where pair p of a lane lies among the n pairs of a head
template <int C>
__device__ __forceinline__ uint32_t lane_place(uint32_t unit, uint32_t p, uint32_t n) {
    return p / 4 * (n / (C / 4)) + 4 * unit + p % 4;
}
__device__ __forceinline__ uint32_t load_position(const QkRopeArgs& a, uint32_t token, uint32_t pair) {
    const uint32_t b = a.seq.div(token), s = token - b * a.seq.d;
    if (!a.positions) return s;
    const int64_t from = int64_t(a.axis[pair]) * a.pos_axis + int64_t(b) * a.pos_b + int64_t(s) * a.pos_s;
    return static_cast<const uint32_t*>(a.positions)[from * a.pos_words];        // low word
}
// where the sine and cosine of a pair lie among those of its token
template <int C, bool HALVES>
__device__ __forceinline__ uint32_t trig_place(const QkRopeArgs& a, uint32_t pair) {
    if (HALVES) return lane_place<C>(pair / C, pair % C, a.pairs.d);
    const uint32_t second = pair >= a.pairs.d / 2 ? 1u : 0u, in_run = pair - second * (a.pairs.d / 2);
    return lane_place<C>(in_run / (C / 2), second * (C / 2) + in_run % (C / 2), a.pairs.d);
}
__device__ __forceinline__ void put_trig(Shared& sm, const QkRopeArgs& a, uint32_t at, uint32_t phase) {
    const float2 v = phase_sincos(phase);
    sm.cos[at] = v.y;
    sm.sin[at] = __uint_as_float(__float_as_uint(v.x) ^ a.sin_sign);
}
// sines and cosines of `count` tokens from token0 on, by the whole block
template <int C, bool HALVES>
__device__ __forceinline__ void fill_trig(Shared& sm, const QkRopeArgs& a, uint32_t token0, uint32_t count) {
    const uint32_t n = count * a.pairs.d;
    for (uint32_t first = threadIdx.x; first < n; first += 2 * kThreads) {
        uint32_t at[2], phase[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {              // both loads before either sine
            const uint32_t i = min(first + e * kThreads, n - 1), t = a.pairs.div(i), pair = i - t * a.pairs.d;
            at[e] = t * a.pairs.d + trig_place<C, HALVES>(a, pair);
            phase[e] = load_position(a, token0 + t, pair) * a.increments[pair];
        }
        put_trig(sm, a, at[0], phase[0]);
        if (first + kThreads < n) put_trig(sm, a, at[1], phase[1]);
    }
}
// The rows of a tile by 32-bit offsets: from the first token's row where a tile is one token, else from its batch entry
// (the host takes tiles of one token where a batch entry's rows reach further than 32 bits).
__device__ __forceinline__ int64_t tile_base(const Rows& r, const QkRopeArgs& a, uint32_t token0, bool one) {
    const uint32_t b = a.seq.div(token0);
    return int64_t(b) * r.b + (one ? int64_t(token0 - b * a.seq.d) * r.s : 0);
}
__device__ __forceinline__ uint32_t tile_row(const Rows& r, const QkRopeArgs& a, uint32_t token0, uint32_t t, bool one) {
    if (one) return 0u;
    const uint32_t b0 = a.seq.div(token0), b = a.seq.div(token0 + t);
    return uint32_t(int64_t(b - b0) * r.b + int64_t(token0 + t - b * a.seq.d) * r.s);
}

// a lane's C floats out of an array in the order of the lanes, as pairs of two
template <int C>
__device__ __forceinline__ void load_lane(uint64_t (&to)[C / 2], const float* from, uint32_t unit, uint32_t n) {
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(from + i * (n / (C / 4)) + 4 * unit);
        to[2 * i] = two(v.x, v.y);
        to[2 * i + 1] = two(v.z, v.w);
    }
}
template <int C>
struct Angles {
    uint64_t cos[C / 2], sin[C / 2];
};
template <int C>
__device__ __forceinline__ Angles<C> lane_angles(const Shared& sm, const QkRopeArgs& a, uint32_t first, uint32_t unit) {
    Angles<C> r;                                   // lanes that do not turn read the first lane's
    load_lane<C>(r.cos, sm.cos + first, unit < uint32_t(a.rotary_units) ? unit : 0u, a.pairs.d);
    load_lane<C>(r.sin, sm.sin + first, unit < uint32_t(a.rotary_units) ? unit : 0u, a.pairs.d);
    return r;
}
template <int C>
__device__ __forceinline__ Pairs<C> lane_weights(const float (&weight)[2][kMaxPairs], const QkRopeArgs& a, uint32_t unit) {
    Pairs<C> w;
    load_lane<C>(w.a, weight[0], unit, uint32_t(a.dim) / 2);
    load_lane<C>(w.b, weight[1], unit, uint32_t(a.dim) / 2);
    return w;
}

// every pair (a, b) -> scale (a cos - b sin, b cos + a sin)
template <int C, bool SCALED>
__device__ __forceinline__ void turn_pairs(Pairs<C>& v, const Angles<C>& angles, float scale) {
    const uint64_t plus = two(scale, scale), minus = two(-scale, -scale);
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
        uint64_t c = angles.cos[j], s = angles.sin[j];
        const uint64_t n = mul2(s, minus);
        if constexpr (SCALED) {
            c = mul2(c, plus);
            s = mul2(s, plus);
        }
        const uint64_t y = fma2(v.b[j], n, mul2(v.a[j], c));
        v.b[j] = fma2(v.a[j], s, mul2(v.b[j], c));
        v.a[j] = y;
    }
}
// The same where there may be dimensions behind the last pair, which are not mixed (a rotation by nothing would carry an
// infinity over as infinity x 0).  Heads that rotate as a whole take a branch that is the same for the launch: asking every
// lane costs 1.5 % of the passes.
template <int C, bool SCALED>
__device__ __forceinline__ void rotate(Pairs<C>& v, const Angles<C>& angles, float scale, const QkRopeArgs& a, bool turns) {
    if (a.rotary_units == a.units) {
        turn_pairs<C, SCALED>(v, angles, scale);
    } else if (turns) {
        turn_pairs<C, SCALED>(v, angles, scale);
    } else if constexpr (SCALED) {
        const uint64_t plus = two(scale, scale);
#pragma unroll
        for (int j = 0; j < C / 2; ++j) {
            v.a[j] = mul2(v.a[j], plus);
            v.b[j] = mul2(v.b[j], plus);
        }
    }
}
template <int C>
__device__ __forceinline__ Pairs<C> times(const Pairs<C>& v, const Pairs<C>& w) {
    Pairs<C> r;
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
        r.a[j] = mul2(v.a[j], w.a[j]);
        r.b[j] = mul2(v.b[j], w.b[j]);
    }
    return r;
}
// the weight of one dimension per thread, ones where there is none, and its place in shared memory
template <int C, bool HALVES>
__device__ __forceinline__ float fetch_weight(const Side& side, const QkRopeArgs& a) {
    const int e = threadIdx.x, u = e / (2 * C), i = e % (2 * C);
    if (e >= a.dim || !side.weight) return 1.0f;
    return load_weight(side.weight, a.weight_dtype, member<C, HALVES>(place<C>(u, a.rotary_units), i % C, i >= C));
}
template <int C>
__device__ __forceinline__ void keep_weight(float (&weight)[2][kMaxPairs], const QkRopeArgs& a, float w) {
    const int e = threadIdx.x, u = e / (2 * C), i = e % (2 * C);
    if (e < a.dim) weight[i / C][lane_place<C>(uint32_t(u), uint32_t(i % C), uint32_t(a.dim) / 2)] = w;
}

// Lanes that hold nothing (heads that do not fill their group) read what lane 0 reads and count as zeros, and a group past
// the last head or token reads the last one: no load is predicated.
// Without the norm nothing passes between the lanes of a head, and groups of exactly as many lanes as hold something (G = 0)
// leave none idle.
// The heads of a token are numbered through, queries first.  A block has the heads [head0, head1) of its tokens (all of
// them where a tile has several tokens); the groups of a token take them in turn.
template <class T, int C, int G, bool HALVES, bool NORM>
__global__ void __launch_bounds__(kThreads, (kFwdBlocks<T, NORM>)) qk_rope_kernel(const __grid_constant__ QkRopeArgs a) {
    constexpr uint32_t kAhead = kStages - 1;
    extern __shared__ __align__(16) char ring_raw[];
    __shared__ Shared sm;
    const Ring<T, C, kStages> ring(ring_raw);
    const uint32_t tile = a.parts.div(blockIdx.x), part = blockIdx.x - tile * a.parts.d;
    const uint32_t token0 = tile * a.tile_tokens, count = min(a.tile_tokens, a.tokens - token0);
    const bool one = a.tile_tokens == 1;
    const uint32_t group = G ? threadIdx.x / G : threadIdx.x / uint32_t(a.units);
    const int lane_unit = int(threadIdx.x - group * (G ? G : uint32_t(a.units)));
    const uint32_t step = a.groups / a.tile_tokens;                                   // groups of a token
    const bool live = lane_unit < a.units && group < step * a.tile_tokens;
    const int unit = live ? lane_unit : 0;
    const Place at = place<C>(unit, a.rotary_units);
    const uint32_t lo = uint32_t(at.lo) * sizeof(T), hi = uint32_t(at.hi) * sizeof(T), out_bytes = uint32_t(a.dim) * sizeof(T);
    const float inv_dim = 1.0f / float(a.dim);

    wait_for_inputs();
    float weight[2];                               // on their way to shared memory under the first loads of x
    if constexpr (NORM) {
        weight[0] = fetch_weight<C, HALVES>(a.side[0], a);
        weight[1] = fetch_weight<C, HALVES>(a.side[1], a);
    }
    const uint32_t my_slot = group / step, slot = min(my_slot, count - 1);
    const uint32_t q_heads = a.side[0].heads, heads = q_heads + a.side[1].heads;
    const uint32_t head0 = part * a.heads_per_part, head1 = min(head0 + a.heads_per_part, heads);
    const uint32_t head = head0 + group % step, rounds = (head1 - head0 + step - 1) / step;
    const uint32_t end = my_slot < count ? head1 : head0;                             // nothing past the last token is stored
    const char* xq = static_cast<const char*>(a.side[0].x) + tile_base(a.side[0].xs, a, token0, one);
    const char* xk = static_cast<const char*>(a.side[1].x) + tile_base(a.side[1].xs, a, token0, one);
    const uint32_t row_q = tile_row(a.side[0].xs, a, token0, slot, one), row_k = tile_row(a.side[1].xs, a, token0, slot, one);
    char* oq = static_cast<char*>(a.side[0].out) + int64_t(token0) * q_heads * out_bytes;
    char* ok = static_cast<char*>(a.side[1].out) + int64_t(token0) * a.side[1].heads * out_bytes;
    const uint32_t to_q = slot * q_heads * out_bytes, to_k = (slot * a.side[1].heads - q_heads) * out_bytes;
    const auto fetch = [&](uint32_t n) {
        const uint32_t h = min(head + n * step, head1 - 1);
        const bool key = h >= q_heads;
        const uint32_t from = key ? row_k + (h - q_heads) * a.side[1].xs.h : row_q + h * a.side[0].xs.h;
        ring.fetch(n % kStages, key ? xk : xq, from + lo, from + hi);
    };
#pragma unroll
    for (uint32_t n = 0; n < kAhead; ++n) {
        if (n < rounds) fetch(n);
        copy_commit();
    }
    fill_trig<C, HALVES>(sm, a, token0, count);
    if constexpr (NORM) {
        keep_weight<C>(sm.weight[0], a, weight[0]);
        keep_weight<C>(sm.weight[1], a, weight[1]);
    }
    __syncthreads();
    const Angles<C> angles = lane_angles<C>(sm, a, slot * a.pairs.d, unit);
    const bool turns = unit < a.rotary_units;
    Pairs<C> w;
    if constexpr (NORM) w = lane_weights<C>(sm.weight[head >= q_heads], a, unit);
    bool keys = head >= q_heads;                   // whose weights w holds
#pragma unroll 1
    for (uint32_t n = 0; n < rounds; ++n) {
        if (n + kAhead < rounds) fetch(n + kAhead);
        copy_commit();
        copy_wait<kAhead>();
        const uint32_t h = head + n * step;
        const bool key = h >= q_heads;
        Pairs<C> v = unpack<T, C, HALVES>(ring.read(n % kStages));
        float r = 1.0f;
        if constexpr (NORM) {
            if (key != keys) {
                w = lane_weights<C>(sm.weight[1], a, unit);
                keys = true;
            }
            uint64_t ssa = 0, ssb = 0;
#pragma unroll
            for (int j = 0; j < C / 2; ++j) {
                ssa = fma2(v.a[j], v.a[j], ssa);
                ssb = fma2(v.b[j], v.b[j], ssb);
            }
            const float2 sa = split(ssa), sb = split(ssb);
            r = rsqrtf(fmaf(group_sum<G>(live ? (sa.x + sa.y) + (sb.x + sb.y) : 0.0f), inv_dim, a.eps));
            v = times(v, w);
        }
        rotate<C, NORM>(v, angles, r, a, turns);
        if (!live || h >= end) continue;
        const Raw<T, C> y = pack<T, C, HALVES>(v);
        char* out = key ? ok : oq;
        const uint32_t to = h * out_bytes + (key ? to_k : to_q);
        store_run(out, to + lo, y.lo);
        store_run(out, to + hi, y.hi);
    }
}

// Persistent blocks, each on one side; every thread keeps the weight gradient of its dimensions over all heads it meets.
template <class T, int C, int G, bool HALVES>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) qk_norm_rope_bwd_kernel(const __grid_constant__ QkRopeArgs a) {
    constexpr uint32_t kGroups = kThreads / G;
    constexpr uint32_t kAhead = kStages - 1;
    extern __shared__ __align__(16) char ring_raw[];
    __shared__ Shared sm;
    const Ring<T, C, kStages> ring_x(ring_raw), ring_g(ring_raw + Ring<T, C, kStages>::kBytes);
    const int keys = blockIdx.x >= a.side[0].share.blocks;
    const Side& side = a.side[keys];
    const uint32_t block = keys ? blockIdx.x - a.side[0].share.blocks : blockIdx.x;
    const int lane_unit = threadIdx.x & (G - 1);
    const bool live = lane_unit < a.units;
    const int unit = live ? lane_unit : 0;
    const bool turns = unit < a.rotary_units;
    const Place at = place<C>(unit, a.rotary_units);
    const uint32_t lo = uint32_t(at.lo) * sizeof(T), hi = uint32_t(at.hi) * sizeof(T), out_bytes = uint32_t(a.dim) * sizeof(T);
    const float inv_dim = 1.0f / float(a.dim);
    const uint32_t heads = side.heads, step = kGroups / side.share.tile_tokens, group = threadIdx.x / G;
    const uint32_t my_slot = group / step, head = group % step, rounds = (heads + step - 1) / step;
    const bool one = side.share.tile_tokens == 1;
    wait_for_inputs();
    // loads run ahead over the tiles: where they are
    uint32_t ahead_tile = block, ahead_round = 0, ahead_stage = 0, row = 0, row_g = 0;
    const char *x = nullptr, *grad = nullptr;
    const auto aim = [&] {
        const uint32_t token0 = ahead_tile * side.share.tile_tokens, slot = min(my_slot, a.tokens - token0 - 1);
        x = static_cast<const char*>(side.x) + tile_base(side.xs, a, token0, one);
        grad = static_cast<const char*>(side.grad) + tile_base(side.gs, a, token0, one);
        row = tile_row(side.xs, a, token0, slot, one);
        row_g = tile_row(side.gs, a, token0, slot, one);
    };
    const auto fetch = [&] {
        if (ahead_tile < side.share.tiles) {
            const uint32_t h = min(head + ahead_round * step, heads - 1);
            const uint32_t from = row + h * side.xs.h, from_g = row_g + h * side.gs.h;
            ring_x.fetch(ahead_stage, x, from + lo, from + hi);
            ring_g.fetch(ahead_stage, grad, from_g + lo, from_g + hi);
            ahead_stage = ahead_stage + 1 == kStages ? 0 : ahead_stage + 1;
            if (++ahead_round == rounds) {
                ahead_round = 0;
                ahead_tile += side.share.blocks;
                if (ahead_tile < side.share.tiles) aim();
            }
        }
        copy_commit();
    };
    aim();
#pragma unroll
    for (uint32_t n = 0; n < kAhead; ++n) fetch();
    // A thread keeps up two sines and cosines of a tile, the same pairs in every tile.  The positions of the next tile are
    // loaded before a tile's heads and used after them, into the other half of the arrays.
    uint32_t trig_slot[2], trig_at[2], trig_pair[2], increment[2], position[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t i = threadIdx.x + e * kThreads;
        trig_slot[e] = a.pairs.div(i);
        trig_pair[e] = i - trig_slot[e] * a.pairs.d;
        trig_at[e] = trig_slot[e] * a.pairs.d + trig_place<C, HALVES>(a, trig_pair[e]);
        if (trig_slot[e] >= side.share.tile_tokens) trig_slot[e] = 0x40000000u;              // no entry
        increment[e] = trig_slot[e] < side.share.tile_tokens ? a.increments[trig_pair[e]] : 0u;
        position[e] = 0;
    }
    const auto load_positions = [&](uint32_t tile) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t token = tile * side.share.tile_tokens + trig_slot[e];
            if (tile < side.share.tiles && token < a.tokens) position[e] = load_position(a, token, trig_pair[e]);
        }
    };
    const auto put = [&](uint32_t half) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (trig_slot[e] < side.share.tile_tokens) put_trig(sm, a, half * kBwdTrig + trig_at[e], position[e] * increment[e]);
    };
    load_positions(block);
    keep_weight<C>(sm.weight[0], a, fetch_weight<C, HALVES>(side, a));
    put(0);
    __syncthreads();
    Pairs<C> dw;
#pragma unroll
    for (int j = 0; j < C / 2; ++j) dw.a[j] = dw.b[j] = 0;
    uint32_t half = 0, stage = 0;
#pragma unroll 1
    for (uint32_t tile = block; tile < side.share.tiles; tile += side.share.blocks, half ^= 1) {
        const uint32_t token0 = tile * side.share.tile_tokens, count = min(side.share.tile_tokens, a.tokens - token0);
        const uint32_t slot = min(my_slot, count - 1), end = my_slot < count ? heads : 0u;
        char* out = static_cast<char*>(side.out) + int64_t(token0) * heads * out_bytes;
        load_positions(tile + side.share.blocks);
        const Angles<C> angles = lane_angles<C>(sm, a, half * kBwdTrig + slot * a.pairs.d, unit);
#pragma unroll 1
        for (uint32_t n = 0; n < rounds; ++n) {
            fetch();
            copy_wait<kAhead>();
            const uint32_t i = head + n * step;
            Pairs<C> g = unpack<T, C, HALVES>(ring_g.read(stage));
            rotate<C, false>(g, angles, 1.0f, a, turns);
            const Pairs<C> f = unpack<T, C, HALVES>(ring_x.read(stage)), h = times(g, lane_weights<C>(sm.weight[0], a, unit));
            stage = stage + 1 == kStages ? 0 : stage + 1;
            uint64_t ssa = 0, ssb = 0, da = 0, db = 0;
#pragma unroll
            for (int j = 0; j < C / 2; ++j) {
                ssa = fma2(f.a[j], f.a[j], ssa);
                ssb = fma2(f.b[j], f.b[j], ssb);
                da = fma2(h.a[j], f.a[j], da);
                db = fma2(h.b[j], f.b[j], db);
            }
            const float2 sa = split(ssa), sb = split(ssb), ea = split(da), eb = split(db);
            const float r = rsqrtf(fmaf(group_sum<G>(live ? (sa.x + sa.y) + (sb.x + sb.y) : 0.0f), inv_dim, a.eps));
            const float m = group_sum<G>(live ? (ea.x + ea.y) + (eb.x + eb.y) : 0.0f) * r * inv_dim;    // mean(h u)
            if (!live || i >= end) continue;
            // dx = r h - x (r^2 m), dw += (r g) x
            const uint64_t r2 = two(r, r), k2 = two(-r * m * r, -r * m * r);
            Pairs<C> d;
#pragma unroll
            for (int j = 0; j < C / 2; ++j) {
                dw.a[j] = fma2(mul2(g.a[j], r2), f.a[j], dw.a[j]);
                dw.b[j] = fma2(mul2(g.b[j], r2), f.b[j], dw.b[j]);
                d.a[j] = fma2(f.a[j], k2, mul2(h.a[j], r2));
                d.b[j] = fma2(f.b[j], k2, mul2(h.b[j], r2));
            }
            const Raw<T, C> y = pack<T, C, HALVES>(d);
            const uint32_t to = (slot * heads + i) * out_bytes;
            store_run(out, to + lo, y.lo);
            store_run(out, to + hi, y.hi);
        }
        if (tile + side.share.blocks < side.share.tiles) put(half ^ 1);
        __syncthreads();               // the next tile's angles are there, this one's have been read
    }
    if (side.partial) {                // sum over the groups of the block, in the order of the groups, where the ring was
        using Sums = float[kThreads][2 * C + 1];
        static_assert(sizeof(Sums) <= 2 * Ring<T, C, kStages>::kBytes, "the sums fit the ring");
        Sums& sums = *reinterpret_cast<Sums*>(ring_raw);
        copy_wait<0>();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C / 2; ++j) {
            const float2 va = split(dw.a[j]), vb = split(dw.b[j]);
            sums[threadIdx.x][4 * j] = va.x;
            sums[threadIdx.x][4 * j + 1] = va.y;
            sums[threadIdx.x][4 * j + 2] = vb.x;
            sums[threadIdx.x][4 * j + 3] = vb.y;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.dim; e += kThreads) {
            const int u = e / (2 * C), i = e % (2 * C);
            float sum = 0.0f;
            for (uint32_t gr = 0; gr < kGroups; ++gr) sum += sums[gr * G + u][i];
            const int p = i / 4 * 2 + (i & 1);
            side.partial[int64_t(block) * a.dim + member<C, HALVES>(place<C>(u, a.rotary_units), p, (i & 2) != 0)] = sum;
        }
    }
}

// dw[column] = sum of the blocks' partial gradients, always in the same order
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* q_partial, const float* k_partial,
                                                          void* q_out, void* k_out, int q_blocks, int k_blocks, int dim, int dtype) {
    __shared__ float part[256];
    wait_for_inputs();
    const float* partial = blockIdx.y ? k_partial : q_partial;
    void* out = blockIdx.y ? k_out : q_out;
    const int blocks = blockIdx.y ? k_blocks : q_blocks;
    if (!out) return;
    const int column = blockIdx.x * 8 + (threadIdx.x & 7), lane = threadIdx.x >> 3;   // 32 threads a column
    float sum = 0.0f;
#pragma unroll 8
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

// Strides in bytes, zero for dimensions of one entry; false where rows do not start on 16-byte boundaries or heads of one
// token lie further apart than 31 bits.
bool rows_of(Rows& r, const void* p, const int64_t* st, int64_t batch, int64_t seq, int64_t heads, int64_t item) {
    const int64_t b = batch > 1 ? st[0] * item : 0, s = seq > 1 ? st[1] * item : 0, h = heads > 1 ? st[2] * item : 0;
    if (reinterpret_cast<uintptr_t>(p) % 16 || b % 16 || s % 16 || h % 16) return false;
    if (b < 0 || s < 0 || h < 0 || h > 0x7fffffff || h * heads > 0x7fffffff) return false;
    r = Rows{b, s, uint32_t(h)};
    return true;
}
// whether tiles of `tokens` tokens reach their rows by 32-bit offsets from their first batch entry
bool reach(const Rows& r, int64_t seq, int64_t heads, int64_t tokens) {
    const int64_t entries = (tokens + seq - 1) / seq;
    return r.b <= (int64_t(1) << 40) && r.s <= (int64_t(1) << 40) && entries * r.b + (seq - 1) * r.s + heads * r.h + 1024 < (int64_t(1) << 32);
}

// dimensions in one run of a lane
int run_length(int64_t head_dim, int64_t pairs) { return head_dim % 16 == 0 && pairs % 8 == 0 ? 8 : 4; }
int group_lanes(int units) {
    int g = 4;
    while (g < units) g *= 2;
    return g;
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
        const int64_t heads = s ? k_heads : q_heads;
        if (heads && !rows_of(d.xs, d.x, st, batch, seq, heads, int64_t(item))) return FPT_ERR_MISALIGNED;
        d.heads = uint32_t(heads);
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
    const int run = run_length(head_dim, pairs);
    a.units = int(head_dim / (2 * run));
    a.rotary_units = int(pairs / run);
    a.weight_dtype = weight_dtype;
    return FPT_OK;
}

// a launch that may begin while the kernel before it in the stream drains
template <class... P, class... A>
int launch(void (*kernel)(P...), dim3 grid, int smem, cudaStream_t stream, const A&... args) {
    if (smem > 32 * 1024) {            // with the static part, above what a kernel has unasked
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return int(e);
    }
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = size_t(smem);
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&config, kernel, P(args)...));
}

// f(type, run, group, pairing) with compile-time arguments
template <class F>
int dispatch(int dtype, int run, int units, int pairing, F&& f) {
    auto by_pairing = [&](auto type, auto c, auto g) {
        return pairing == FPT_PAIRS_HALVES ? f(type, c, g, std::true_type{}) : f(type, c, g, std::false_type{});
    };
    auto by_group = [&](auto type, auto c) {
        switch (group_lanes(units)) {
        case 4: return by_pairing(type, c, IC<4>{});
        case 8: return by_pairing(type, c, IC<8>{});
        case 16: return by_pairing(type, c, IC<16>{});
        default:
            if constexpr (decltype(c)::value == 4) return by_pairing(type, c, IC<32>{});
            return FPT_ERR_UNSUPPORTED_SHAPE;              // 16 lanes of 16 dimensions hold every head
        }
    };
    auto by_run = [&](auto type) { return run == 8 ? by_group(type, IC<8>{}) : by_group(type, IC<4>{}); };
    if (dtype == FPT_FP32) return by_run(float{});
    if (dtype == FPT_BF16) return by_run(__nv_bfloat16{});
    return by_run(__half{});
}

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
    // One head per group and block while all blocks are resident at once (single tokens: the shortest chain of loads); beyond
    // it a block takes all heads of as many tokens as leave every group at least four heads.  Measured with 32 + 8 heads of
    // 128 in bf16, us one way and the other: 4 tokens 2.4 / 3.8, 128 tokens 3.5 / 4.0, 256 tokens (not resident) 4.9 / 4.1,
    // 512 tokens 7.3 / 4.3; rotation alone, 256 tokens (resident) 3.1 / 3.3.
    const uint32_t groups = uint32_t(kThreads / (norm ? group_lanes(a.units) : a.units)), heads = a.side[0].heads + a.side[1].heads;
    a.groups = groups;
    const uint32_t resident = uint32_t(dev.sm_count * (dtype == FPT_FP32 ? kFwdBlocks<float, true> : norm ? kFwdBlocks<__half, true> : kFwdBlocks<__half, false>));
    const bool few = uint64_t(a.tokens) * ((heads + groups - 1) / groups) <= resident;
    a.tile_tokens = few ? 1u : tile_tokens(groups, heads, uint32_t(pairs), 4, kMaxTrig);
    for (const Side& s : a.side)
        if (!reach(s.xs, seq, s.heads, a.tile_tokens)) a.tile_tokens = 1u;
    const uint32_t tiles = (a.tokens + a.tile_tokens - 1) / a.tile_tokens;
    a.heads_per_part = few ? std::min(groups, heads) : heads;
    a.parts = divider((heads + a.heads_per_part - 1) / a.heads_per_part);
    const unsigned grid = tiles * a.parts.d;
    return dispatch(dtype, run_length(head_dim, pairs), a.units, pairing, [&](auto type, auto c, auto g, auto halves) {
        using T = decltype(type);
        constexpr int C = decltype(c)::value, G = decltype(g)::value;
        constexpr bool H = decltype(halves)::value;
        return norm ? launch(qk_rope_kernel<T, C, G, H, true>, grid, Ring<T, C, kStages>::kBytes, stream, a)
                    : launch(qk_rope_kernel<T, C, 0, H, false>, grid, Ring<T, C, kStages>::kBytes, stream, a);
    });
}

extern "C" int64_t fpt_qk_norm_rope_bwd_workspace_bytes(int64_t q_heads, int64_t k_heads, int64_t head_dim) {
    if (q_heads < 0 || k_heads < 0 || q_heads + k_heads == 0 || head_dim <= 0) return 0;
    DeviceInfo dev;
    if (current_device_info(&dev)) return 0;
    return int64_t(dev.sm_count) * kBwdBlocks * head_dim * int64_t(sizeof(float));
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
        for (int s = 0; s < 2; ++s) {
            Side& d = a.side[s];
            d.grad = s ? dk_out : dq_out;
            if (d.heads && !rows_of(d.gs, d.grad, s ? dk_out_strides : dq_out_strides, batch, seq, d.heads, int64_t(item))) return FPT_ERR_MISALIGNED;
        }
    }
    if (weights && reinterpret_cast<uintptr_t>(workspace) % 4) return FPT_ERR_MISALIGNED;
    DeviceInfo dev;
    if (int rc = current_device_info(&dev)) return rc;
    uint32_t blocks[2] = {0, 0};
    if (weights && a.tokens) {
        if (!workspace) return FPT_ERR_NULL_POINTER;
        if (workspace_bytes < int64_t(dev.sm_count) * kBwdBlocks * head_dim * int64_t(sizeof(float))) return FPT_ERR_SCRATCH_TOO_SMALL;
    }
    float* partial = static_cast<float*>(workspace);
    if (a.tokens) {
        a.eps = eps;
        a.sin_sign = 0x80000000u;
        const uint32_t groups = uint32_t(kThreads / group_lanes(a.units));
        share_blocks(a.side[0].share, a.side[0].heads, a.side[1].share, a.side[1].heads, a.tokens, groups, a.pairs.d,
                     uint32_t(dev.sm_count * kBwdBlocks), [&](int s, uint32_t tile) {
                         return reach(a.side[s].xs, seq, a.side[s].heads, tile) && reach(a.side[s].gs, seq, a.side[s].heads, tile);
                     });
        for (int s = 0; s < 2; ++s) blocks[s] = a.side[s].heads ? a.side[s].share.blocks : 0u;
        for (int s = 0; s < 2; ++s)
            a.side[s].partial = (s ? dk_weight : dq_weight) ? partial + (s ? int64_t(blocks[0]) * head_dim : 0) : nullptr;
        const unsigned grid = blocks[0] + blocks[1];
        const int rc = dispatch(dtype, run_length(head_dim, pairs), a.units, pairing, [&](auto type, auto c, auto g, auto halves) {
            using T = decltype(type);
            constexpr int C = decltype(c)::value;
            return launch(qk_norm_rope_bwd_kernel<T, C, decltype(g)::value, decltype(halves)::value>, grid, 2 * Ring<T, C, kStages>::kBytes, stream, a);
        });
        if (rc) return rc;
    }
    if (weights) {                     // without tokens: zeros
        const float* k_partial = partial ? partial + int64_t(blocks[0]) * head_dim : nullptr;
        return launch(weight_grad_kernel, dim3(unsigned(head_dim / 8), 2), 0, stream, partial, k_partial, dq_weight, dk_weight,
                      int(blocks[0]), int(blocks[1]), int(head_dim), weight_dtype);
    }
    return FPT_OK;
}
