// The norm of every query and key head, and the position rotation, in one pass over the tensors:
//
//     r = 1 / sqrt(mean(x^2) + eps),   n = x r w,
//     y[j] = n[j] cos[j] - n[j + half] sin[j],   y[j + half] = n[j + half] cos[j + half] + n[j] sin[j + half]
//
// over a head's d features, the first dim = 2 half of which are rotated by their token's row of the tables; and the gradient of that,
// with g the gradient of y turned back (the transpose of the rotation) and a = g w:
//
//     dw = sum over tokens and heads of g x r,   dx = r a - x r^3 sum(x a) / d.
//
// Everything between the load and the store is f32, so a result is rounded once (the rotation alone, rope.cu, rounds its products as
// the reference's whole-tensor form does; here there is no such form to follow).  Nothing is kept for the backward: it
// reads x anyway and r is one reduction away.  Both are a read and a write of each tensor (the backward two reads), bound by HBM.
//
// A head belongs to a few neighbouring lanes.  A lane holds V columns of the lower half of the rotated features and the V
// they are paired with (behind the rotated ones: V columns and the V half of the rest further on), so that the rotation is within a
// lane and the norm is a sum over the lanes of a head, three shuffles at d = 128.  A warp takes one token's heads of one tensor,
// HG to a lane, so that the token's row of the tables and the weights are fetched once for them and all loads are on their way before
// the first is used.
#include <algorithm>

#include "common.cuh"
#include "qk_norm.h"
#include "sm100_ptx.cuh"

namespace dash {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ int64_t index_at(const void *p, int bytes, int64_t i) {
    return bytes == 8 ? static_cast<const int64_t *>(p)[i] : static_cast<int64_t>(static_cast<const int32_t *>(p)[i]);
}

Over over_of(int64_t d) {   // (1 <= d < 2^31)
    int l = 0;
    while ((int64_t(1) << l) < d) ++l;
    return Over{(uint32_t)((uint64_t(1) << 32) * ((uint64_t(1) << l) - d) / d + 1), l};
}

// What a warp of the ring kernel takes of one tensor at a time.
struct RingPlan {
    int heads, units;    // of a token; units of them to a token
    int tokens;          // of a stage
    int slots;           // of them that the lanes of a warp take at once, a power of two
    int stage;           // bytes
};

// n / d for 0 <= n < 2^31 and d >= 1 by a multiplication (Granlund and Montgomery: m = floor(2^32 (2^l - d) / d) + 1, l = ceil(log2 d)).
__device__ __forceinline__ uint32_t over(uint32_t n, const Over &o) { return (__umulhi(n, o.mul) + n) >> o.shift; }

// n = (batch element, token of it).
__device__ __forceinline__ void token_of(const NormArgs &a, int64_t n, int64_t &bi, int64_t &ti) {
    bi = 0;
    ti = n;
    if (a.b == 1) return;
    if (((n | a.t) >> 31) == 0) {
        bi = over((uint32_t)n, a.over_t);
        ti = (uint32_t)n - (uint32_t)bi * (uint32_t)a.t;
    } else {
        bi = n / a.t;
        ti = n - bi * a.t;
    }
}

// The tokens [from, to) of the packed sequence that was found last (of no sequence where `held` is false): tokens are asked for in their
// order, and most are of the sequence of the one before.
struct Sequence {
    int64_t from = 0, to = 0;
    bool held = false;
};

// The position of token n = (.., ti): its row of the tables; -1 for one outside them, -2 for a token of no sequence.  Each lane for itself.
__device__ __forceinline__ int64_t table_row(const NormArgs &a, int64_t n, int64_t ti, Sequence &seq) {
    int64_t pos;
    if (a.positions) {
        pos = index_at(a.positions, a.pos_bytes, n);
    } else if (a.cu) {
        if (n < seq.from || n >= seq.to) {
            // The last offset that is <= n.
            int lo = -1, hi = a.sequences + 1;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (index_at(a.cu, a.cu_bytes, mid) <= n) lo = mid; else hi = mid;
            }
            seq.held = lo >= 0 && lo < a.sequences;
            seq.from = lo >= 0 ? index_at(a.cu, a.cu_bytes, lo) : 0;
            seq.to = lo < a.sequences ? index_at(a.cu, a.cu_bytes, lo + 1) : 0x7fffffffffffffffLL;
        }
        if (!seq.held) return -2;
        pos = a.start + n - seq.from;
    } else {
        pos = a.start + ti;
    }
    return pos >= 0 && pos < a.len ? pos : -1;
}
// The same where all 32 lanes ask for one token, once: each looks at one offset, 32 of them a look, so that a batch of up to 31 sequences
// takes one trip to memory where the bisection takes one per step.
__device__ __forceinline__ int64_t table_row_warp(const NormArgs &a, int64_t n, int64_t ti) {
    int64_t pos;
    if (!a.positions && a.cu) {
        const int lane = threadIdx.x & 31;
        int lo = 0, count = a.sequences + 1;   // among count offsets from lo on lies the last one that is <= n, if any
        int64_t from = 0;
        for (;;) {
            const int hop = (count + 31) / 32, mine = lo + lane * hop;
            const int64_t offset = mine < lo + count ? index_at(a.cu, a.cu_bytes, mine) : 0x7fffffffffffffffLL;
            const unsigned below = __ballot_sync(0xffffffffu, offset <= n);
            if (below == 0) return -2;   // (only at the first look: before the first offset)
            const int last = 31 - __clz(below);
            from = __shfl_sync(0xffffffffu, offset, last);
            count = min(hop, count - last * hop);
            lo += last * hop;
            if (hop == 1) break;
        }
        if (lo >= a.sequences) return -2;   // behind the last offset
        pos = a.start + n - from;
    } else {
        pos = a.positions ? index_at(a.positions, a.pos_bytes, n) : a.start + ti;
    }
    return pos >= 0 && pos < a.len ? pos : -1;
}

// V elements of T as they lie in memory, 16 bytes or 8 (weights in f32 beside 16-bit tensors: twice that), and as pairs of f32, two
// to a packed instruction.
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? 8 : 16) Vec { T e[V]; };
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load(const T *p) {
    Vec<T, V> v;
    if constexpr (sizeof(v) == 8) *reinterpret_cast<uint2 *>(&v) = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
    for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4 *>(&v)[i] = reinterpret_cast<const uint4 *>(p)[i];
    return v;
}
template <typename T, int V> __device__ __forceinline__ void store(T *p, const Vec<T, V> &v) {
    if constexpr (sizeof(v) == 8) *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(&v);
    else *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&v);
}
template <int V> __device__ __forceinline__ float2 pair(const Vec<float, V> &v, int i) { return make_float2(v.e[2 * i], v.e[2 * i + 1]); }
template <int V> __device__ __forceinline__ float2 pair(const Vec<__nv_bfloat16, V> &v, int i) {
    const uint32_t u = reinterpret_cast<const uint32_t *>(&v)[i];
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <int V> __device__ __forceinline__ float2 pair(const Vec<__half, V> &v, int i) { return __half22float2(reinterpret_cast<const __half2 *>(&v)[i]); }
template <int V> __device__ __forceinline__ void put(Vec<float, V> &v, int i, float2 x) { v.e[2 * i] = x.x; v.e[2 * i + 1] = x.y; }
template <int V> __device__ __forceinline__ void put(Vec<__nv_bfloat16, V> &v, int i, float2 x) { reinterpret_cast<__nv_bfloat162 *>(&v)[i] = __float22bfloat162_rn(x); }
template <int V> __device__ __forceinline__ void put(Vec<__half, V> &v, int i, float2 x) { reinterpret_cast<__half2 *>(&v)[i] = __float22half2_rn(x); }

template <int LPH> __device__ __forceinline__ float head_sum(float x) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }

// A lane's place in a head of the vector kernels.
template <int V, int LPH> struct Place {
    int c1, c2;      // its columns: c1 .. c1 + V and c2 .. c2 + V
    bool live, rotated;
    __device__ __forceinline__ Place(const NormArgs &a, int lane) {
        const int i = lane % LPH, pairs = a.dim / (2 * V);
        live = i < a.d / (2 * V);
        rotated = i < pairs;
        c1 = rotated ? i * V : a.dim + (i - pairs) * V;
        c2 = c1 + (rotated ? a.dim : a.d - a.dim) / 2;
    }
};

// The weights of a lane's columns, as they lie in memory; ones where there are none.
template <typename TW, int V, int LPH> struct Weights {
    Vec<TW, V> w1, w2;
    __device__ __forceinline__ Weights(const void *w, const Place<V, LPH> &at) {
#pragma unroll
        for (int e = 0; e < V; ++e) w1.e[e] = w2.e[e] = Num<TW>::from_f32(1.f);
        if (w && at.live) {
            w1 = load<TW, V>(static_cast<const TW *>(w) + at.c1);
            w2 = load<TW, V>(static_cast<const TW *>(w) + at.c2);
        }
    }
};

// Cosines and sines of a lane's columns, as they lie in memory: the token's row; NaN for a position outside the tables (nothing is read there);
// no rotation for columns behind the rotated ones.
template <typename T, int V, int LPH> struct Turn {
    Vec<T, V> c1, c2, s1, s2;
    __device__ __forceinline__ Turn(const NormArgs &a, int64_t row, const Place<V, LPH> &at) {
        const bool turned = at.live && at.rotated;
        if (turned && row >= 0) {
            const T *cs = static_cast<const T *>(a.cos) + row * a.dim + at.c1, *sn = static_cast<const T *>(a.sin) + row * a.dim + at.c1;
            c1 = load<T, V>(cs);
            c2 = load<T, V>(cs + a.dim / 2);
            s1 = load<T, V>(sn);
            s2 = load<T, V>(sn + a.dim / 2);
        } else {
            const T c = Num<T>::from_f32(turned ? nan_f32() : 1.f), s = Num<T>::from_f32(turned ? nan_f32() : 0.f);
#pragma unroll
            for (int e = 0; e < V; ++e) { c1.e[e] = c2.e[e] = c; s1.e[e] = s2.e[e] = s; }
        }
    }
};

// The weight is multiplied into the token's cosines and sines, once for all heads of the lane: y1 = r (x1 w1 c1 - x2 w2 s1) and
// y2 = r (x2 w2 c2 + x1 w1 s2) are then two products and two sums a column.
template <typename T, typename TW, int V, int LPH, int HG>
__global__ void __launch_bounds__(THREADS) qk_norm_kernel(NormArgs a, int units_q, int units, Over over_units) {
    constexpr int NG = 32 / LPH;   // heads of a warp's load
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int64_t n = (warp >> 31) == 0 ? (int64_t)over((uint32_t)warp, over_units) : warp / units;
    if (n >= a.b * a.t) return;
    const int unit = (int)(warp - n * units);
    const bool is_k = unit >= units_q;
    const NormTensor &t = is_k ? a.k : a.q;
    const int h0 = (is_k ? unit - units_q : unit) * NG * HG + lane / LPH;
    const Place<V, LPH> at(a, lane);
    int64_t bi, ti;
    token_of(a, n, bi, ti);
    const int64_t hop = NG * t.sh;
    const T *x = static_cast<const T *>(t.x) + bi * t.sb + ti * t.st + h0 * t.sh + at.c1;
    T *out = static_cast<T *>(t.out) + (n * t.heads + h0) * a.d + at.c1;
    const int other = at.c2 - at.c1;
    Vec<T, V> x1[HG], x2[HG];
#pragma unroll
    for (int g = 0; g < HG; ++g) {
        if (at.live && h0 + g * NG < t.heads) {
            x1[g] = load<T, V>(x + g * hop);
            x2[g] = load<T, V>(x + g * hop + other);
        }
    }
    const Weights<TW, V, LPH> w(t.w, at);
    const int64_t row = table_row_warp(a, n, ti);
    float2 k1[V / 2], k2[V / 2], z1[V / 2], z2[V / 2];   // w1 c1, w2 c2, -w2 s1, w1 s2
    {
        const Turn<T, V, LPH> turn(a, row, at);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            k1[i] = ptx::mul2(pair<V>(w.w1, i), pair<V>(turn.c1, i));
            k2[i] = ptx::mul2(pair<V>(w.w2, i), pair<V>(turn.c2, i));
            z1[i] = at.rotated ? neg2(ptx::mul2(pair<V>(w.w2, i), pair<V>(turn.s1, i))) : both(0.f);
            z2[i] = at.rotated ? ptx::mul2(pair<V>(w.w1, i), pair<V>(turn.s2, i)) : both(0.f);
        }
    }
    const float inv_d = 1.f / a.d;
#pragma unroll
    for (int g = 0; g < HG; ++g) {
        const bool live = at.live && h0 + g * NG < t.heads;
        float2 u1[V / 2], u2[V / 2], sum = both(0.f);
        if (live) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                u1[i] = pair<V>(x1[g], i);
                u2[i] = pair<V>(x2[g], i);
                sum = ptx::fma2(u1[i], u1[i], ptx::fma2(u2[i], u2[i], sum));
            }
        }
        const float r = rsqrtf(fmaf(head_sum<LPH>(sum.x + sum.y), inv_d, a.eps));
        if (!live) continue;
        if (row != -2) {   // (a token of no sequence passes unchanged)
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                put<V>(x1[g], i, ptx::mul2(ptx::fma2(u1[i], k1[i], ptx::mul2(u2[i], z1[i])), both(r)));
                put<V>(x2[g], i, ptx::mul2(ptx::fma2(u2[i], k2[i], ptx::mul2(u1[i], z2[i])), both(r)));
            }
            if (r == 0.f && !at.rotated) {   // an infinity in the head: columns behind the rotated ones are no partners, and it times a sine of zero no zero
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    put<V>(x1[g], i, ptx::mul2(ptx::mul2(u1[i], k1[i]), both(r)));
                    put<V>(x2[g], i, ptx::mul2(ptx::mul2(u2[i], k2[i]), both(r)));
                }
            }
        }
        store<T, V>(out + g * NG * a.d, x1[g]);
        store<T, V>(out + g * NG * a.d + other, x2[g]);
    }
}

// A block's sums of the weight's gradient, from its warps' lanes, into its row of the scratch.
template <int V, int LPH, int NW>
__device__ __forceinline__ void leave_part(const NormArgs &a, const Place<V, LPH> &at, const float2 (&d1)[V / 2], const float2 (&d2)[V / 2], float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float u1 = e & 1 ? d1[e / 2].y : d1[e / 2].x, u2 = e & 1 ? d2[e / 2].y : d2[e / 2].x;
#pragma unroll
        for (int o = LPH; o < 32; o <<= 1) {
            u1 += __shfl_xor_sync(0xffffffffu, u1, o);
            u2 += __shfl_xor_sync(0xffffffffu, u2, o);
        }
        if (lane < LPH && at.live) {
            red[warp * a.d + at.c1 + e] = u1;
            red[warp * a.d + at.c2 + e] = u2;
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += NW * 32) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += red[i * a.d + c];
        a.part[(int64_t)blockIdx.x * a.d + c] = sum;
    }
}

// ---------------------------------------------------------------------------------------------
// Calls of many tokens, and the gradient
// ---------------------------------------------------------------------------------------------
// The blocks up to blocks_q take the queries, the others the keys; a warp takes the same heads of one token after another, or, where a
// token's heads are few, all heads of several tokens at a time.  What it needs of a token - its heads, the gradient of them, the token's
// row of the tables - comes as whole runs of bytes, each asked for by one lane, into a ring of two stages of shared memory of the
// warp's own: the tokens behind the ones it works on are on their way meanwhile at the price of neither registers nor instructions, and
// the warps of a block know nothing of one another.
// The weight's gradient: a lane's sums are one tensor's columns and stay in registers to the end.
__device__ unsigned int g_qk_norm_status = 0;   // sticky: non-zero once a bounded wait has run out

// Of a stage: HG loads of 32 / LPH heads each.  Four warps a block and three blocks a multiprocessor: 168 registers, with which next to nothing spills (backward in 16 bits one to five words).
template <bool BACK> struct Ring {
    static constexpr int HG = BACK ? 4 : 8, STAGES = 2, WARPS = 4, BLOCKS = 3;
};
constexpr int STAGE_MOST = 9216;   // bytes: three blocks of four warps of two fill a multiprocessor's shared memory
constexpr int stage_bytes(bool back, int heads, int tokens, int d, int dim, int eb) { return (heads * d * (back ? 2 : 1) + tokens * 2 * dim) * eb; }

// `heads` of a token, `sh` elements apart: one run where they lie side by side, else one each.
template <typename T>
__device__ __forceinline__ void heads_load(const NormArgs &a, const T *x, int64_t sh, int heads, uint32_t to, uint32_t bar) {
    const int size = a.d * (int)sizeof(T);
    if (sh == a.d) {
        ptx::bulk_load(to, x, heads * size, bar);
    } else {
        for (int h = 0; h < heads; ++h) ptx::bulk_load(to + h * size, x + h * sh, size, bar);
    }
}

// A lane's cosines and sines as f32 pairs; forward the weight is multiplied in, once for all heads of a token:
// y1 = r (x1 k1 + x2 z1), y2 = r (x2 k2 + x1 z2) with k1 = w1 c1, k2 = w2 c2, z1 = -w2 s1, z2 = w1 s2; backward c1, c2, -s1, s2.
// `kind` 0: the row is there; else NaN.  Columns behind the rotated ones: no rotation.
template <typename T, typename TW, int V, int LPH, bool BACK>
struct Factors {
    float2 k1[V / 2], k2[V / 2], z1[V / 2], z2[V / 2];
    __device__ __forceinline__ void set(const T *row, int dim, const Place<V, LPH> &at, const Weights<TW, V, LPH> &w, unsigned kind) {
        Vec<T, V> c1, c2, s1, s2;
        const bool turned = at.live && at.rotated;
        if (turned && kind == 0) {
            c1 = load<T, V>(row + at.c1);
            c2 = load<T, V>(row + at.c2);
            s1 = load<T, V>(row + dim + at.c1);
            s2 = load<T, V>(row + dim + at.c2);
        } else {
            const T c = Num<T>::from_f32(turned ? nan_f32() : 1.f), z = Num<T>::from_f32(turned ? nan_f32() : 0.f);
#pragma unroll
            for (int e = 0; e < V; ++e) { c1.e[e] = c2.e[e] = c; s1.e[e] = s2.e[e] = z; }
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            k1[i] = pair<V>(c1, i);
            k2[i] = pair<V>(c2, i);
            z1[i] = neg2(pair<V>(s1, i));
            z2[i] = pair<V>(s2, i);
            if constexpr (!BACK) {
                const float2 w1 = pair<V>(w.w1, i), w2 = pair<V>(w.w2, i);
                k1[i] = ptx::mul2(k1[i], w1);
                k2[i] = ptx::mul2(k2[i], w2);
                z1[i] = at.rotated ? ptx::mul2(z1[i], w2) : both(0.f);
                z2[i] = at.rotated ? ptx::mul2(z2[i], w1) : both(0.f);
            }
        }
    }
};

template <typename T, typename TW, int V, int LPH, bool BACK>
__global__ void __launch_bounds__(Ring<BACK>::WARPS * 32, Ring<BACK>::BLOCKS) qk_norm_ring_kernel(NormArgs a, RingPlan of_q, RingPlan of_k, int blocks_q) {
    using R = Ring<BACK>;
    constexpr int NG = 32 / LPH, STAGES = R::STAGES, NW = R::WARPS;
    extern __shared__ __align__(128) uint8_t smem[];   // barriers [NW][STAGES], rings [NW][STAGES][stage]; at the end the sums [NW][d]
    if constexpr (BACK) allow_beside();   // the sums over the blocks
    const int lane = threadIdx.x & 31, wib = threadIdx.x >> 5;
    const bool is_k = (int)blockIdx.x >= blocks_q;
    const NormTensor &t = is_k ? a.k : a.q;
    const RingPlan &plan = is_k ? of_k : of_q;
    const int units = plan.units, each = plan.tokens;
    const bool many = each > 1;
    const int row_size = a.dim * (int)sizeof(T), head_size = a.d * (int)sizeof(T);
    const int xs_at = each * 2 * row_size, ys_at = xs_at + plan.heads * each * head_size;   // in a stage: the tables' rows, x, the gradients
    uint8_t *mine = smem + 128 + wib * STAGES * plan.stage;
    const uint32_t mine_u32 = ptx::smem_u32(mine), bars = ptx::smem_u32(smem) + wib * STAGES * 8;
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) ptx::mbar_init(bars + 8 * s, many ? 32 : 1);
        ptx::fence_mbar_init();
    }
    __syncwarp();
    // Warps in whole sets of `units`; what is left over (fewer than `units`) stands by.  (More units than warps: one set, in rounds.)
    const int warps = (is_k ? gridDim.x - blocks_q : blocks_q) * NW, number = (is_k ? blockIdx.x - blocks_q : blockIdx.x) * NW + wib;
    const int sets = max(warps / units, 1), set = warps >= units ? number / units : 0;
    bool failed = *reinterpret_cast<volatile unsigned int *>(&g_qk_norm_status) != 0;   // (an earlier launch's: nothing is done)
    const int64_t tokens = set < sets && !failed ? a.b * a.t : 0;
    const int64_t first = (int64_t)set * each, step = (int64_t)sets * each;
    const Place<V, LPH> at(a, lane);
    const int slots = plan.slots, beside = NG / slots, slot = lane / LPH / beside, part = lane / LPH % beside;   // tokens at once, heads of each
    const Weights<TW, V, LPH> w(t.w, at);
    const float inv_d = 1.f / a.d;
    float2 d1[V / 2], d2[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) d1[i] = d2[i] = both(0.f);
    unsigned phase = 0, pending = 0;   // bit per stage: the parity waited for next; whether its copies have been asked for and not met
    for (int unit = number - set * units; unit < units && !failed; unit += warps >= units ? units : warps) {
        const int h0 = unit * plan.heads, heads = min(plan.heads, t.heads - h0);
        unsigned what = 0;   // two bits per stage, of this lane's token: 0 a row of the tables is there, 1 the position is outside them, 2 a token of no sequence
        Sequence seq;
        // The tokens from n on into stage s: lane i asks for the i-th of them.
        auto ask = [&](int64_t n, int s) {
            if (n >= tokens) return;
            pending |= 1u << s;
            if (!many && lane != 0) return;
            const uint32_t bar = bars + 8 * s, to = mine_u32 + s * plan.stage;
            n += lane;
            if (lane >= each || n >= tokens) {
                ptx::mbar_arrive(bar);
                return;
            }
            int64_t bi, ti;
            token_of(a, n, bi, ti);
            const int64_t row = table_row(a, n, ti, seq);
            what = (what & ~(3u << (2 * s))) | ((unsigned)(row >= 0 ? 0 : -row) << (2 * s));
            ptx::mbar_expect_tx(bar, (BACK ? 2 : 1) * heads * head_size + (row >= 0 ? 2 * row_size : 0));
            if (row >= 0) {
                ptx::bulk_load(to + lane * 2 * row_size, static_cast<const T *>(a.cos) + row * a.dim, row_size, bar);
                ptx::bulk_load(to + lane * 2 * row_size + row_size, static_cast<const T *>(a.sin) + row * a.dim, row_size, bar);
            }
            heads_load<T>(a, static_cast<const T *>(t.x) + bi * t.sb + ti * t.st + h0 * t.sh, t.sh, heads, to + xs_at + lane * heads * head_size, bar);
            if constexpr (BACK)
                heads_load<T>(a, static_cast<const T *>(t.g) + bi * t.gb + ti * t.gt + h0 * t.gh, t.gh, heads, to + ys_at + lane * heads * head_size, bar);
        };
        ask(first, 0);
        int s = 0;
        for (int64_t n = first; n < tokens; n += step) {
            __syncwarp();   // (the stage that is asked for next has been read by every lane)
            ask(n + step, s ^ 1);
            __syncwarp();
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(bars + 8 * s, phase >> s & 1u))) { failed = true; break; }
            phase ^= 1u << s;
            pending &= ~(1u << s);
            const uint8_t *stage = mine + s * plan.stage;
            const T *xs = reinterpret_cast<const T *>(stage + xs_at), *ys = reinterpret_cast<const T *>(stage + ys_at);
            T *out = static_cast<T *>(t.out) + (n * t.heads + h0) * a.d;
            const unsigned kinds = what >> (2 * s) & 3u;
            const int there = (int)min((int64_t)each, tokens - n);
            // The lanes of a head take heads of one token in turn, so that its factors, which cost more than a head, are made once for them.
            for (int token0 = 0; token0 < there; token0 += slots) {
                const int token = min(token0 + slot, there - 1);
                const unsigned kind = __shfl_sync(0xffffffffu, kinds, token);
                Factors<T, TW, V, LPH, BACK> f;
                f.set(reinterpret_cast<const T *>(stage + token * 2 * row_size), a.dim, at, w, kind);
#pragma unroll 2
                for (int r0 = 0; r0 < heads; r0 += beside) {
                    const int row = token * heads + r0 + part;   // the head, of the stage's all
                    const bool live = at.live && r0 + part < heads && token0 + slot < there;
                    float2 u1[V / 2], u2[V / 2], g1[V / 2], g2[V / 2], square = both(0.f), along = both(0.f);
                    Vec<T, V> y1, y2;
                    if (live) {
                        const Vec<T, V> x1 = load<T, V>(xs + row * a.d + at.c1), x2 = load<T, V>(xs + row * a.d + at.c2);
                        if constexpr (BACK) {
                            y1 = load<T, V>(ys + row * a.d + at.c1);
                            y2 = load<T, V>(ys + row * a.d + at.c2);
                        } else {
                            y1 = x1;
                            y2 = x2;
                        }
#pragma unroll
                        for (int i = 0; i < V / 2; ++i) {
                            u1[i] = pair<V>(x1, i);
                            u2[i] = pair<V>(x2, i);
                            square = ptx::fma2(u1[i], u1[i], ptx::fma2(u2[i], u2[i], square));
                            if constexpr (BACK) {
                                g1[i] = pair<V>(y1, i);
                                g2[i] = pair<V>(y2, i);
                                if (at.rotated) {   // (no partners behind the rotated ones: an infinite one times a sine of zero would be no zero)
                                    const float2 v1 = g1[i], v2 = g2[i];
                                    g1[i] = ptx::fma2(v1, f.k1[i], ptx::mul2(v2, f.z2[i]));
                                    g2[i] = ptx::fma2(v2, f.k2[i], ptx::mul2(v1, f.z1[i]));
                                }
                                along = ptx::fma2(ptx::mul2(g1[i], pair<V>(w.w1, i)), u1[i], ptx::fma2(ptx::mul2(g2[i], pair<V>(w.w2, i)), u2[i], along));
                            }
                        }
                    }
                    const float r = rsqrtf(fmaf(head_sum<LPH>(square.x + square.y), inv_d, a.eps));
                    const float back = BACK ? -head_sum<LPH>(along.x + along.y) * inv_d * r : 0.f;
                    if (!live) continue;
                    if (kind != 2) {   // (a token of no sequence passes unchanged, and so does its gradient)
#pragma unroll
                        for (int i = 0; i < V / 2; ++i) {
                            if constexpr (BACK) {
                                const float2 n1 = ptx::mul2(u1[i], both(r)), n2 = ptx::mul2(u2[i], both(r));
                                put<V>(y1, i, ptx::mul2(ptx::fma2(n1, both(back), ptx::mul2(g1[i], pair<V>(w.w1, i))), both(r)));
                                put<V>(y2, i, ptx::mul2(ptx::fma2(n2, both(back), ptx::mul2(g2[i], pair<V>(w.w2, i))), both(r)));
                                d1[i] = ptx::fma2(g1[i], n1, d1[i]);
                                d2[i] = ptx::fma2(g2[i], n2, d2[i]);
                            } else {
                                put<V>(y1, i, ptx::mul2(ptx::fma2(u1[i], f.k1[i], ptx::mul2(u2[i], f.z1[i])), both(r)));
                                put<V>(y2, i, ptx::mul2(ptx::fma2(u2[i], f.k2[i], ptx::mul2(u1[i], f.z2[i])), both(r)));
                            }
                        }
                        if (!BACK && r == 0.f && !at.rotated) {   // (an infinity in the head, as above)
#pragma unroll
                            for (int i = 0; i < V / 2; ++i) {
                                put<V>(y1, i, ptx::mul2(ptx::mul2(u1[i], f.k1[i]), both(r)));
                                put<V>(y2, i, ptx::mul2(ptx::mul2(u2[i], f.k2[i]), both(r)));
                            }
                        }
                    }
                    store<T, V>(out + row * a.d + at.c1, y1);
                    store<T, V>(out + row * a.d + at.c2, y2);
                }
            }
            s ^= 1;
        }
        __syncwarp();
    }
    if (failed) {
        // The sums are not what they should be, and look like none that are.
        if constexpr (BACK) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) d1[i] = d2[i] = both(nan_f32());
        }
        // A copy did not come: the call has failed and says so; what else is on its way is waited for (again not for ever).
        for (int s = 0; s < STAGES; ++s)
            if (pending >> s & 1u) ptx::mbar_wait(bars + 8 * s, phase >> s & 1u);
        if (lane == 0) atomicOr(&g_qk_norm_status, 16u);
    }
    if constexpr (BACK) {
        __syncthreads();   // (the sums lie over the rings)
        leave_part<V, LPH, NW>(a, at, d1, d2, reinterpret_cast<float *>(smem + 128));
    }
}

// ---------------------------------------------------------------------------------------------
// Head dimensions, strides and addresses that do not allow 16 bytes at a time: a warp a head, an element at a time
// ---------------------------------------------------------------------------------------------
constexpr int EACH = 8;   // items of a lane: pairs first, then the features behind the rotated ones, at most 256 in all

template <typename T> __device__ __forceinline__ float at_f32(const void *p, int64_t i) { return Num<T>::to_f32(static_cast<const T *>(p)[i]); }
__device__ __forceinline__ float weight_at(const void *w, bool f32, bool bf16, int c) {
    if (!w) return 1.f;
    if (f32) return static_cast<const float *>(w)[c];
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(w)[c]) : __half2float(static_cast<const __half *>(w)[c]);
}
template <typename T> struct IsBf16 { static constexpr bool value = false; };
template <> struct IsBf16<__nv_bfloat16> { static constexpr bool value = true; };

// Item i of a head: columns c1 and, for a pair, c2.
__device__ __forceinline__ bool item_of(const NormArgs &a, int i, int &c1, int &c2, bool &pair) {
    const int half = a.dim / 2;
    pair = i < half;
    c1 = pair ? i : i + half;
    c2 = pair ? i + half : c1;
    return i < a.d - half;
}

template <typename T, bool BACK>
__global__ void __launch_bounds__(THREADS) qk_norm_elements_kernel(NormArgs a, int blocks_q) {
    extern __shared__ float red[];
    if constexpr (BACK) allow_beside();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool w_f32 = a.w_f32 || sizeof(T) == 4;
    const bool is_k = (int)blockIdx.x >= blocks_q;
    const NormTensor &t = is_k ? a.k : a.q;
    const int64_t first = (int64_t)(is_k ? blockIdx.x - blocks_q : blockIdx.x) * WARPS + warp;
    const int64_t step = (int64_t)(is_k ? gridDim.x - blocks_q : blocks_q) * WARPS, all = a.b * a.t * t.heads;
    float d1[EACH], d2[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) d1[e] = d2[e] = 0.f;
    Sequence seq;
    for (int64_t item = first; item < all; item += step) {
        const int64_t n = item / t.heads;
        const int h = (int)(item - n * t.heads);
        int64_t bi, ti;
        token_of(a, n, bi, ti);
        const int64_t xo = bi * t.sb + ti * t.st + h * t.sh, go = bi * t.gb + ti * t.gt + h * t.gh, oo = item * a.d;
        const int64_t row = table_row(a, n, ti, seq);
        float u1[EACH], u2[EACH], g1[EACH], g2[EACH], square = 0.f, along = 0.f;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            int c1, c2;
            bool pair;
            u1[e] = u2[e] = g1[e] = g2[e] = 0.f;
            if (!item_of(a, lane + 32 * e, c1, c2, pair)) continue;
            u1[e] = at_f32<T>(t.x, xo + c1);
            if (pair) u2[e] = at_f32<T>(t.x, xo + c2);
            square = fmaf(u1[e], u1[e], fmaf(u2[e], u2[e], square));
            if constexpr (BACK) {
                const float v1 = at_f32<T>(t.g, go + c1), v2 = pair ? at_f32<T>(t.g, go + c2) : 0.f;
                if (row == -2) {
                    g1[e] = v1;
                    g2[e] = v2;
                    continue;
                }
                g1[e] = v1;
                if (pair) {
                    const bool known = row >= 0;
                    const float k1 = known ? at_f32<T>(a.cos, row * a.dim + c1) : nan_f32(), k2 = known ? at_f32<T>(a.cos, row * a.dim + c2) : nan_f32();
                    const float s1 = known ? at_f32<T>(a.sin, row * a.dim + c1) : nan_f32(), s2 = known ? at_f32<T>(a.sin, row * a.dim + c2) : nan_f32();
                    g1[e] = v1 * k1 + v2 * s2;
                    g2[e] = v2 * k2 - v1 * s1;
                }
                along = fmaf(u1[e] * weight_at(t.w, w_f32, IsBf16<T>::value, c1), g1[e], along);
                if (pair) along = fmaf(u2[e] * weight_at(t.w, w_f32, IsBf16<T>::value, c2), g2[e], along);
            }
        }
        const float r = rsqrtf(warp_sum(square) / a.d + a.eps);
        const float back = BACK ? warp_sum(along) / a.d * r * r * r : 0.f;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            int c1, c2;
            bool pair;
            if (!item_of(a, lane + 32 * e, c1, c2, pair)) continue;
            T *out = static_cast<T *>(t.out) + oo;
            if (row == -2) {
                const void *from = BACK ? t.g : t.x;
                const int64_t o = BACK ? go : xo;
                out[c1] = static_cast<const T *>(from)[o + c1];
                if (pair) out[c2] = static_cast<const T *>(from)[o + c2];
                continue;
            }
            const float w1 = weight_at(t.w, w_f32, IsBf16<T>::value, c1), w2 = pair ? weight_at(t.w, w_f32, IsBf16<T>::value, c2) : 0.f;
            if constexpr (BACK) {
                out[c1] = Num<T>::from_f32(r * w1 * g1[e] - u1[e] * back);
                if (pair) out[c2] = Num<T>::from_f32(r * w2 * g2[e] - u2[e] * back);
                d1[e] = fmaf(g1[e], u1[e] * r, d1[e]);
                d2[e] = fmaf(g2[e], u2[e] * r, d2[e]);
            } else {
                const float n1 = u1[e] * r * w1, n2 = u2[e] * r * w2;
                float y1 = n1, y2 = n2;
                if (pair) {
                    const bool known = row >= 0;
                    const float k1 = known ? at_f32<T>(a.cos, row * a.dim + c1) : nan_f32(), k2 = known ? at_f32<T>(a.cos, row * a.dim + c2) : nan_f32();
                    const float s1 = known ? at_f32<T>(a.sin, row * a.dim + c1) : nan_f32(), s2 = known ? at_f32<T>(a.sin, row * a.dim + c2) : nan_f32();
                    y1 = n1 * k1 - n2 * s1;
                    y2 = n2 * k2 + n1 * s2;
                }
                out[c1] = Num<T>::from_f32(y1);
                if (pair) out[c2] = Num<T>::from_f32(y2);
            }
        }
    }
    if constexpr (BACK) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            int c1, c2;
            bool pair;
            if (!item_of(a, lane + 32 * e, c1, c2, pair)) continue;
            red[warp * a.d + c1] = d1[e];
            if (pair) red[warp * a.d + c2] = d2[e];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.d; c += THREADS) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) sum += red[i * a.d + c];
            a.part[(int64_t)blockIdx.x * a.d + c] = sum;
        }
    }
}

// The weight's gradient from the blocks' rows, in their order: a block 32 columns of one tensor, as many warps as it may have, so that each has
// one trip or two to memory (the gradient of 1000 tokens of 16 / 4 heads of 128, 8 warps | 32: 12.0 | 10.0 us).
constexpr int SUM_WARPS = 32;
template <typename TW>
__global__ void __launch_bounds__(SUM_WARPS * 32) qk_norm_sum_kernel(NormArgs a, int blocks_q, int blocks) {
    __shared__ float red[SUM_WARPS][32];
    wait_before();
    const bool is_k = blockIdx.y == 1;
    const NormTensor &t = is_k ? a.k : a.q;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const int b0 = is_k ? blocks_q : 0, b1 = is_k ? blocks : blocks_q;
    float sum = 0.f;
    if (t.dw && c < a.d) {
#pragma unroll 8
        for (int i = b0 + warp; i < b1; i += SUM_WARPS) sum += a.part[(int64_t)i * a.d + c];
    }
    red[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || !t.dw || c >= a.d) return;
#pragma unroll
    for (int i = 1; i < SUM_WARPS; ++i) sum += red[i][lane];
    static_cast<TW *>(t.dw)[c] = Num<TW>::from_f32(sum);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
enum Way { ELEMENTS, HEADS, RING };
struct Plan {
    Way way;
    int columns, lph;        // of a lane, twice; lanes of a head
    int units_q, units_k;    // HEADS: warps of a token
    RingPlan ring_q, ring_k;
    int blocks_q, blocks;    // the ring's and the element kernels' blocks: the queries', and all
};

constexpr int HEADS_EACH = 2;          // loads of a token's heads by a warp of the kernel of few tokens
constexpr int MAX_BLOCKS = 148 * 8;    // rows of the backward's scratch

Plan plan_of(int dtype, const NormArgs &a, bool back) {
    const int eb = dtype == 0 ? 4 : 2, v = 16 / eb;
    auto aligned = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    auto vectors = [&](const NormTensor &t) {
        return t.heads == 0 || (aligned(t.x) && aligned(t.out) && t.sb % v == 0 && t.st % v == 0 && t.sh % v == 0 && aligned(t.w) &&
                                (!back || (aligned(t.g) && t.gb % v == 0 && t.gt % v == 0 && t.gh % v == 0)));
    };
    Plan p{};
    // A lane's columns are 16 bytes where the halves that are paired are whole vectors, else (40 rotated of 80 in 16 bits) 8; the rows and the heads
    // are whole vectors in any case, for the copies.  (16384 tokens of 16 / 4 such heads, element by element | so: 184 | 48 us, backward 411 | 70.)
    auto whole = [&](int columns) { return a.dim % (2 * columns) == 0 && a.d % (2 * columns) == 0; };
    p.columns = eb == 2 && !whole(v) ? v / 2 : v;
    const bool vec = whole(p.columns) && aligned(a.cos) && aligned(a.sin) && vectors(a.q) && vectors(a.k);
    const int items = a.d / (2 * p.columns);
    p.lph = items <= 4 ? 4 : items <= 8 ? 8 : items <= 16 ? 16 : 32;
    const int ng = 32 / p.lph;
    const int64_t tokens = a.b * a.t;
    const int hg = back ? Ring<true>::HG : Ring<false>::HG, nw = back ? Ring<true>::WARPS : Ring<false>::WARPS;
    const int room = 148 * (back ? Ring<true>::BLOCKS : Ring<false>::BLOCKS);
    // Warps that the tensors have work for, and what it costs, in loads of `ng` heads: a stage about as much as one and a half for its waiting,
    // and where it is of several tokens, each turn of them one for their factors, and forward their loads more than half as much again.  (16384
    // tokens, loads counted alike | as here, us: 32 / 8 heads of 128 71.0 | 66.1, 8 / 1 of 256 41.7 | 32.5: the blocks of one tensor waited for the other's.)
    int64_t want_q, want_k;
    double cost_q, cost_k;
    auto ring = [&](RingPlan &r, const NormTensor &t, int64_t &want, double &cost) {
        // As many heads as a stage holds; where a token has at most half as many, several tokens.
        r.heads = std::min(t.heads, ng * hg);
        while (r.heads > ng && stage_bytes(back, r.heads, 1, a.d, a.dim, eb) > STAGE_MOST) r.heads -= ng;
        r.units = r.heads ? (t.heads + r.heads - 1) / r.heads : 0;
        r.tokens = r.units == 1 ? std::max(1, std::min(32, ng * hg / r.heads)) : 1;
        r.tokens = (int)std::min<int64_t>(r.tokens, std::max<int64_t>(1, tokens / (room * nw / 2)));   // (few tokens: rather more warps)
        while (r.tokens > 1 && stage_bytes(back, r.heads * r.tokens, r.tokens, a.d, a.dim, eb) > STAGE_MOST) --r.tokens;
        r.stage = stage_bytes(back, r.heads * r.tokens, r.tokens, a.d, a.dim, eb);
        for (r.slots = 1; 2 * r.slots <= std::min(ng, r.tokens);) r.slots *= 2;
        want = ((tokens + r.tokens - 1) / r.tokens * r.units + nw - 1) / nw;
        const int turns = (r.tokens + r.slots - 1) / r.slots, beside = ng / r.slots;
        cost = r.units * (turns * ((r.heads + beside - 1) / beside * (r.tokens == 1 || back ? 1. : 1.6) + (r.tokens == 1 ? 0. : 1.)) + 1.5) / r.tokens;
    };
    ring(p.ring_q, a.q, want_q, cost_q);
    ring(p.ring_k, a.k, want_k, cost_k);
    // The ring for the gradient, and forward in 16 bits where its warps get one and a half stages each or more: one alone is waited for (us, ring |
    // a warp for every token: bf16, 32 / 8 heads of 128, 1000 tokens 8.4 | 6.7, 16384 64 | 92; 16 / 4 of 128, 2500 8.9 | 8.4, 5000 14.0 | 16.5;
    // 8 / 1 of 64, 2500 6.5 | 5.9, 16384 15.7 | 25.9).  In f32 a byte has
    // half the instructions, and loads into registers keep up with HBM (16384 tokens of 32 / 8 heads of 128 130 | 118) unless heads leave lanes
    // idle and tokens are many (five stages a warp: 16 / 16 of 80, 5000 24.6 | 26.4, 16384 64.8 | 81.5; 32 / 8 of 96, 16384 85.6 | 108; below,
    // 16 / 4 of 80, 5000 19.4 | 16.6).
    const int64_t want = want_q + want_k;
    const bool staged = eb == 2 ? 2 * want >= 3 * room : items < p.lph && want >= 5 * room;
    p.way = !vec ? ELEMENTS : back || staged ? RING : HEADS;
    if (p.way == HEADS) {
        p.units_q = (a.q.heads + ng * HEADS_EACH - 1) / (ng * HEADS_EACH);
        p.units_k = (a.k.heads + ng * HEADS_EACH - 1) / (ng * HEADS_EACH);
        return p;
    }
    const int most = p.way == RING ? room : MAX_BLOCKS;
    if (p.way == ELEMENTS) {
        want_q = (tokens * a.q.heads + WARPS - 1) / WARPS;
        want_k = (tokens * a.k.heads + WARPS - 1) / WARPS;
        cost_q = a.q.heads;
        cost_k = a.k.heads;
    }
    int64_t bq = want_q, bk = want_k;
    if (bq + bk > most) {   // blocks that run until the tokens are done, the keys' share of them by what they cost
        bk = want_k == 0 ? 0 : want_q == 0 ? most : std::min<int64_t>(most - 1, std::max<int64_t>(1, (int64_t)(most * cost_k / (cost_q + cost_k) + 0.5)));
        bq = most - bk;
    }
    p.blocks_q = (int)bq;
    p.blocks = (int)(bq + bk);
    return p;
}

template <typename T, typename TW, int V, int LPH, bool BACK>
cudaError_t run_ring(const NormArgs &a, const Plan &p, cudaStream_t stream) {
    using R = Ring<BACK>;
    const auto kernel = qk_norm_ring_kernel<T, TW, V, LPH, BACK>;
    const int bytes = 128 + std::max(R::WARPS * R::STAGES * std::max(p.ring_q.stage, p.ring_k.stage), BACK ? R::WARPS * a.d * 4 : 0);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 + R::WARPS * R::STAGES * STAGE_MOST);
    if (e != cudaSuccess) return e;
    kernel<<<p.blocks, R::WARPS * 32, bytes, stream>>>(a, p.ring_q, p.ring_k, p.blocks_q);
    return cudaGetLastError();
}

template <typename T, typename TW, int V, int LPH>
cudaError_t run_vec(const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    if (p.way == RING) return back ? run_ring<T, TW, V, LPH, true>(a, p, stream) : run_ring<T, TW, V, LPH, false>(a, p, stream);
    const int64_t blocks = (a.b * a.t * (p.units_q + p.units_k) + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    qk_norm_kernel<T, TW, V, LPH, HEADS_EACH><<<(unsigned)blocks, THREADS, 0, stream>>>(a, p.units_q, p.units_q + p.units_k, over_of(p.units_q + p.units_k));
    return cudaGetLastError();
}

template <typename T, typename TW, int V>
cudaError_t run_columns(const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    switch (p.lph) {
        case 4: return run_vec<T, TW, V, 4>(a, p, back, stream);
        case 8: return run_vec<T, TW, V, 8>(a, p, back, stream);
        case 16: return run_vec<T, TW, V, 16>(a, p, back, stream);
        default: return run_vec<T, TW, V, 32>(a, p, back, stream);
    }
}

template <typename T, typename TW>
cudaError_t run_t(const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (p.way == ELEMENTS) {
        if (back) qk_norm_elements_kernel<T, true><<<p.blocks, THREADS, sizeof(float) * WARPS * a.d, stream>>>(a, p.blocks_q);
        else qk_norm_elements_kernel<T, false><<<p.blocks, THREADS, 0, stream>>>(a, p.blocks_q);
        return cudaGetLastError();
    }
    if constexpr (sizeof(T) == 2)
        if (p.columns < V) return run_columns<T, TW, V / 2>(a, p, back, stream);
    return run_columns<T, TW, V>(a, p, back, stream);
}

cudaError_t run(int dtype, const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    switch (dtype) {
        case 0: return run_t<float, float>(a, p, back, stream);
        case 1: return a.w_f32 ? run_t<__nv_bfloat16, float>(a, p, back, stream) : run_t<__nv_bfloat16, __nv_bfloat16>(a, p, back, stream);
        default: return a.w_f32 ? run_t<__half, float>(a, p, back, stream) : run_t<__half, __half>(a, p, back, stream);
    }
}

bool nothing(const NormArgs &a) { return a.b * a.t == 0 || a.q.heads + a.k.heads == 0 || a.d == 0; }

// Where a token's position does not go by its batch element, and every tensor's batch elements follow one another, they are one.
NormArgs prepared(NormArgs a) {
    auto one = [&](const NormTensor &t) { return t.heads == 0 || (t.sb == a.t * t.st && (!t.g || t.gb == a.t * t.gt)); };
    if (a.b > 1 && (a.positions || a.cu) && one(a.q) && one(a.k)) {
        a.t *= a.b;
        a.b = 1;
    }
    if (a.t < (int64_t(1) << 31)) a.over_t = over_of(a.t);
    return a;
}

}  // namespace

// As many rows as the larger of the two ways needs: which one runs depends on addresses, which a workspace query does not have.
size_t qk_norm_part_floats(int d) { return (size_t)MAX_BLOCKS * d; }

cudaError_t launch_qk_norm(int dtype, const NormArgs &given, cudaStream_t stream, int *launches) {
    if (nothing(given)) return cudaSuccess;
    const NormArgs a = prepared(given);
    *launches += 1;
    return run(dtype, a, plan_of(dtype, a, false), false, stream);
}

cudaError_t launch_qk_norm_backward(int dtype, const NormArgs &given, cudaStream_t stream, int *launches) {
    if (nothing(given)) return cudaSuccess;
    const NormArgs a = prepared(given);
    const Plan p = plan_of(dtype, a, true);
    *launches += 1;
    cudaError_t e = run(dtype, a, p, true, stream);
    if (e != cudaSuccess || (!a.q.dw && !a.k.dw)) return e;
    *launches += 1;
    const dim3 grid((unsigned)((a.d + 31) / 32), 2);
    if (dtype == 0 || a.w_f32) return launch_beside(qk_norm_sum_kernel<float>, grid, SUM_WARPS * 32, 0, stream, true, a, p.blocks_q, p.blocks);
    if (dtype == 1) return launch_beside(qk_norm_sum_kernel<__nv_bfloat16>, grid, SUM_WARPS * 32, 0, stream, true, a, p.blocks_q, p.blocks);
    return launch_beside(qk_norm_sum_kernel<__half>, grid, SUM_WARPS * 32, 0, stream, true, a, p.blocks_q, p.blocks);
}

cudaError_t read_qk_norm_status(unsigned int *status, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_qk_norm_status, sizeof(unsigned int));
    if (e != cudaSuccess) return e;
    if (clear && *status) {
        unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_qk_norm_status, &zero, sizeof(unsigned int));
    }
    return e;
}

}  // namespace dash
