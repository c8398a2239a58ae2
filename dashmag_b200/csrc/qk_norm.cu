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

namespace dash {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ int64_t index_at(const void *p, int bytes, int64_t i) {
    return bytes == 8 ? static_cast<const int64_t *>(p)[i] : static_cast<int64_t>(static_cast<const int32_t *>(p)[i]);
}

// n = (batch element, token of it), in 32 bits where both fit.
__device__ __forceinline__ void token_of(const NormArgs &a, int64_t n, int64_t &bi, int64_t &ti) {
    if (((n | a.t) >> 32) == 0) {
        bi = (uint32_t)n / (uint32_t)a.t;
        ti = (uint32_t)n - (uint32_t)bi * (uint32_t)a.t;
    } else {
        bi = n / a.t;
        ti = n - bi * a.t;
    }
}

// The position of token n = (.., ti): its row of the tables; -1 for one outside them, -2 for a token of no sequence.
__device__ __forceinline__ int64_t table_row(const NormArgs &a, int64_t n, int64_t ti) {
    int64_t pos;
    if (a.positions) {
        pos = index_at(a.positions, a.pos_bytes, n);
    } else if (a.cu) {
        if (a.sequences <= 0 || n < index_at(a.cu, a.cu_bytes, 0) || n >= index_at(a.cu, a.cu_bytes, a.sequences)) return -2;
        int lo = 0, hi = a.sequences;   // the last sequence whose offset is <= n
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (index_at(a.cu, a.cu_bytes, mid) <= n) lo = mid; else hi = mid;
        }
        pos = a.start + n - index_at(a.cu, a.cu_bytes, lo);
    } else {
        pos = a.start + ti;
    }
    return pos >= 0 && pos < a.len ? pos : -1;
}

// V elements of T as they lie in memory, 16 bytes (weights in f32 beside 16-bit tensors: 32).
template <typename T, int V> struct alignas(16) Vec { T e[V]; };
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load(const T *p) {
    Vec<T, V> v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4 *>(&v)[i] = reinterpret_cast<const uint4 *>(p)[i];
    return v;
}
template <typename T, int V> __device__ __forceinline__ void store(T *p, const Vec<T, V> &v) {
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&v);
}
template <typename T, int V> __device__ __forceinline__ void widen(const Vec<T, V> &v, float (&x)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = Num<T>::to_f32(v.e[e]);
}
template <typename T, int V> __device__ __forceinline__ Vec<T, V> narrow(const float (&x)[V]) {
    Vec<T, V> v;
#pragma unroll
    for (int e = 0; e < V; ++e) v.e[e] = Num<T>::from_f32(x[e]);
    return v;
}
template <typename TW, int V> __device__ __forceinline__ void weights(const void *w, int col, bool live, float (&x)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = 1.f;
    if (w && live) widen<TW, V>(load<TW, V>(static_cast<const TW *>(w) + col), x);
}
template <int LPH> __device__ __forceinline__ float head_sum(float x) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }

// Cosines and sines of a lane's two columns: the token's row, NaN for a position outside the tables (nothing is read there), and no
// rotation for columns behind the rotated ones.
template <typename T, int V> struct Turn {
    float c1[V], c2[V], s1[V], s2[V];
    __device__ __forceinline__ Turn(const NormArgs &a, int64_t row, bool rotated, int c, int half) {
        const float none = rotated ? nan_f32() : 1.f, off = rotated ? none : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) { c1[e] = c2[e] = none; s1[e] = s2[e] = off; }
        if (rotated && row >= 0) {
            const T *cs = static_cast<const T *>(a.cos) + row * a.dim + c, *sn = static_cast<const T *>(a.sin) + row * a.dim + c;
            widen<T, V>(load<T, V>(cs), c1);
            widen<T, V>(load<T, V>(cs + half), c2);
            widen<T, V>(load<T, V>(sn), s1);
            widen<T, V>(load<T, V>(sn + half), s2);
        }
    }
};

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

template <typename T, typename TW, int V, int LPH, int HG>
__global__ void __launch_bounds__(THREADS) qk_norm_kernel(NormArgs a, int units_q, int units_k) {
    constexpr int NG = 32 / LPH;   // heads of a warp's load
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int units = units_q + units_k;
    const int64_t n = (warp >> 31) == 0 ? (int64_t)((uint32_t)warp / (uint32_t)units) : warp / units;
    if (n >= a.b * a.t) return;
    const int unit = (int)(warp - n * units);
    const bool is_k = unit >= units_q;
    const NormTensor &t = is_k ? a.k : a.q;
    const int h0 = (is_k ? unit - units_q : unit) * NG * HG + lane / LPH;
    const Place<V, LPH> at(a, lane);
    int64_t bi, ti;
    token_of(a, n, bi, ti);
    const T *x = static_cast<const T *>(t.x) + bi * t.sb + ti * t.st;
    T *out = static_cast<T *>(t.out) + n * t.heads * a.d;
    Vec<T, V> x1[HG], x2[HG];
#pragma unroll
    for (int g = 0; g < HG; ++g) {
        const int h = min(h0 + g * NG, t.heads - 1);
        if (at.live) {
            x1[g] = load<T, V>(x + h * t.sh + at.c1);
            x2[g] = load<T, V>(x + h * t.sh + at.c2);
        }
    }
    float w1[V], w2[V];
    weights<TW, V>(t.w, at.c1, at.live, w1);
    weights<TW, V>(t.w, at.c2, at.live, w2);
    const int64_t row = table_row(a, n, ti);
    const Turn<T, V> turn(a, row, at.live && at.rotated, at.c1, a.dim / 2);
#pragma unroll
    for (int g = 0; g < HG; ++g) {
        const int h = h0 + g * NG;
        float u1[V], u2[V], sum = 0.f;
        if (at.live) {
            widen<T, V>(x1[g], u1);
            widen<T, V>(x2[g], u2);
#pragma unroll
            for (int e = 0; e < V; ++e) sum = fmaf(u1[e], u1[e], fmaf(u2[e], u2[e], sum));
        }
        const float r = rsqrtf(head_sum<LPH>(sum) / a.d + a.eps);
        if (!at.live || h >= t.heads) continue;
        Vec<T, V> y1 = x1[g], y2 = x2[g];
        if (row != -2) {   // (a token of no sequence passes unchanged)
            float z1[V], z2[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float n1 = u1[e] * r * w1[e], n2 = u2[e] * r * w2[e];
                z1[e] = n1 * turn.c1[e] - n2 * turn.s1[e];
                z2[e] = n2 * turn.c2[e] + n1 * turn.s2[e];
            }
            y1 = narrow<T, V>(z1);
            y2 = narrow<T, V>(z2);
        }
        store<T, V>(out + h * a.d + at.c1, y1);
        store<T, V>(out + h * a.d + at.c2, y2);
    }
}

// A block's sums of the weight's gradient, from its warps' lanes, into its row of the scratch.
template <int V, int LPH>
__device__ __forceinline__ void leave_part(const NormArgs &a, const Place<V, LPH> &at, float (&d1)[V], float (&d2)[V], float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int o = LPH; o < 32; o <<= 1) {
            d1[e] += __shfl_xor_sync(0xffffffffu, d1[e], o);
            d2[e] += __shfl_xor_sync(0xffffffffu, d2[e], o);
        }
        if (lane < LPH && at.live) {
            red[warp * a.d + at.c1 + e] = d1[e];
            red[warp * a.d + at.c2 + e] = d2[e];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) sum += red[i * a.d + c];
        a.part[(int64_t)blockIdx.x * a.d + c] = sum;
    }
}

// The blocks up to blocks_q take the queries' units in turn, the others the keys', so that a lane's sums of the weight's gradient
// are one tensor's and stay in registers to the end.
template <typename T, typename TW, int V, int LPH, int HG>
__global__ void __launch_bounds__(THREADS) qk_norm_backward_kernel(NormArgs a, int units_q, int units_k, int blocks_q) {
    constexpr int NG = 32 / LPH;
    extern __shared__ float red[];   // [WARPS][d]
    allow_beside();   // the sums over the blocks
    const int lane = threadIdx.x & 31;
    const bool is_k = (int)blockIdx.x >= blocks_q;
    const NormTensor &t = is_k ? a.k : a.q;
    const int units = is_k ? units_k : units_q;
    const int64_t first = (int64_t)(is_k ? blockIdx.x - blocks_q : blockIdx.x) * WARPS + (threadIdx.x >> 5);
    const int64_t step = (int64_t)(is_k ? gridDim.x - blocks_q : blocks_q) * WARPS, all = a.b * a.t * units;
    const Place<V, LPH> at(a, lane);
    float w1[V], w2[V], d1[V], d2[V];
    weights<TW, V>(t.w, at.c1, at.live, w1);
    weights<TW, V>(t.w, at.c2, at.live, w2);
#pragma unroll
    for (int e = 0; e < V; ++e) d1[e] = d2[e] = 0.f;
    for (int64_t item = first; item < all; item += step) {
        const int64_t n = (item >> 31) == 0 ? (int64_t)((uint32_t)item / (uint32_t)units) : item / units;
        const int h0 = (int)(item - n * units) * NG * HG + lane / LPH;
        int64_t bi, ti;
        token_of(a, n, bi, ti);
        const T *x = static_cast<const T *>(t.x) + bi * t.sb + ti * t.st, *dy = static_cast<const T *>(t.g) + bi * t.gb + ti * t.gt;
        T *out = static_cast<T *>(t.out) + n * t.heads * a.d;
        Vec<T, V> x1[HG], x2[HG], y1[HG], y2[HG];
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            const int h = min(h0 + g * NG, t.heads - 1);
            if (at.live) {
                x1[g] = load<T, V>(x + h * t.sh + at.c1);
                x2[g] = load<T, V>(x + h * t.sh + at.c2);
                y1[g] = load<T, V>(dy + h * t.gh + at.c1);
                y2[g] = load<T, V>(dy + h * t.gh + at.c2);
            }
        }
        const int64_t row = table_row(a, n, ti);
        const Turn<T, V> turn(a, row, at.live && at.rotated, at.c1, a.dim / 2);
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            const int h = h0 + g * NG;
            float u1[V], u2[V], g1[V], g2[V], square = 0.f, along = 0.f;
            if (at.live) {
                float v1[V], v2[V];
                widen<T, V>(x1[g], u1);
                widen<T, V>(x2[g], u2);
                widen<T, V>(y1[g], v1);
                widen<T, V>(y2[g], v2);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    g1[e] = v1[e] * turn.c1[e] + v2[e] * turn.s2[e];
                    g2[e] = v2[e] * turn.c2[e] - v1[e] * turn.s1[e];
                    square = fmaf(u1[e], u1[e], fmaf(u2[e], u2[e], square));
                    along = fmaf(u1[e] * w1[e], g1[e], fmaf(u2[e] * w2[e], g2[e], along));
                }
            }
            const float r = rsqrtf(head_sum<LPH>(square) / a.d + a.eps);
            const float back = head_sum<LPH>(along) / a.d * r * r * r;
            if (!at.live || h >= t.heads) continue;
            Vec<T, V> z1 = y1[g], z2 = y2[g];
            if (row != -2) {
                float e1[V], e2[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    e1[e] = r * w1[e] * g1[e] - u1[e] * back;
                    e2[e] = r * w2[e] * g2[e] - u2[e] * back;
                    d1[e] = fmaf(g1[e], u1[e] * r, d1[e]);
                    d2[e] = fmaf(g2[e], u2[e] * r, d2[e]);
                }
                z1 = narrow<T, V>(e1);
                z2 = narrow<T, V>(e2);
            }
            store<T, V>(out + h * a.d + at.c1, z1);
            store<T, V>(out + h * a.d + at.c2, z2);
        }
    }
    leave_part<V, LPH>(a, at, d1, d2, red);
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
    for (int64_t item = first; item < all; item += step) {
        const int64_t n = item / t.heads;
        const int h = (int)(item - n * t.heads);
        int64_t bi, ti;
        token_of(a, n, bi, ti);
        const int64_t xo = bi * t.sb + ti * t.st + h * t.sh, go = bi * t.gb + ti * t.gt + h * t.gh, oo = item * a.d;
        const int64_t row = table_row(a, n, ti);
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

// The weight's gradient from the blocks' rows, in their order: a block 32 columns of one tensor.
template <typename TW>
__global__ void __launch_bounds__(THREADS) qk_norm_sum_kernel(NormArgs a, int blocks_q, int blocks) {
    __shared__ float red[WARPS][32];
    wait_before();
    const bool is_k = blockIdx.y == 1;
    const NormTensor &t = is_k ? a.k : a.q;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const int b0 = is_k ? blocks_q : 0, b1 = is_k ? blocks : blocks_q;
    float sum = 0.f;
    if (t.dw && c < a.d) {
#pragma unroll 8
        for (int i = b0 + warp; i < b1; i += WARPS) sum += a.part[(int64_t)i * a.d + c];
    }
    red[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || !t.dw || c >= a.d) return;
    for (int i = 1; i < WARPS; ++i) sum += red[i][lane];
    static_cast<TW *>(t.dw)[c] = Num<TW>::from_f32(sum);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
struct Plan {
    bool vec;
    int lph;                 // lanes of a head
    int units_q, units_k;    // warps of a token
    int blocks_q, blocks;    // backward, and the element kernels
};

constexpr int HEADS_EACH = 2;   // heads of a lane
constexpr int MAX_BLOCKS = 148 * 8;

Plan plan_of(int dtype, const NormArgs &a, bool back) {
    const int eb = dtype == 0 ? 4 : 2, v = 16 / eb;
    auto aligned = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    auto ok = [&](const NormTensor &t) {
        return t.heads == 0 || (aligned(t.x) && aligned(t.out) && t.sb % v == 0 && t.st % v == 0 && t.sh % v == 0 && aligned(t.w) &&
                                (!back || (aligned(t.g) && t.gb % v == 0 && t.gt % v == 0 && t.gh % v == 0)));
    };
    Plan p{};
    p.vec = a.dim % (2 * v) == 0 && a.d % (2 * v) == 0 && aligned(a.cos) && aligned(a.sin) && ok(a.q) && ok(a.k);
    const int items = a.d / (2 * v);
    p.lph = items <= 4 ? 4 : items <= 8 ? 8 : items <= 16 ? 16 : 32;
    const int per = 32 / p.lph * HEADS_EACH;
    p.units_q = (a.q.heads + per - 1) / per;
    p.units_k = (a.k.heads + per - 1) / per;
    // Blocks that run until the tokens are done: eight a multiprocessor, the keys' share of them by their units.
    const int64_t tokens = a.b * a.t, uq = p.vec ? p.units_q : a.q.heads, uk = p.vec ? p.units_k : a.k.heads;
    const int64_t want_q = (tokens * uq + WARPS - 1) / WARPS, want_k = (tokens * uk + WARPS - 1) / WARPS, room = MAX_BLOCKS;
    int64_t bq = want_q, bk = want_k;
    if (bq + bk > room) {
        bk = want_k == 0 ? 0 : std::max<int64_t>(1, room * uk / (uq + uk));
        bq = want_q == 0 ? 0 : room - bk;
    }
    p.blocks_q = (int)bq;
    p.blocks = (int)(bq + bk);
    return p;
}

template <typename T, typename TW, int V, int LPH>
cudaError_t run_vec(const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    if (back) {
        qk_norm_backward_kernel<T, TW, V, LPH, HEADS_EACH>
            <<<p.blocks, THREADS, sizeof(float) * WARPS * a.d, stream>>>(a, p.units_q, p.units_k, p.blocks_q);
    } else {
        const int64_t blocks = (a.b * a.t * (p.units_q + p.units_k) + WARPS - 1) / WARPS;
        if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
        qk_norm_kernel<T, TW, V, LPH, HEADS_EACH><<<(unsigned)blocks, THREADS, 0, stream>>>(a, p.units_q, p.units_k);
    }
    return cudaGetLastError();
}

template <typename T, typename TW>
cudaError_t run_t(const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (!p.vec) {
        if (back) qk_norm_elements_kernel<T, true><<<p.blocks, THREADS, sizeof(float) * WARPS * a.d, stream>>>(a, p.blocks_q);
        else qk_norm_elements_kernel<T, false><<<p.blocks, THREADS, 0, stream>>>(a, p.blocks_q);
        return cudaGetLastError();
    }
    switch (p.lph) {
        case 4: return run_vec<T, TW, V, 4>(a, p, back, stream);
        case 8: return run_vec<T, TW, V, 8>(a, p, back, stream);
        case 16: return run_vec<T, TW, V, 16>(a, p, back, stream);
        default: return run_vec<T, TW, V, 32>(a, p, back, stream);
    }
}

cudaError_t run(int dtype, const NormArgs &a, const Plan &p, bool back, cudaStream_t stream) {
    switch (dtype) {
        case 0: return run_t<float, float>(a, p, back, stream);
        case 1: return a.w_f32 ? run_t<__nv_bfloat16, float>(a, p, back, stream) : run_t<__nv_bfloat16, __nv_bfloat16>(a, p, back, stream);
        default: return a.w_f32 ? run_t<__half, float>(a, p, back, stream) : run_t<__half, __half>(a, p, back, stream);
    }
}

bool nothing(const NormArgs &a) { return a.b * a.t == 0 || a.q.heads + a.k.heads == 0 || a.d == 0; }

}  // namespace

// As many rows as the larger of the two ways needs: which one runs depends on addresses, which a workspace query does not have.
size_t qk_norm_part_floats(int d) { return (size_t)MAX_BLOCKS * d; }

cudaError_t launch_qk_norm(int dtype, const NormArgs &a, cudaStream_t stream, int *launches) {
    if (nothing(a)) return cudaSuccess;
    *launches += 1;
    return run(dtype, a, plan_of(dtype, a, false), false, stream);
}

cudaError_t launch_qk_norm_backward(int dtype, const NormArgs &a, cudaStream_t stream, int *launches) {
    if (nothing(a)) return cudaSuccess;
    const Plan p = plan_of(dtype, a, true);
    *launches += 1;
    cudaError_t e = run(dtype, a, p, true, stream);
    if (e != cudaSuccess || (!a.q.dw && !a.k.dw)) return e;
    *launches += 1;
    const dim3 grid((unsigned)((a.d + 31) / 32), a.k.heads > 0 ? 2 : 1);
    if (dtype == 0 || a.w_f32) return launch_beside(qk_norm_sum_kernel<float>, grid, THREADS, 0, stream, true, a, p.blocks_q, p.blocks);
    if (dtype == 1) return launch_beside(qk_norm_sum_kernel<__nv_bfloat16>, grid, THREADS, 0, stream, true, a, p.blocks_q, p.blocks);
    return launch_beside(qk_norm_sum_kernel<__half>, grid, THREADS, 0, stream, true, a, p.blocks_q, p.blocks);
}

}  // namespace dash
