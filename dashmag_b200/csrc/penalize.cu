// The rules a server puts on a step's logits, in one pass over them: with seen[v] whether token v is anywhere in the row's history and
// count[v] how often it is in what the model has answered (the ids behind the prompt's),
//
//     z = seen ? (z > 0 ? z / repetition : z repetition) : z,   z = z - frequency count - presence [count > 0] + bias,
//     z = -inf where the grammar does not allow v,
//
// in f32 and rounded once to the logits' dtype.
//
// A block takes a piece of one row's vocabulary and keeps a word per token of it in shared memory: the count, and the top bit for a
// token of the prompt.  It reads the row's history, counts the ids that fall into its piece (integer additions, whose order does not
// matter), and then makes the pass over its logits, which were asked for before the history.  Nothing is sorted and no
// scratch is needed.  What a block waits for is one trip to memory: its logits, the grammar's words, the row's numbers and the first ids are
// all asked for before any is looked at, the ids before it is known how many are the row's.  (One after another, four trips: 251 rows of
// 38531 tokens with a grammar and next to no history 19.8 us, now XX.)  The pieces cost the history read once for each, from L2;
// clusters of eight blocks that read a share each and count for one another in distributed shared memory were slower (256 rows of
// 100003, 8192 ids, 107 us against 68: half of a text's ids are a few tokens, whose words all eight blocks then wait for).
// The pass itself is a read and a write of the logits, bound by HBM.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "penalize.h"

namespace dash {
namespace {

constexpr int THREADS = 256;
#ifndef MINB
#define MINB 3
#define MAXE 4
#endif
constexpr unsigned IN_PROMPT = 0x80000000u;

template <typename T, int V> struct alignas(16) Vec { T e[V]; };

// What a row's tokens go through.
struct Rules {
    float repetition, frequency, presence;
    const uint32_t *allowed;
};

// One token's logit: `word` its count and mark, `bias` and `open` the grammar's bit where there are any.
__device__ __forceinline__ float ruled(const Rules &r, float z, unsigned word, float bias, bool open) {
    if (word) {
        z = z > 0.f ? z / r.repetition : z * r.repetition;
        const unsigned count = word & ~IN_PROMPT;
        if (count) z = z - r.frequency * (float)count - r.presence;
    }
    z += bias;
    return open ? z : -INFINITY;
}

// Index i of an array of i32 / i64 as it stands there; `none` where there is no array.
__device__ __forceinline__ int64_t number(const void *p, int bytes, int i, int none) {
    return !p ? none : bytes == 8 ? static_cast<const int64_t *>(p)[i] : static_cast<int64_t>(static_cast<const int32_t *>(p)[i]);
}
__device__ __forceinline__ int within(int64_t x, int top) { return (int)min(max(x, (int64_t)0), (int64_t)top); }

constexpr int AHEAD = 8;   // ids of a thread on their way at once

// EACH vectors a thread: a piece of THREADS * EACH * V tokens.  I: the ids' integers.
template <typename T, typename I, int EACH>
__global__ void __launch_bounds__(THREADS, MINB) penalize_kernel(PenalizeArgs a, int pieces) {
    constexpr int V = 16 / sizeof(T), PIECE = THREADS * EACH * V;
    __shared__ alignas(16) unsigned words[PIECE];
    const int row = blockIdx.x / pieces, piece = blockIdx.x - row * pieces;
    const T *in = static_cast<const T *>(a.logits) + (int64_t)row * a.stride;
    T *out = static_cast<T *>(a.out) + (int64_t)row * a.out_stride;
    // Places are counted from the 16-byte boundary at or before the row, so that whole vectors are aligned whatever the row's address.
    const int skew = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    const bool vec = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int first = piece * PIECE - skew;   // the token of the piece's first place (negative: there is none)
    if (first >= a.v) return;

    const I *ids = static_cast<const I *>(a.ids) + (int64_t)row * a.ids_stride;
    I id[AHEAD];
    int64_t length = 0, prompt_length = 0;
    auto ask = [&](int i0, int end) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) id[e] = i0 + e * THREADS < end ? ids[i0 + e * THREADS] : I(-1);
    };
    if (a.ids) {
        length = number(a.lengths, a.lengths_bytes, row, a.t);
        prompt_length = number(a.prompt, a.prompt_bytes, row, 0);
        ask(threadIdx.x, a.t);
    }
    Rules r;
    r.repetition = a.repetition ? a.repetition[row] : a.repetition_all;
    r.frequency = a.frequency ? a.frequency[row] : a.frequency_all;
    r.presence = a.presence ? a.presence[row] : a.presence_all;
    r.allowed = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride : nullptr;
    Vec<T, V> x[EACH];
    uint32_t open[EACH], open2[EACH];   // the words a whole vector's V bits lie in
    auto token = [&](int j) { return first + (j * THREADS + (int)threadIdx.x) * V; };
    auto whole = [&](int v0) { return vec && v0 >= 0 && v0 <= a.v - V; };
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int v0 = token(j);
        if (whole(v0)) {
            *reinterpret_cast<uint4 *>(&x[j]) = *reinterpret_cast<const uint4 *>(in + v0);
            if (r.allowed) {
                open[j] = r.allowed[v0 >> 5];
                open2[j] = skew ? r.allowed[(v0 + V - 1) >> 5] : 0;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (v0 + e >= 0 && v0 + e < a.v) x[j].e[e] = in[v0 + e];
        }
    }
    if (a.ids) {
        for (int i = threadIdx.x; i < PIECE / 4; i += THREADS) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int len = within(length, a.t), prompt = within(prompt_length, len);
        for (int i0 = threadIdx.x; i0 < len; i0 += THREADS * AHEAD) {
            if (i0 >= THREADS * AHEAD) ask(i0, len);
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                // (Ids outside the vocabulary, padding's -1 among them, count for nothing; another piece's come out past this one's places.)
                const unsigned at = (unsigned)((int)id[e] - first);
                const int i = i0 + e * THREADS;
                if ((std::make_unsigned_t<I>)id[e] >= (std::make_unsigned_t<I>)a.v || at >= (unsigned)PIECE || i >= len) continue;
                if (i < prompt) atomicOr(&words[at], IN_PROMPT);
                else atomicAdd(&words[at], 1u);
            }
        }
        __syncthreads();
    }

    const int64_t bias0 = (int64_t)row * a.bias_stride;
    auto bias_at = [&](int v) {
        return a.bias_f32 ? static_cast<const float *>(a.bias)[bias0 + v] : Num<T>::to_f32(static_cast<const T *>(a.bias)[bias0 + v]);
    };
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int v0 = token(j);
        if (v0 >= a.v || v0 + V <= 0) continue;
        unsigned w[V], any = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = 0;
        if (a.ids) {
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<uint4 *>(&w[e]) = reinterpret_cast<const uint4 *>(words)[((j * THREADS + threadIdx.x) * V + e) / 4];
#pragma unroll
            for (int e = 0; e < V; ++e) any |= w[e];
        }
        if (!whole(v0)) {   // the row's ends
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int v = v0 + e;
                if (v >= 0 && v < a.v)
                    out[v] = Num<T>::from_f32(ruled(r, Num<T>::to_f32(x[j].e[e]), w[e], a.bias ? bias_at(v) : 0.f, !r.allowed || (r.allowed[v >> 5] >> (v & 31) & 1u)));
            }
            continue;
        }
        float z[V];
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = Num<T>::to_f32(x[j].e[e]);
        if (any) {
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = ruled(r, z[e], w[e], 0.f, true);
        }
        if (a.bias) {
            const bool four = a.bias_f32 && (reinterpret_cast<uintptr_t>(static_cast<const float *>(a.bias) + bias0 + v0) & 15) == 0;
            if (four) {
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.bias) + bias0 + v0 + e);
                    z[e] += b.x; z[e + 1] += b.y; z[e + 2] += b.z; z[e + 3] += b.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] += bias_at(v0 + e);
            }
        }
        if (r.allowed) {
            const uint32_t bits = __funnelshift_r(open[j], open2[j], v0 & 31);
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = bits >> e & 1u ? z[e] : -INFINITY;
        }
        Vec<T, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e) y.e[e] = Num<T>::from_f32(z[e]);
        *reinterpret_cast<uint4 *>(out + v0) = *reinterpret_cast<const uint4 *>(&y);
    }
}

template <typename T, int EACH>
cudaError_t run(const PenalizeArgs &a, int pieces, cudaStream_t stream) {
    const int64_t blocks = (int64_t)pieces * a.b;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (a.ids_bytes == 8) penalize_kernel<T, int64_t, EACH><<<(unsigned)blocks, THREADS, 0, stream>>>(a, pieces);
    else penalize_kernel<T, int32_t, EACH><<<(unsigned)blocks, THREADS, 0, stream>>>(a, pieces);
    return cudaGetLastError();
}

template <typename T>
cudaError_t penalize_t(const PenalizeArgs &a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    auto pieces = [&](int each) { return (int)(((int64_t)a.v + V - 1 + THREADS * each * V - 1) / (THREADS * each * V)); };
    // The largest piece (the history is read once per piece) that still leaves four blocks to a multiprocessor.
    int each = MAXE;
    while (each > 1 && (int64_t)pieces(each) * a.b < 148 * 4) each /= 2;
    return each == 4 ? run<T, 4>(a, pieces(4), stream) : each == 2 ? run<T, 2>(a, pieces(2), stream) : run<T, 1>(a, pieces(1), stream);
}

}  // namespace

cudaError_t launch_penalize(int dtype, const PenalizeArgs &a, cudaStream_t stream, int *launches) {
    if (a.b == 0 || a.v == 0) return cudaSuccess;
    *launches += 1;
    switch (dtype) {
        case 0: return penalize_t<float>(a, stream);
        case 1: return penalize_t<__nv_bfloat16>(a, stream);
        default: return penalize_t<__half>(a, stream);
    }
}

}  // namespace dash
