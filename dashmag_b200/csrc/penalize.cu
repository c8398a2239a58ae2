// The rules a server puts on a step's logits, in one pass over them: with seen[v] whether token v is anywhere in the row's history and
// count[v] how often it is in what the model has answered (the ids behind the prompt's),
//
//     z = seen ? (z > 0 ? z / repetition : z repetition) : z,   z = z - frequency count - presence [count > 0] + bias,
//     z = -inf where the grammar does not allow v,
//
// in f32 and rounded once to the logits' dtype.
//
// A block takes a piece of one row's vocabulary and keeps a word per token of it in shared memory: the count, and the top bit for a
// token of the prompt.  It reads the row's whole history, counts the ids that fall into its piece (integer additions, whose order does not
// matter), and then makes the pass over its logits, which were asked for before the history.  Nothing is sorted and no
// scratch is needed; what the pieces cost is the history read once per piece, from L2.  The pass itself is a read and a write of the
// logits, bound by HBM.
#include <algorithm>

#include "common.cuh"
#include "penalize.h"

namespace dash {
namespace {

constexpr int THREADS = 256;
constexpr unsigned IN_PROMPT = 0x80000000u;

// Index i of an array of i32 / i64, as far as an int holds it.
__device__ __forceinline__ int held(const void *p, int bytes, int i, int none, int top) {
    return p ? min(max(load_index(p, bytes, i), 0), top) : none;
}

template <typename T, int V> struct alignas(16) Vec { T e[V]; };

// EACH vectors a thread: a piece of THREADS * EACH * V tokens.
template <typename T, int EACH>
__global__ void __launch_bounds__(THREADS) penalize_kernel(PenalizeArgs a, int pieces) {
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

    Vec<T, V> x[EACH];
    auto token = [&](int j) { return first + (j * THREADS + (int)threadIdx.x) * V; };
    auto whole = [&](int v0) { return vec && v0 >= 0 && v0 <= a.v - V; };
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int v0 = token(j);
        if (whole(v0)) {
            *reinterpret_cast<uint4 *>(&x[j]) = *reinterpret_cast<const uint4 *>(in + v0);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (v0 + e >= 0 && v0 + e < a.v) x[j].e[e] = in[v0 + e];
        }
    }

    const int len = a.ids ? held(a.lengths, a.lengths_bytes, row, a.t, a.t) : 0;
    if (len > 0) {
        const int prompt = held(a.prompt, a.prompt_bytes, row, 0, len);
        for (int i = threadIdx.x; i < PIECE / 4; i += THREADS) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto take = [&](int64_t id, int i) {
            const int64_t at = id - first;   // (ids outside the vocabulary, padding's -1 among them, count for nothing)
            if (id < 0 || id >= a.v || at < 0 || at >= PIECE) return;
            if (i < prompt) atomicOr(&words[at], IN_PROMPT);
            else atomicAdd(&words[at], 1u);
        };
        if (a.ids_bytes == 4) {
            const int32_t *ids = static_cast<const int32_t *>(a.ids) + (int64_t)row * a.ids_stride;
#pragma unroll 4
            for (int i = threadIdx.x; i < len; i += THREADS) take(ids[i], i);
        } else {
            const int64_t *ids = static_cast<const int64_t *>(a.ids) + (int64_t)row * a.ids_stride;
#pragma unroll 4
            for (int i = threadIdx.x; i < len; i += THREADS) take(ids[i], i);
        }
        __syncthreads();
    }

    const float repetition = a.repetition ? a.repetition[row] : a.repetition_all;
    const float frequency = a.frequency ? a.frequency[row] : a.frequency_all;
    const float presence = a.presence ? a.presence[row] : a.presence_all;
    const uint32_t *allowed = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride : nullptr;
    const int64_t bias0 = (int64_t)row * a.bias_stride;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int v0 = token(j);
        if (v0 >= a.v || v0 + V <= 0) continue;
        unsigned w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = 0;
        if (len > 0) {
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<uint4 *>(&w[e]) = reinterpret_cast<const uint4 *>(words)[((j * THREADS + threadIdx.x) * V + e) / 4];
        }
        Vec<T, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int v = v0 + e;
            if (v < 0 || v >= a.v) continue;
            float z = Num<T>::to_f32(x[j].e[e]);
            if (w[e]) {
                z = z > 0.f ? z / repetition : z * repetition;
                const unsigned count = w[e] & ~IN_PROMPT;
                if (count) z = z - frequency * (float)count - presence;
            }
            if (a.bias) z += a.bias_f32 ? static_cast<const float *>(a.bias)[bias0 + v] : Num<T>::to_f32(static_cast<const T *>(a.bias)[bias0 + v]);
            if (allowed && !(allowed[v >> 5] >> (v & 31) & 1u)) z = -INFINITY;
            y.e[e] = Num<T>::from_f32(z);
        }
        if (whole(v0)) {
            *reinterpret_cast<uint4 *>(out + v0) = *reinterpret_cast<const uint4 *>(&y);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (v0 + e >= 0 && v0 + e < a.v) out[v0 + e] = y.e[e];
        }
    }
}

template <typename T>
cudaError_t penalize_t(const PenalizeArgs &a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    auto pieces = [&](int each) { return (int)(((int64_t)a.v + V - 1 + THREADS * each * V - 1) / (THREADS * each * V)); };
    // The largest piece (the history is read once per piece) that still leaves four blocks to a multiprocessor.
    int each = 4;
    while (each > 1 && (int64_t)pieces(each) * a.b < 148 * 4) each /= 2;
    const int64_t blocks = (int64_t)pieces(each) * a.b;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (each == 4) penalize_kernel<T, 4><<<(unsigned)blocks, THREADS, 0, stream>>>(a, pieces(4));
    else if (each == 2) penalize_kernel<T, 2><<<(unsigned)blocks, THREADS, 0, stream>>>(a, pieces(2));
    else penalize_kernel<T, 1><<<(unsigned)blocks, THREADS, 0, stream>>>(a, pieces(1));
    return cudaGetLastError();
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
