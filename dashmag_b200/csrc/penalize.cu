// The rules a server puts on a step's logits, in one pass over them: with seen[v] whether token v is anywhere in the row's history and
// count[v] how often it is in what the model has answered (the ids behind the prompt's),
//
//     z = seen ? (z > 0 ? z / repetition : z repetition) : z,   z = z - frequency count - presence [count > 0] + bias,
//     z = -inf where the grammar does not allow v,
//
// in f32 and rounded once to the logits' dtype.
//
// A block takes a piece of one row's vocabulary and keeps a counter per token of it in shared memory: the count, and the top bit for a
// token of the prompt.  It reads the row's whole history, counts the ids that fall into its piece (integer additions, whose order does not
// matter), and then makes the pass over its logits, a chunk of a vector a thread at a time.  Nothing is sorted and no scratch is needed.
// The first chunks, the grammar's words, the row's numbers and the first ids are all asked for before any is looked at, the ids before it is
// known how many are the row's: a block waits for one trip to memory before it counts, and in the pass its chunks are DEPTH ahead.
// The history is read once per piece, from L2, so pieces are long - counters of 16 bits where no history overflows them - as far as the
// blocks still fill the GPU evenly (chunks_of).  The pass is a read and a write of the logits, bound by HBM.
// (Pieces of 8192 tokens held in registers, counters of 32 bits, four trips one after another: 256 rows of 100003 tokens with up to 8192
// ids 85 us, one trip 58, now 43; clusters of eight blocks that read a share of the history each and count for one another in
// distributed shared memory 107: half of a text's ids are a few tokens, whose words all eight then wait for.)
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "penalize.h"

namespace dash {
namespace {

constexpr int THREADS = 256, BLOCKS = 5, DEPTH = 2;   // (blocks of a multiprocessor)

// Counters of tokens: bits, the mark of a prompt's token, the count.
template <typename C> struct Counter {
    static constexpr unsigned MARK = 1u << (8 * sizeof(C) - 1);
    static constexpr int PER = 4 / sizeof(C);   // of a 32-bit word
    // One more of the token whose counter is at place `at`; the mark of the prompt's token there.
    static __device__ __forceinline__ void add(unsigned *words, unsigned at) { atomicAdd(&words[at / PER], 1u << (at % PER * 8 * sizeof(C))); }
    static __device__ __forceinline__ void mark(unsigned *words, unsigned at) { atomicOr(&words[at / PER], MARK << (at % PER * 8 * sizeof(C))); }
    static __device__ __forceinline__ unsigned get(const unsigned *w, int e) { return w[e / PER] >> (e % PER * 8 * sizeof(C)) & (MARK | (MARK - 1)); }
};

template <typename T, int V> struct alignas(16) Vec { T e[V]; };

// What a row's tokens go through.
struct Rules {
    float repetition, inverse, frequency, presence;   // (inverse: of the repetition penalty)
};
// One token's logit by its counter.  The quotient by division (QUOTIENT), or as a product with the reciprocal: two roundings of 2^-24 instead of one, of which
// a 16-bit result shows nothing but a tie now and then, and for which the reciprocal has to be finite (256 rows of 100003 tokens with up to 8192 ids,
// bf16: 47.5 us by division, 43.1 so; in f32, whose results show it, 64 rows with 2048 ids 18.7 by division, 20.0 so).
template <typename C, bool QUOTIENT> __device__ __forceinline__ float ruled(const Rules &r, float z, unsigned word) {
    if constexpr (QUOTIENT) {
        if (word) z = z > 0.f ? z / r.repetition : z * r.repetition;
    } else {
        const float factor = z > 0.f ? r.inverse : r.repetition;
        z *= word ? factor : 1.f;
    }
    const unsigned count = word & (Counter<C>::MARK - 1);
    // (As a f32: of fewer than 24 bits by the number 2^23 they are the last bits of, off the conversions' pipe.)
    const float times = sizeof(C) == 2 ? __uint_as_float(0x4b000000u | count) - 8388608.f : (float)count;
    return fmaf(-r.frequency, times, z) - (count ? r.presence : 0.f);
}

// Index i of an array of i32 / i64 as it stands there; `none` where there is no array.
__device__ __forceinline__ int64_t number(const void *p, int bytes, int i, int none) {
    return !p ? none : bytes == 8 ? static_cast<const int64_t *>(p)[i] : static_cast<int64_t>(static_cast<const int32_t *>(p)[i]);
}
__device__ __forceinline__ int within(int64_t x, int top) { return (int)min(max(x, (int64_t)0), (int64_t)top); }

constexpr int AHEAD = 4;   // ids of a thread on their way at once

// A block a piece of `chunks` times THREADS * V places.  I: the ids' integers, C: the counters'.
template <typename T, typename I, typename C>
__global__ void __launch_bounds__(THREADS, BLOCKS) penalize_kernel(PenalizeArgs a, int pieces, int chunks) {
    constexpr int V = 16 / sizeof(T), CHUNK = THREADS * V, WORDS = V * sizeof(C) / 4;
    extern __shared__ uint4 smem[];
    unsigned *words = reinterpret_cast<unsigned *>(smem);
    const int row = blockIdx.x / pieces, piece = blockIdx.x - row * pieces;
    const T *in = static_cast<const T *>(a.logits) + (int64_t)row * a.stride;
    T *out = static_cast<T *>(a.out) + (int64_t)row * a.out_stride;
    // Places are counted from the 16-byte boundary at or before the row, so that whole vectors are aligned whatever the row's address.
    const int skew = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    const bool vec = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int places = chunks * CHUNK, first = piece * places - skew;   // the token of the piece's first place (negative: there is none)
    if (first >= a.v) return;
    const int last = (int)min((int64_t)first + places, (int64_t)a.v);   // past the piece's last token

    const I *ids = static_cast<const I *>(a.ids) + (int64_t)row * a.ids_stride;
    I id[AHEAD];
    int64_t length, prompt_length;
    auto ask = [&](int i0, int end) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) id[e] = i0 + e * THREADS < end ? ids[i0 + e * THREADS] : I(-1);
    };
    length = number(a.lengths, a.lengths_bytes, row, a.t);
    prompt_length = number(a.prompt, a.prompt_bytes, row, 0);
    ask(threadIdx.x, a.t);
    Rules r;
    r.repetition = a.repetition ? a.repetition[row] : a.repetition_all;
    r.inverse = 1.f / r.repetition;
    r.frequency = a.frequency ? a.frequency[row] : a.frequency_all;
    r.presence = a.presence ? a.presence[row] : a.presence_all;
    const uint32_t *allowed = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride : nullptr;
    Vec<T, V> x[DEPTH];
    uint32_t open[DEPTH], open2[DEPTH];   // the words that hold a whole vector's bits of the grammar: one, or two where the row begins off a boundary
    auto whole = [&](int v0) { return vec && v0 >= 0 && v0 <= a.v - V; };
    auto fetch = [&](int v0, Vec<T, V> &x, uint32_t &open, uint32_t &open2) {
        if (v0 < last && whole(v0)) {
            *reinterpret_cast<uint4 *>(&x) = *reinterpret_cast<const uint4 *>(in + v0);
            if (allowed) {   // (not looked at before the pass: that would be a wait for them here)
                open = allowed[v0 >> 5];
                if (skew) open2 = allowed[(v0 + V - 1) >> 5];
            }
        }
    };
    const int v_first = first + (int)threadIdx.x * V;
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) fetch(v_first + j * CHUNK, x[j], open[j], open2[j]);
    const int len = within(length, a.t), prompt = within(prompt_length, len);
    if (len > 0) {
        for (int i = threadIdx.x; i < places / (4 * Counter<C>::PER); i += THREADS) smem[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int i0 = threadIdx.x; i0 < len; i0 += THREADS * AHEAD) {
            if (i0 >= THREADS * AHEAD) ask(i0, len);
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                // (Ids outside the vocabulary, padding's -1 among them, count for nothing; another piece's come out past this one's places.)
                const unsigned at = (unsigned)((int)id[e] - first);
                const int i = i0 + e * THREADS;
                if ((std::make_unsigned_t<I>)id[e] >= (std::make_unsigned_t<I>)a.v || at >= (unsigned)places || i >= len) continue;
                if (i < prompt) Counter<C>::mark(words, at);
                else Counter<C>::add(words, at);
            }
        }
        __syncthreads();
    }

    const int64_t bias0 = (int64_t)row * a.bias_stride;
    auto bias_at = [&](int v) {
        return a.bias_f32 ? static_cast<const float *>(a.bias)[bias0 + v] : Num<T>::to_f32(static_cast<const T *>(a.bias)[bias0 + v]);
    };
    const bool quotient = sizeof(T) == 4 || isinf(r.inverse);
    auto pass = [&](int v0, const Vec<T, V> &x, uint32_t bits) {
        alignas(16) unsigned w[WORDS];
#pragma unroll
        for (int e = 0; e < WORDS; ++e) w[e] = 0;
        if (len > 0) {
            const unsigned *at = words + (v0 - first) / Counter<C>::PER;
#pragma unroll
            for (int e = 0; e < WORDS; e += WORDS < 4 ? 2 : 4) {
                if constexpr (WORDS < 4) *reinterpret_cast<uint2 *>(&w[e]) = *reinterpret_cast<const uint2 *>(at + e);
                else *reinterpret_cast<uint4 *>(&w[e]) = *reinterpret_cast<const uint4 *>(at + e);
            }
        }
        if (!whole(v0)) {   // the row's ends
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int v = v0 + e;
                if (v < 0 || v >= a.v) continue;
                float z = Num<T>::to_f32(in[v]);
                z = quotient ? ruled<C, true>(r, z, Counter<C>::get(w, e)) : ruled<C, false>(r, z, Counter<C>::get(w, e));
                if (a.bias) z += bias_at(v);
                if (allowed && !(allowed[v >> 5] >> (v & 31) & 1u)) z = -INFINITY;
                out[v] = Num<T>::from_f32(z);
            }
            return;
        }
        float z[V];
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = Num<T>::to_f32(x.e[e]);
        if (len > 0) {
            // (All of a vector or nothing: a history of some thousands touches one vector in ten, nearly every warp's 32 of them; word by word the
            // branches cost what they spare.)
            unsigned any = 0;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) any |= w[i];
            if (any && quotient) {
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = ruled<C, true>(r, z[e], Counter<C>::get(w, e));
            } else if (any) {
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = ruled<C, false>(r, z[e], Counter<C>::get(w, e));
            }
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
        if (allowed) {
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = bits >> e & 1u ? z[e] : -INFINITY;
        }
        Vec<T, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e) y.e[e] = Num<T>::from_f32(z[e]);
        *reinterpret_cast<uint4 *>(out + v0) = *reinterpret_cast<const uint4 *>(&y);
    };
    for (int v0 = v_first; v0 < last; v0 += DEPTH * CHUNK) {
#pragma unroll
        for (int j = 0; j < DEPTH; ++j) {
            const int v = v0 + j * CHUNK;
            if (v >= last) break;
            const Vec<T, V> now = x[j];
            const uint32_t bits = open[j], bits2 = open2[j];
            fetch(v + DEPTH * CHUNK, x[j], open[j], open2[j]);
            pass(v, now, skew ? __funnelshift_r(bits, bits2, v & 31) : bits >> (v & 31));
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Calls without a history
// ---------------------------------------------------------------------------------------------
// The bias and the grammar alone.  EACH vectors a thread, all asked for at once, a block as long as they take: nothing is counted, and nobody
// waits for anybody (256 rows of 100003 tokens in bf16 18 us, 5.8 TB/s, where the kernel above takes 26 for histories of one id).
// (Rows with short histories this way too, with their ids' logits made in a kernel beside it and put over its results: 25 us against 30 at 512
// ids a row, but 29 against 32 at 2048, 44 against 41 at 8192, and 5.7 against 3.3 for one row of 32768.)
template <typename T, int EACH>
__global__ void __launch_bounds__(THREADS) penalize_all_kernel(PenalizeArgs a, int pieces) {
    constexpr int V = 16 / sizeof(T), PIECE = THREADS * EACH * V;
    const int row = blockIdx.x / pieces, piece = blockIdx.x - row * pieces;
    const T *in = static_cast<const T *>(a.logits) + (int64_t)row * a.stride;
    T *out = static_cast<T *>(a.out) + (int64_t)row * a.out_stride;
    const int skew = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    const bool vec = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int first = piece * PIECE - skew;
    const uint32_t *allowed = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride : nullptr;
    const int64_t bias0 = (int64_t)row * a.bias_stride;
    auto token = [&](int j) { return first + (j * THREADS + (int)threadIdx.x) * V; };
    auto whole = [&](int v0) { return vec && v0 >= 0 && v0 <= a.v - V; };
    auto bias_at = [&](int v) {
        return a.bias_f32 ? static_cast<const float *>(a.bias)[bias0 + v] : Num<T>::to_f32(static_cast<const T *>(a.bias)[bias0 + v]);
    };
    Vec<T, V> x[EACH];
    uint32_t open[EACH], open2[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int v0 = token(j);
        if (!whole(v0)) continue;
        *reinterpret_cast<uint4 *>(&x[j]) = *reinterpret_cast<const uint4 *>(in + v0);
        if (allowed) {
            open[j] = allowed[v0 >> 5];
            if (skew) open2[j] = allowed[(v0 + V - 1) >> 5];
        }
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int v0 = token(j);
        if (!whole(v0)) {   // the row's ends
            for (int v = max(v0, 0); v < min(v0 + V, a.v); ++v) {
                float z = Num<T>::to_f32(in[v]);
                if (a.bias) z += bias_at(v);
                if (allowed && !(allowed[v >> 5] >> (v & 31) & 1u)) z = -INFINITY;
                out[v] = Num<T>::from_f32(z);
            }
            continue;
        }
        if (a.bias || allowed) {
            float z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = Num<T>::to_f32(x[j].e[e]);
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
            if (allowed) {
                const uint32_t bits = skew ? __funnelshift_r(open[j], open2[j], v0 & 31) : open[j] >> (v0 & 31);
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = bits >> e & 1u ? z[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) x[j].e[e] = Num<T>::from_f32(z[e]);
        }
        *reinterpret_cast<uint4 *>(out + v0) = *reinterpret_cast<const uint4 *>(&x[j]);
    }
}

constexpr int MOST_BYTES = 40 * 1024;   // of counters

// Chunks of a piece.  The blocks run in waves of five a multiprocessor; a block costs its chunks, and about three and a half of them until
// its first is there, and the history.
int chunks_of(int64_t chunks_of_row, int b, int t, int most) {
    int best = 1;
    double least = 0.;
    for (int k = 1; k <= most; ++k) {
        const int64_t blocks = (chunks_of_row + k - 1) / k * b, waves = (blocks + BLOCKS * 148 - 1) / (BLOCKS * 148);
        const double cost = waves * (k + 3.5 + t / 1500.);
        if (k == 1 || cost < least) { best = k; least = cost; }
        if (k >= chunks_of_row) break;
    }
    return best;
}

template <typename T, typename I, typename C>
cudaError_t run(const PenalizeArgs &a, cudaStream_t stream) {
    constexpr int CHUNK = THREADS * 16 / (int)sizeof(T);
    const int64_t row = ((int64_t)a.v + 16 / (int)sizeof(T) - 1 + CHUNK - 1) / CHUNK;
    const int chunks = chunks_of(row, a.b, a.t, MOST_BYTES / (CHUNK * (int)sizeof(C)));
    const int64_t pieces = (row + chunks - 1) / chunks, blocks = pieces * a.b;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const auto kernel = penalize_kernel<T, I, C>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_BYTES);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)blocks, THREADS, (size_t)chunks * CHUNK * sizeof(C), stream>>>(a, (int)pieces, chunks);
    return cudaGetLastError();
}

template <typename T>
cudaError_t penalize_t(const PenalizeArgs &a, cudaStream_t stream) {
    if (!a.ids) {
        constexpr int V = 16 / sizeof(T), EACH = 4, PIECE = THREADS * EACH * V;
        const int64_t pieces = ((int64_t)a.v + V - 1 + PIECE - 1) / PIECE, blocks = pieces * a.b;
        if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
        penalize_all_kernel<T, EACH><<<(unsigned)blocks, THREADS, 0, stream>>>(a, (int)pieces);
        return cudaGetLastError();
    }
    // (A counter of 16 bits counts to 32767.)
    const bool small = a.t <= 0x7fff;
    if (a.ids_bytes == 8) return small ? run<T, int64_t, uint16_t>(a, stream) : run<T, int64_t, uint32_t>(a, stream);
    return small ? run<T, int32_t, uint16_t>(a, stream) : run<T, int32_t, uint32_t>(a, stream);
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
