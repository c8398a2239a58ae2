// The decoding step of a batch whose sequences share prompts.  Sequence b's keys are those of its prompt, b / each, and its own behind
// them; one softmax over both:
//
//     out = sum over parts of exp(lse_i - max) o_i / sum of exp(lse_i - max),
//
// with o_i the normalised output over one run of keys and lse_i the logarithm of its sum of exponentials.  The parts over the
// sequences' own keys are those of the decoding step's split pass (decode.cu).  The parts over a prompt's keys come from a pass in
// which all of the prompt's sequences are the rows of one product, each x group of them against every key-value head, so that a
// prompt's keys are read once per tile of rows (of 256, of 128 where heads are longer than 128; of 32 here) and not once per sequence: on the
// tensor cores the training forward's kernels take it
// (fwd2_sm100.cu, fwd_sm100.cu, the prefix form; 16-bit, head dimensions of whole 16-byte vectors), else the kernel here.  Own keys that the
// split pass could only read element by element are swept the same way, every sequence a prompt of one.
// The passes touch nothing of one another: that over the own keys, which HBM bounds, is launched beside the prompts', which is cut into no
// more blocks than leave it multiprocessors (sm100_prefix_splits), and the merge under its end.
#include <algorithm>

#include "common.cuh"
#include "launch.h"
#include "prefix.h"
#include "sm100_kernels.h"

namespace dash {
namespace {

// ---------------------------------------------------------------------------------------------
// The prompts' part on the CUDA cores
// ---------------------------------------------------------------------------------------------
// A block takes 32 rows (sequence, head) of a prompt's key-value head and a run of its keys, 64 at a time: queries, keys and then the
// values of the same keys in shared memory as f32, scores and outputs in registers, two rows of four keys and of D / 16 features to a
// thread, sixteen threads to a row.  The values are on their way to registers while the scores are made, the next keys while the outputs
// are.  f32 products and sums throughout, bound by the FMA pipe and its operands from shared memory; with few rows by the trips to
// memory (two prompts of 777 keys, three sequences each, 6 / 2 heads of 80 in f32: 41 us one element a load, waited for, now 19 for all of the step).
constexpr int ROWS = 32, KEYS = 64, THREADS = 256, MAX_D = 256;

// Floats between rows of shared memory: whole 16-byte vectors, an odd number of them, so that eight rows' lie in banks of their own.
__host__ __device__ constexpr int pitch_of(int d) { return 4 * (((d + 3) / 4) | 1); }
size_t generic_smem(int d) { return sizeof(float) * ((size_t)(ROWS + KEYS) * pitch_of(d) + ROWS * (KEYS + 4)); }

// 64 keys' rows on their way into shared memory, VE elements a load (16 bytes, or one element): up to AHEAD loads of a thread in registers,
// what is more when they are put down.
template <typename T, int VE> struct Rows {
    static constexpr int AHEAD = VE > 1 ? 8 : 16;
    struct alignas(VE > 1 ? 16 : sizeof(T)) Item { T e[VE]; };
    Item held[AHEAD];
    const T *base;   // the head's first key
    int64_t st, sd;
    int per, kmax;   // loads of a row; past the run's last key
    __device__ __forceinline__ Rows(const View4 &v, int n, int hk, int d, int kmax)
        : base(static_cast<const T *>(v.ptr) + (int64_t)n * v.sb + (int64_t)hk * v.sh), st(v.st), sd(v.sd), per(d / VE), kmax(kmax) {}
    __device__ __forceinline__ Item load(int k0, int i) const {
        const int k = i / per, c = (i - k * per) * VE;
        Item x;
        // (Keys past the run are zeros, whatever lies there.)
        if (k < KEYS && k0 + k < kmax) {
            const T *from = base + (int64_t)(k0 + k) * st + (int64_t)c * (VE > 1 ? 1 : sd);
            if constexpr (VE > 1) *reinterpret_cast<uint4 *>(&x) = *reinterpret_cast<const uint4 *>(from);
            else x.e[0] = *from;
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) x.e[e] = Num<T>::from_f32(0.f);
        }
        return x;
    }
    __device__ __forceinline__ void ask(int k0) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (a * THREADS < KEYS * per) held[a] = load(k0, threadIdx.x + a * THREADS);
    }
    __device__ __forceinline__ void put(float *to, int pitch, int k0) {
#pragma unroll 1
        for (int i0 = 0; i0 < KEYS * per; i0 += AHEAD * THREADS) {
            if (i0 > 0) {
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) held[a] = load(k0, i0 + threadIdx.x + a * THREADS);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int i = i0 + threadIdx.x + a * THREADS, k = i / per, c = (i - k * per) * VE;
                if (k >= KEYS) break;
                float *at = to + k * pitch + c;
                if constexpr (VE == 1) {
                    at[0] = Num<T>::to_f32(held[a].e[0]);
                } else {
#pragma unroll
                    for (int e = 0; e < VE; e += 4)
                        *reinterpret_cast<float4 *>(at + e) = make_float4(Num<T>::to_f32(held[a].e[e]), Num<T>::to_f32(held[a].e[e + 1]),
                                                                          Num<T>::to_f32(held[a].e[e + 2]), Num<T>::to_f32(held[a].e[e + 3]));
                }
            }
        }
    }
};

// VE: elements a load of keys and values; J: groups of 64 features, a quarter of a group to a thread.
template <typename T, int VE, int J>
__global__ void __launch_bounds__(THREADS) prefix_generic_kernel(PrefixArgs a) {
    extern __shared__ float4 smem4[];
    __shared__ int row_lo[ROWS], row_hi[ROWS], span[2];
    allow_beside();   // the merge
    const int pitch = pitch_of(a.d), d4 = (a.d + 3) / 4;
    float *qs = reinterpret_cast<float *>(smem4), *ks = qs + ROWS * pitch, *ps = ks + KEYS * pitch;
    const int group = a.hq / a.hkv, split = blockIdx.x % a.splits, hk = blockIdx.x / a.splits % a.hkv;
    const int64_t r0 = (int64_t)(blockIdx.x / a.splits / a.hkv) * ROWS, rows = (int64_t)a.each * group;
    const int n = blockIdx.y, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    auto sequence = [&](int64_t r) { return (int64_t)n * a.each + r / group; };
    auto head = [&](int64_t r) { return hk * group + (int)(r % group); };

    static_assert(ROWS == 32, "a warp's lanes are the rows");
    if (threadIdx.x < ROWS) {
        int lo = a.p, hi = 0;
        const int64_t r = r0 + threadIdx.x;
        if (r < rows) prefix_bounds(a.reach, n, sequence(r), lo, hi);
        row_lo[threadIdx.x] = lo;
        row_hi[threadIdx.x] = hi;
        lo = warp_min_i(hi > lo ? lo : a.p);
        hi = warp_max_i(hi);
        if (threadIdx.x == 0) { span[0] = lo; span[1] = hi; }
    }
    // The queries: eight threads a row, eight loads of each at once, asked for beside the lengths.
    // (Columns behind the features, up to a whole vector: zeros, in the keys too, which are written but for them.)
    {
        struct alignas(VE > 1 ? 16 : sizeof(T)) Item { T e[VE]; };
        const int qr = threadIdx.x / 8, per = a.d / VE;
        const int64_t r = r0 + qr;
        const T *from = static_cast<const T *>(a.q) + (r < rows ? sequence(r) * a.q_sb + head(r) * a.q_sh : 0);
        float *to = qs + qr * pitch;
        for (int i0 = threadIdx.x % 8; i0 < per; i0 += 64) {
            Item x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (r >= rows || i0 + 8 * j >= per) continue;
                if constexpr (VE > 1) *reinterpret_cast<uint4 *>(&x[j]) = *reinterpret_cast<const uint4 *>(from + (i0 + 8 * j) * VE);
                else x[j].e[0] = from[(i0 + 8 * j) * a.q_sd];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i0 + 8 * j >= per) continue;
#pragma unroll
                for (int e = 0; e < VE; ++e) to[(i0 + 8 * j) * VE + e] = r < rows ? Num<T>::to_f32(x[j].e[e]) : 0.f;
            }
        }
        if (threadIdx.x % 8 == 0)
            for (int c = a.d; c < 4 * d4; ++c) to[c] = 0.f;
    }
    if (a.d % 4 != 0)
        for (int i = threadIdx.x; i < KEYS * 4; i += THREADS)
            if (4 * (d4 - 1) + i % 4 >= a.d) ks[i / 4 * pitch + 4 * (d4 - 1) + i % 4] = 0.f;
    __syncthreads();
    int kmin = span[0], kmax = span[1];
    split_keys(split, a.splits, KEYS, kmin, kmax);

    float4 acc[2][J];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) acc[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    Rows<T, VE> keys(a.k, n, hk, a.d, kmax), values(a.v, n, hk, a.d, kmax);
    const int lo0 = row_lo[2 * ty], lo1 = row_lo[2 * ty + 1], hi0 = row_hi[2 * ty], hi1 = row_hi[2 * ty + 1];
    if (kmin < kmax) keys.ask(kmin);
    for (int k0 = kmin; k0 < kmax; k0 += KEYS) {
        keys.put(ks, pitch, k0);
        __syncthreads();
        values.ask(k0);
        float s[2][4] = {};
        const float4 *q0 = reinterpret_cast<const float4 *>(qs + 2 * ty * pitch), *q1 = q0 + pitch / 4, *kk = reinterpret_cast<const float4 *>(ks + tx * pitch);
#pragma unroll 2
        for (int c = 0; c < d4; ++c) {
            const float4 x = q0[c], y = q1[c];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 k = kk[j * 4 * pitch + c];   // key tx + 16 j
                s[0][j] = fmaf(x.x, k.x, fmaf(x.y, k.y, fmaf(x.z, k.z, fmaf(x.w, k.w, s[0][j]))));
                s[1][j] = fmaf(y.x, k.x, fmaf(y.y, k.y, fmaf(y.z, k.z, fmaf(y.w, k.w, s[1][j]))));
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int lo = i ? lo1 : lo0, hi = i ? hi1 : hi0;
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = k0 + tx + 16 * j;
                s[i][j] = key >= lo && key < hi && key < kmax ? s[i][j] * a.scale : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, corr = expf(m[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = expf(s[i][j] - base);
                sum += p;
                ps[(2 * ty + i) * (KEYS + 4) + tx + 16 * j] = p;
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[i] = l[i] * corr + sum;
            m[i] = mn;
#pragma unroll
            for (int j = 0; j < J; ++j) { acc[i][j].x *= corr; acc[i][j].y *= corr; acc[i][j].z *= corr; acc[i][j].w *= corr; }
        }
        __syncthreads();
        values.put(ks, pitch, k0);
        __syncthreads();
        if (k0 + KEYS < kmax) keys.ask(k0 + KEYS);
        const int there = min(KEYS, kmax - k0);
        const float *p0 = ps + 2 * ty * (KEYS + 4), *p1 = p0 + KEYS + 4;
#pragma unroll 8
        for (int k = 0; k < there; ++k) {
            const float w0 = p0[k], w1 = p1[k];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (tx + 16 * j >= d4) break;
                const float4 v = *reinterpret_cast<const float4 *>(ks + k * pitch + 4 * (tx + 16 * j));
                acc[0][j].x = fmaf(w0, v.x, acc[0][j].x); acc[0][j].y = fmaf(w0, v.y, acc[0][j].y);
                acc[0][j].z = fmaf(w0, v.z, acc[0][j].z); acc[0][j].w = fmaf(w0, v.w, acc[0][j].w);
                acc[1][j].x = fmaf(w1, v.x, acc[1][j].x); acc[1][j].y = fmaf(w1, v.y, acc[1][j].y);
                acc[1][j].z = fmaf(w1, v.z, acc[1][j].z); acc[1][j].w = fmaf(w1, v.w, acc[1][j].w);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t r = r0 + 2 * ty + i;
        if (r >= rows) continue;
        const int64_t at = (int64_t)split * a.n * a.each * a.hq + sequence(r) * a.hq + head(r);
        // (A part that met a NaN leaves one: -inf is the mark of a part without keys.)
        if (tx == 0) a.part_lse[at] = l[i] != 0.f ? m[i] + logf(l[i]) : -INFINITY;
        const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;
        float *po = a.part_o + at * a.d;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int c = 4 * (tx + 16 * j);
            if (c < a.d) po[c] = acc[i][j].x * inv;
            if (c + 1 < a.d) po[c + 1] = acc[i][j].y * inv;
            if (c + 2 < a.d) po[c + 2] = acc[i][j].z * inv;
            if (c + 3 < a.d) po[c + 3] = acc[i][j].w * inv;
        }
    }
    end_beside();
}

// A warp a row of one cache.
template <typename T>
__global__ void __launch_bounds__(THREADS) prefix_append_kernel(DecodeArgs a) {
    const int64_t item = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    if (item >= (int64_t)a.b * a.hkv * 2) return;
    const bool is_v = item & 1;
    const int b = (int)(item / 2 / a.hkv), hk = (int)(item / 2 % a.hkv), at = decode_append_at(a, b);
    if (at < 0) return;
    const View4 &to = is_v ? a.v : a.k;
    const T *from = static_cast<const T *>(is_v ? a.v_new : a.k_new) + ((int64_t)b * a.hkv + hk) * a.d;
    T *row = static_cast<T *>(const_cast<void *>(to.ptr)) + (int64_t)b * to.sb + (int64_t)at * to.st + (int64_t)hk * to.sh;
    for (int c = threadIdx.x & 31; c < a.d; c += 32) row[(int64_t)c * to.sd] = from[c];
}

// ---------------------------------------------------------------------------------------------
// The merge
// ---------------------------------------------------------------------------------------------
// WARPS warps a row; LANES lanes a part (16 where a head is at most 64 features, else 32), four features or J times four each.  A lane asks for EACH
// parts' log-sum-exps and features at once, the first of them before it is known how many chunks the sequence's own keys make, and keeps
// maximum, sum and outputs as the softmax does; the lanes' groups and the warps meet in order, so the bits repeat.
// Bound by launch and latency, the parts being in L2: one trip to memory for most calls (one for the lengths, one for the log-sum-exps, one for the
// parts: 32 prompts of sixteen answers, 8192 rows of 64, 56 us the step, with one 51).
constexpr int MERGE_THREADS = 128;

template <typename T, int WARPS, int EACH, int LANES, int J>
__global__ void __launch_bounds__(MERGE_THREADS) prefix_merge_kernel(PrefixMergeArgs a) {
    constexpr int AT_ONCE = MERGE_THREADS / 32 / WARPS, SUBS = 32 / LANES, STEP = WARPS * SUBS;   // rows of a block; groups of lanes; parts of a round
    __shared__ float4 red[AT_ONCE][WARPS][J][32];
    __shared__ float2 stat[AT_ONCE][WARPS][32];
    wait_before();   // the passes
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS, mine = (threadIdx.x >> 5) / WARPS;
    const int slot = warp * SUBS + lane / LANES, col = lane % LANES;
    const int64_t row = (int64_t)blockIdx.x * AT_ONCE + mine;
    const bool live = row < a.rows, vec = a.d % 4 == 0;
    const bool chunked = a.own.s > 0 && a.own_splits == 0;   // the own keys' parts are the split pass's chunks
    const int most = live ? a.splits + (chunked ? a.own.splits : a.own_splits) : 0;
    // Where part i of the row lies, counted in rows of its array.
    auto own_at = [&](int i) { return chunked ? row * a.own.splits + i - a.splits : (int64_t)(i - a.splits) * a.rows + row; };
    float lse[EACH];
    float4 x[EACH][J];
    auto ask = [&](int i0, int end) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int i = i0 + e * STEP + slot;
            lse[e] = -INFINITY;
#pragma unroll
            for (int j = 0; j < J; ++j) x[e][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i >= end) continue;
            const int64_t at = i < a.splits ? i * a.rows + row : own_at(i);
            lse[e] = (i < a.splits ? a.part_lse : a.own.part_lse)[at];
            const float *po = (i < a.splits ? a.part_o : a.own.part_o) + at * a.d;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int c = 4 * (col + LANES * j);
                if (vec) {
                    if (c < a.d) x[e][j] = *reinterpret_cast<const float4 *>(po + c);
                } else {
                    if (c < a.d) x[e][j].x = po[c];
                    if (c + 1 < a.d) x[e][j].y = po[c + 1];
                    if (c + 2 < a.d) x[e][j].z = po[c + 2];
                    if (c + 3 < a.d) x[e][j].w = po[c + 3];
                }
            }
        }
    };
    ask(0, most);
    int parts = most;
    if (live && chunked) {
        int first, len;
        decode_range(a.own, (int)(row / a.hq), first, len);
        parts = a.splits + (len > first ? (len - first + a.own.chunk - 1) / a.own.chunk : 0);   // those that hold keys
    }
    float top = -INFINITY, den = 0.f;
    float4 num[J];
#pragma unroll
    for (int j = 0; j < J; ++j) num[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    // Whether there is such a part: a run that saw no key left nothing.  (A chunk of the sequence's own always left something; a NaN in it is one of the row.)
    auto there = [&](int i, float lse) { return i < parts && ((chunked && i >= a.splits) || lse != -INFINITY); };
    auto scaled = [&](float by) {
        den *= by;
#pragma unroll
        for (int j = 0; j < J; ++j) { num[j].x *= by; num[j].y *= by; num[j].z *= by; num[j].w *= by; }
    };
    auto weight = [](float x, float top) { return expf(x - (top == -INFINITY ? 0.f : top)); };
    for (int i0 = 0; i0 < parts; i0 += EACH * STEP) {
        if (i0 > 0) ask(i0, parts);
        float now = top;
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            if (there(i0 + e * STEP + slot, lse[e])) now = fmaxf(now, lse[e]);
        scaled(weight(top, now));
        top = now;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            if (!there(i0 + e * STEP + slot, lse[e])) continue;
            const float w = weight(lse[e], top);
            den += w;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                num[j].x = fmaf(w, x[e][j].x, num[j].x);
                num[j].y = fmaf(w, x[e][j].y, num[j].y);
                num[j].z = fmaf(w, x[e][j].z, num[j].z);
                num[j].w = fmaf(w, x[e][j].w, num[j].w);
            }
        }
    }
    auto join = [&](float o_top, float o_den, auto &&o_num) {
        const float both = fmaxf(top, o_top), w = weight(o_top, both);
        scaled(weight(top, both));
        top = both;
        den = fmaf(w, o_den, den);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float4 y = o_num(j);
            num[j].x = fmaf(w, y.x, num[j].x);
            num[j].y = fmaf(w, y.y, num[j].y);
            num[j].z = fmaf(w, y.z, num[j].z);
            num[j].w = fmaf(w, y.w, num[j].w);
        }
    };
    if constexpr (SUBS == 2) {
        const float o_top = __shfl_down_sync(0xffffffffu, top, 16), o_den = __shfl_down_sync(0xffffffffu, den, 16);
        float4 o[J];
#pragma unroll
        for (int j = 0; j < J; ++j)
            o[j] = make_float4(__shfl_down_sync(0xffffffffu, num[j].x, 16), __shfl_down_sync(0xffffffffu, num[j].y, 16),
                               __shfl_down_sync(0xffffffffu, num[j].z, 16), __shfl_down_sync(0xffffffffu, num[j].w, 16));
        join(o_top, o_den, [&](int j) { return o[j]; });   // (the upper lanes' own are of no use to anybody)
    }
    if constexpr (WARPS > 1) {
        stat[mine][warp][lane] = make_float2(top, den);
#pragma unroll
        for (int j = 0; j < J; ++j) red[mine][warp][j][lane] = num[j];
        __syncthreads();
        if (warp != 0) return;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            const float2 o = stat[mine][w][lane];
            join(o.x, o.y, [&](int j) { return red[mine][w][j][lane]; });
        }
    }
    if (!live || lane >= LANES) return;
    const float inv = den != 0.f ? 1.f / den : 0.f;
    T *out = static_cast<T *>(a.out) + row * a.d;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = 4 * (col + LANES * j);
        if (c < a.d) out[c] = Num<T>::from_f32(num[j].x * inv);
        if (c + 1 < a.d) out[c + 1] = Num<T>::from_f32(num[j].y * inv);
        if (c + 2 < a.d) out[c + 2] = Num<T>::from_f32(num[j].z * inv);
        if (c + 3 < a.d) out[c + 3] = Num<T>::from_f32(num[j].w * inv);
    }
}

template <typename T, int VE, int J>
cudaError_t generic_j(const PrefixArgs &a, dim3 grid, cudaStream_t stream) {
    const auto kernel = prefix_generic_kernel<T, VE, J>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)generic_smem(64 * J));
    if (e != cudaSuccess) return e;
    return launch_beside(kernel, grid, THREADS, generic_smem(a.d), stream, a.beside != 0, a);
}
template <typename T, int VE>
cudaError_t generic_v(const PrefixArgs &a, dim3 grid, cudaStream_t stream) {
    return a.d <= 64 ? generic_j<T, VE, 1>(a, grid, stream) : a.d <= 128 ? generic_j<T, VE, 2>(a, grid, stream) : generic_j<T, VE, 4>(a, grid, stream);
}
template <typename T>
cudaError_t generic_t(const PrefixArgs &a, dim3 grid, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    auto vectors = [&](const View4 &t) {
        return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0 && t.sd == 1 && t.sb % V == 0 && t.st % V == 0 && t.sh % V == 0;
    };
    return a.d % V == 0 && vectors(a.k) && vectors(a.v) && vectors(View4{a.q, 0, a.q_sb, a.q_sh, a.q_sd}) ? generic_v<T, V>(a, grid, stream) : generic_v<T, 1>(a, grid, stream);
}

template <typename T, int WARPS, int EACH>
cudaError_t merge_w(const PrefixMergeArgs &a, cudaStream_t stream) {
    constexpr int AT_ONCE = MERGE_THREADS / 32 / WARPS;
    const int64_t blocks = (a.rows + AT_ONCE - 1) / AT_ONCE;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const auto kernel = a.d <= 64 ? prefix_merge_kernel<T, WARPS, EACH, 16, 1> : a.d <= 128 ? prefix_merge_kernel<T, WARPS, EACH, 32, 1> : prefix_merge_kernel<T, WARPS, EACH, 32, 2>;
    return launch_beside(kernel, dim3((unsigned)blocks), MERGE_THREADS, 0, stream, true, a);
}
// Several warps a row where one would not have all parts on their way at once, and rows are few.  (The step, us, one warp of eight parts | two of
// four | four of four: 2048 rows of 128, 42.3 | 42.4 | 43.3, 1536 34.1 | 33.7 | 34.8, 512 31.0 | 29.8 | 28.4, 128 35.6 | 32.7 | 29.4, the
// sweep over the prompts 1 to 3 us shorter than it is now, with probabilities of one part.)
template <typename T>
cudaError_t merge_t(const PrefixMergeArgs &a, cudaStream_t stream) {
    const int parts = a.splits + (a.own.s > 0 ? std::max(a.own_splits, a.own_splits > 0 ? 0 : a.own.splits) : 0);
    if (parts <= 8 * (a.d <= 64 ? 2 : 1) || a.rows > 148 * 16) return merge_w<T, 1, 8>(a, stream);
    return a.rows <= 148 * 8 ? merge_w<T, 4, 4>(a, stream) : merge_w<T, 2, 4>(a, stream);
}

int64_t generic_units(int n, int each, int hq, int hkv) { return (int64_t)n * hkv * (((int64_t)each * (hq / hkv) + ROWS - 1) / ROWS); }

}  // namespace

// As many runs of keys as fill the multiprocessors twice, of a tile at least.
int prefix_generic_splits(int n, int each, int p, int hq, int hkv) {
    const int64_t units = generic_units(n, each, hq, hkv), tiles = (p + KEYS - 1) / KEYS;
    return (int)std::max<int64_t>(1, std::min<int64_t>(tiles, 2 * 148 / std::max<int64_t>(units, 1)));
}

cudaError_t launch_prefix_generic(int dtype, const PrefixArgs &a, cudaStream_t stream, int *launches) {
    const int64_t x = generic_units(1, a.each, a.hq, a.hkv) * a.splits;
    if (x > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)x, (unsigned)a.n);
    *launches += 1;
    switch (dtype) {
        case 0: return generic_t<float>(a, grid, stream);
        case 1: return generic_t<__nv_bfloat16>(a, grid, stream);
        default: return generic_t<__half>(a, grid, stream);
    }
}

cudaError_t launch_prefix_append(int dtype, const DecodeArgs &a, cudaStream_t stream, int *launches) {
    const int64_t blocks = ((int64_t)a.b * a.hkv * 2 + THREADS / 32 - 1) / (THREADS / 32);
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    *launches += 1;
    if (dtype == 0) prefix_append_kernel<float><<<(unsigned)blocks, THREADS, 0, stream>>>(a);
    else if (dtype == 1) prefix_append_kernel<__nv_bfloat16><<<(unsigned)blocks, THREADS, 0, stream>>>(a);
    else prefix_append_kernel<__half><<<(unsigned)blocks, THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_prefix_merge(int dtype, const PrefixMergeArgs &a, cudaStream_t stream, int *launches) {
    *launches += 1;
    switch (dtype) {
        case 0: return merge_t<float>(a, stream);
        case 1: return merge_t<__nv_bfloat16>(a, stream);
        default: return merge_t<__half>(a, stream);
    }
}

}  // namespace dash
