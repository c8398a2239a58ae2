// The decoding step of a batch whose sequences share prompts.  Sequence b's keys are those of its prompt, b / each, and its own behind
// them; one softmax over both:
//
//     out = sum over parts of exp(lse_i - max) o_i / sum of exp(lse_i - max),
//
// with o_i the normalised output over one run of keys and lse_i the logarithm of its sum of exponentials.  The parts over the
// sequences' own keys are those of the decoding step's split pass (decode.cu).  The parts over a prompt's keys come from a pass in
// which all of the prompt's sequences are the rows of one product, each x group of them against every key-value head, so that a
// prompt's keys are read from HBM once and not once per sequence: on the tensor cores the training forward's kernels take it
// (fwd2_sm100.cu, fwd_sm100.cu, the prefix form; 16-bit, head dimension 64, 128 or 256), else the kernel here.
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
// thread, sixteen threads to a row.  f32 products and sums throughout, bound by the FMA pipe and its operands from shared memory.
constexpr int ROWS = 32, KEYS = 64, THREADS = 256, MAX_D = 256;

size_t generic_smem(int d) { return sizeof(float) * ((size_t)ROWS * (d + 1) + (size_t)KEYS * (d + 1) + ROWS * (KEYS + 1)); }

template <typename T>
__global__ void __launch_bounds__(THREADS) prefix_generic_kernel(PrefixArgs a) {
    extern __shared__ float smem[];
    __shared__ int row_lo[ROWS], row_hi[ROWS];
    allow_beside();   // the merge
    const int pitch = a.d + 1;
    float *qs = smem, *ks = qs + ROWS * pitch, *ps = ks + KEYS * pitch;
    const int group = a.hq / a.hkv, split = blockIdx.x % a.splits, hk = blockIdx.x / a.splits % a.hkv;
    const int64_t r0 = (int64_t)(blockIdx.x / a.splits / a.hkv) * ROWS, rows = (int64_t)a.each * group;
    const int n = blockIdx.y, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    auto sequence = [&](int64_t r) { return (int64_t)n * a.each + r / group; };
    auto head = [&](int64_t r) { return hk * group + (int)(r % group); };

    if (threadIdx.x < ROWS) {
        int lo = a.p, hi = 0;
        const int64_t r = r0 + threadIdx.x;
        if (r < rows) prefix_bounds(a.reach, n, sequence(r), lo, hi);
        row_lo[threadIdx.x] = lo;
        row_hi[threadIdx.x] = hi;
    }
    for (int i = threadIdx.x; i < ROWS * a.d; i += THREADS) {
        const int r = i / a.d, c = i - r * a.d;
        qs[r * pitch + c] = r0 + r < rows ? Num<T>::to_f32(static_cast<const T *>(a.q)[sequence(r0 + r) * a.q_sb + head(r0 + r) * a.q_sh + c * a.q_sd]) : 0.f;
    }
    __syncthreads();
    int kmin = a.p, kmax = 0;
    for (int i = 0; i < ROWS; ++i) { kmin = min(kmin, row_hi[i] > row_lo[i] ? row_lo[i] : a.p); kmax = max(kmax, row_hi[i]); }
    split_keys(split, a.splits, KEYS, kmin, kmax);

    float acc[2][MAX_D / 16], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MAX_D / 16; ++j) acc[i][j] = 0.f;
    // (Keys past the run are zeros, whatever lies there.)
    auto fill = [&](const View4 &t, int k0) {
        for (int i = threadIdx.x; i < KEYS * a.d; i += THREADS) {
            const int k = i / a.d, c = i - k * a.d;
            ks[k * pitch + c] = k0 + k < kmax ? load_f32<T>(t, n, k0 + k, hk, c) : 0.f;
        }
    };
    for (int k0 = kmin; k0 < kmax; k0 += KEYS) {
        fill(a.k, k0);
        __syncthreads();
        float s[2][4] = {};
#pragma unroll 4
        for (int c = 0; c < a.d; ++c) {
            const float q0 = qs[(2 * ty) * pitch + c], q1 = qs[(2 * ty + 1) * pitch + c];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float k = ks[(tx + 16 * j) * pitch + c];
                s[0][j] = fmaf(q0, k, s[0][j]);
                s[1][j] = fmaf(q1, k, s[1][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int lo = row_lo[2 * ty + i], hi = row_hi[2 * ty + i];
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = k0 + tx + 16 * j;
                s[i][j] = key >= lo && key < hi ? s[i][j] * a.scale : -INFINITY;
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
                ps[(2 * ty + i) * (KEYS + 1) + tx + 16 * j] = p;
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[i] = l[i] * corr + sum;
            m[i] = mn;
#pragma unroll
            for (int j = 0; j < MAX_D / 16; ++j) acc[i][j] *= corr;
        }
        __syncthreads();
        fill(a.v, k0);
        __syncthreads();
        const int keys = min(KEYS, kmax - k0);
        for (int k = 0; k < keys; ++k) {
            const float p0 = ps[(2 * ty) * (KEYS + 1) + k], p1 = ps[(2 * ty + 1) * (KEYS + 1) + k];
#pragma unroll
            for (int j = 0; j < MAX_D / 16; ++j) {
                if (tx + 16 * j >= a.d) break;
                const float v = ks[k * pitch + tx + 16 * j];
                acc[0][j] = fmaf(p0, v, acc[0][j]);
                acc[1][j] = fmaf(p1, v, acc[1][j]);
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
#pragma unroll
        for (int j = 0; j < MAX_D / 16; ++j)
            if (tx + 16 * j < a.d) a.part_o[at * a.d + tx + 16 * j] = acc[i][j] * inv;
    }
}

// ---------------------------------------------------------------------------------------------
// The merge
// ---------------------------------------------------------------------------------------------
// WARPS warps a row, a lane up to four (D <= 128) or eight neighbouring features' worth of each part; the warps take the parts in turn and
// meet in shared memory in their order, so the bits repeat.  Bound by launch and latency: the parts are in L2.
constexpr int MERGE_THREADS = 128;

template <typename T, int WARPS>
__global__ void __launch_bounds__(MERGE_THREADS) prefix_merge_kernel(PrefixMergeArgs a) {
    constexpr int PER = MAX_D / 32, AT_ONCE = MERGE_THREADS / 32 / WARPS;   // rows of a block
    __shared__ float red[AT_ONCE][WARPS][PER + 1][32];
    __shared__ float tops[AT_ONCE][WARPS];
    wait_before();   // the passes
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS, mine = (threadIdx.x >> 5) / WARPS;
    const int64_t row = (int64_t)blockIdx.x * AT_ONCE + mine;
    const bool live = row < a.rows;
    int chunks = 0;
    if (live && a.own.s > 0) {
        int first, len;
        decode_range(a.own, (int)(row / a.hq), first, len);
        chunks = len > first ? (len - first + a.own.chunk - 1) / a.own.chunk : 0;   // those that hold keys
    }
    const int parts = live ? a.splits + chunks : 0;
    auto lse_of = [&](int i) { return i < a.splits ? a.part_lse[i * a.rows + row] : a.own.part_lse[row * a.own.splits + i - a.splits]; };
    float top = -INFINITY;
    for (int i = lane * WARPS + warp; i < parts; i += 32 * WARPS) top = fmaxf(top, lse_of(i));
    top = warp_max(top);
    if constexpr (WARPS > 1) {
        if (lane == 0) tops[mine][warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, tops[mine][w]);
    }
    if (top == -INFINITY) top = 0.f;
    float num[PER], den = 0.f;
#pragma unroll
    for (int c = 0; c < PER; ++c) num[c] = 0.f;
    const bool vec = a.d % 4 == 0;   // features 4 lane + 128 j + (0..3), else lane + 32 j
#pragma unroll 4
    for (int i = warp; i < parts; i += WARPS) {
        const float lse = lse_of(i);
        // A prompt's part that saw no key left nothing.  (A chunk of the sequence's own always left something; a NaN in it is one of the row.)
        if (i < a.splits && lse == -INFINITY) continue;
        const float w = expf(lse - top);
        const float *po = i < a.splits ? a.part_o + (i * a.rows + row) * a.d : a.own.part_o + (row * a.own.splits + i - a.splits) * a.d;
        den += w;
        if (vec) {
#pragma unroll
            for (int j = 0; j < PER / 4; ++j) {
                const int c = 4 * lane + 128 * j;
                if (c >= a.d) break;
                const float4 x = *reinterpret_cast<const float4 *>(po + c);
                num[4 * j] = fmaf(w, x.x, num[4 * j]);
                num[4 * j + 1] = fmaf(w, x.y, num[4 * j + 1]);
                num[4 * j + 2] = fmaf(w, x.z, num[4 * j + 2]);
                num[4 * j + 3] = fmaf(w, x.w, num[4 * j + 3]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (lane + 32 * j >= a.d) break;
                num[j] = fmaf(w, po[lane + 32 * j], num[j]);
            }
        }
    }
    if constexpr (WARPS > 1) {
#pragma unroll
        for (int c = 0; c < PER; ++c) red[mine][warp][c][lane] = num[c];
        red[mine][warp][PER][lane] = den;
        __syncthreads();
        if (warp != 0) return;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
#pragma unroll
            for (int c = 0; c < PER; ++c) num[c] += red[mine][w][c][lane];
            den += red[mine][w][PER][lane];
        }
    }
    if (!live) return;
    const float inv = den != 0.f ? 1.f / den : 0.f;
    T *out = static_cast<T *>(a.out) + row * a.d;
#pragma unroll
    for (int c = 0; c < PER; ++c) {
        const int f = vec ? 4 * lane + 128 * (c / 4) + c % 4 : lane + 32 * c;
        if (f < a.d) out[f] = Num<T>::from_f32(num[c] * inv);
    }
}

template <typename T>
cudaError_t generic_t(const PrefixArgs &a, dim3 grid, cudaStream_t stream) {
    const size_t smem = generic_smem(a.d);
    cudaError_t e = cudaFuncSetAttribute(prefix_generic_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)generic_smem(MAX_D));
    if (e != cudaSuccess) return e;
    prefix_generic_kernel<T><<<grid, THREADS, smem, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t merge_t(const PrefixMergeArgs &a, cudaStream_t stream) {
    // Four warps a row where one would leave multiprocessors idle.
    const bool few = a.rows <= 148 * 16;
    const int at_once = MERGE_THREADS / 32 / (few ? 4 : 1);
    const int64_t blocks = (a.rows + at_once - 1) / at_once;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_beside(few ? prefix_merge_kernel<T, 4> : prefix_merge_kernel<T, 1>, dim3((unsigned)blocks), MERGE_THREADS, 0, stream, true, a);
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

cudaError_t launch_prefix_merge(int dtype, const PrefixMergeArgs &a, cudaStream_t stream, int *launches) {
    *launches += 1;
    switch (dtype) {
        case 0: return merge_t<float>(a, stream);
        case 1: return merge_t<__nv_bfloat16>(a, stream);
        default: return merge_t<__half>(a, stream);
    }
}

}  // namespace dash
