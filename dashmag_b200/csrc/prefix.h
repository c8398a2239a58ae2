// The decoding step of a batch whose sequences share prompts: arguments and launchers (the step itself: dash_attn_decode_shared).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace dash {

// Queries of `n` prompts' sequences, `each` a prompt, against the prompts' keys: parts for the merge.
struct PrefixArgs {
    int n, each, p, hq, hkv, d;
    float scale;
    const void *q;             // [n * each, hq, d]
    int64_t q_sb, q_sh, q_sd;
    View4 k, v;                // [n, p, hkv, d]
    PrefixReach reach;
    int beside;                // 1: beside the launch in front of it, whose end is then this one's too
    int splits;                // runs of a prompt's keys
    float *part_o;             // [splits][n * each, hq, d]
    float *part_lse;           // [splits][n * each, hq], -inf: the part saw no key and left nothing
};

// Parts of prompts and of the sequences' own keys, of one (sequence, query head) each, as one softmax.
struct PrefixMergeArgs {
    int64_t rows;              // n * each * hq
    int hq, d;
    int splits;
    const float *part_o, *part_lse;       // as above
    // The own keys' parts: the chunks of the decoding step's split pass, [rows][own.splits], or (own_splits > 0) runs as above.
    DecodeArgs own;                       // own.s == 0: there are none
    int own_splits;
    void *out;                            // [rows, d] contiguous
};

// The step's new rows into the caches, for a sweep over them (the decoding step's own pass writes them itself).
cudaError_t launch_prefix_append(int dtype, const DecodeArgs &a, cudaStream_t stream, int *launches);
// On the CUDA cores: any dtype, strides and head dimension up to 256.
int prefix_generic_splits(int n, int each, int p, int hq, int hkv);
cudaError_t launch_prefix_generic(int dtype, const PrefixArgs &a, cudaStream_t stream, int *launches);
cudaError_t launch_prefix_merge(int dtype, const PrefixMergeArgs &a, cudaStream_t stream, int *launches);
// On the tensor cores (sm100.cu): whether a call may run there as far as its shape says (0 splits: no), and, its pointers and strides
// allowing, that it does.
// `own_bytes`: what the pass over the sequences' own keys reads beside it.
int sm100_prefix_splits(int dtype, float scale, int n, int each, int p, int hq, int hkv, int d, double own_bytes);
bool sm100_prefix_takes(const PrefixArgs &a);
// False: the driver refused a tensor map.
bool sm100_prefix(int dtype, const PrefixArgs &a, cudaStream_t stream, int *launches, cudaError_t *error);

}  // namespace dash
