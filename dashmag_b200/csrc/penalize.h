// The rules a server puts on a step's logits: arguments and launcher.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dash {

struct PenalizeArgs {
    const void *logits;       // [b, v], rows `stride` elements apart, the vocabulary contiguous
    void *out;                // the same with rows `out_stride` apart; may be the logits themselves
    int b, v;
    int64_t stride, out_stride;
    const void *ids;          // [b, t] i32 / i64, rows `ids_stride` apart, or null: no history
    int t, ids_bytes;
    int64_t ids_stride;
    const void *lengths;      // [b] i32 / i64: ids held by each row; null: t
    const void *prompt;       // [b] i32 / i64: how many of them are the prompt's; null: 0
    int lengths_bytes, prompt_bytes;
    const float *repetition, *frequency, *presence;   // [b], or null: the value beside it for every row
    float repetition_all, frequency_all, presence_all;
    const void *bias;         // [b, v] or null; rows `bias_stride` apart (0: one row for all)
    int bias_f32;             // f32, else the logits' dtype
    int64_t bias_stride;
    const uint32_t *allowed;  // [b, ceil(v / 32)] or null; bit v % 32 of word v / 32 set: token v may come; rows `allowed_stride` words apart
    int64_t allowed_stride;
};

cudaError_t launch_penalize(int dtype, const PenalizeArgs &a, cudaStream_t stream, int *launches);

}  // namespace dash
