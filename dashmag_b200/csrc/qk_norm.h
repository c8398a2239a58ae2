// The norm of every query and key head with the position rotation in the same pass: arguments and launchers.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dash {

// One tensor [b, t, heads, d] (strides in elements, the features contiguous) and what goes with it; everything written is contiguous.
struct NormTensor {
    const void *x;
    int64_t sb, st, sh;
    const void *g;         // backward: the gradient of the normed and rotated tensor
    int64_t gb, gt, gh;
    void *out;             // forward: the result; backward: the gradient of x
    const void *w;         // [d], null: ones
    void *dw;              // backward: the weight's gradient, null: not wanted
    int heads;
};

struct Over { uint32_t mul; int shift; };   // a division by a known number, as a multiplication

struct NormArgs {
    NormTensor q, k;       // k.heads == 0: one tensor only.  Both share the tokens' positions.
    int b;
    int64_t t;             // tokens of a batch element; token n is (n / t, n % t)
    int d, dim;            // the first `dim` features of a head are rotated
    float eps;
    int w_f32;             // the weights (and their gradients) are f32, else the tensors' dtype
    const void *cos, *sin; // [len, dim], the tensors' dtype
    int64_t len;
    // The position of token n, first rule that applies:
    const void *positions; // [b * t] i32 / i64
    int pos_bytes;
    const void *cu;        // [sequences + 1] i32 / i64: start + n - cu[s] for cu[s] <= n < cu[s + 1]
    int cu_bytes, sequences;
    int64_t start;         // start + n % t
    Over over_t;           // set by the launchers
    float *part;           // backward scratch: a row of d sums per block
};

// Floats of backward scratch.
size_t qk_norm_part_floats(int d);
cudaError_t launch_qk_norm(int dtype, const NormArgs &a, cudaStream_t stream, int *launches);
cudaError_t launch_qk_norm_backward(int dtype, const NormArgs &a, cudaStream_t stream, int *launches);

// The sticky device word that a bounded wait of these kernels raises when it runs out.
cudaError_t read_qk_norm_status(unsigned int *status, bool clear);

}  // namespace dash
