/*
 * lamq_b200 step operators — the part of liblamq_b200.so's C ABI that a training step runs around its blocks and after its
 * backward pass: the norms before and after a block joined with the block's gate, its scale and the residual addition,
 * and the global norm of many gradients with its clipping. The conventions are lamq_b200.h's: plain device pointers and
 * sizes, asynchronous on the given stream, an int status, buffers and workspaces owned by the caller, nothing allocated
 * by a call. Pointers lie at a multiple of their element's size. No kernel waits on another block, so there are no status words.
 */
#ifndef LAMQ_B200_STEP_H
#define LAMQ_B200_STEP_H

#include "lamq_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows of d contiguous elements: row i begins (i / inner)·outer + (i % inner)·row elements behind `data` (the heads of a
 * projection's output have an inner count; plain matrices have inner >= their number of rows, and so have a join's).
 */
typedef struct lamq_rows {
    void *data;
    int64_t inner, row, outer;
} lamq_rows;

/*
 * A block's end: with N(x; w) = x · (mean(x²) + eps)^-1/2 · (offset + w), over `rows` rows of d (1..16384) elements
 *
 *   p = N(branch; post), or branch where post is NULL
 *   h = residual + scale · gate ⊙ p          (gate NULL: 1; row i uses gate row i / gate_span, gate rows are contiguous)
 *   y = N(h; weight)                         (weight NULL: no y)
 *
 * or, where branch.data is NULL, the norm alone: y = N(residual; weight), no h.
 * residual, h and their gradients have residual_dtype; branch, y and theirs branch_dtype; weight, post and gate types of
 * their own, which their gradients share. Types are LAMQ_F32 and LAMQ_BF16; a bf16 residual takes bf16 branches only.
 * All sums are fp32 and results are rounded once (y comes from the unrounded h). Outputs (h, y and the gradients) are
 * contiguous rows x d and overlap no input. Rows that do not begin and end on 16 bytes are read in the aligned 16-byte pieces that
 * hold them: up to 14 bytes in front of a tensor's first row and behind its last come along, are not used, and may change
 * meanwhile. A suballocator that lets tensors begin anywhere needs a pool of whole 16-byte pieces (cudaMalloc's are).
 * 264 bytes, no padding (`reserved` is ignored).
 */
typedef struct lamq_norm_args {
    int64_t rows, gate_span;
    int d, residual_dtype, branch_dtype, weight_dtype, post_dtype, gate_dtype;
    float scale, eps, offset;
    int reserved;
    lamq_rows residual, branch;
    const void *weight, *post, *gate;
    void *h, *y;
    lamq_rows dh, dy;
    void *d_residual, *d_branch, *d_weight, *d_post, *d_gate;
} lamq_norm_args;

/* Writes h and y; nothing where there are no rows or no elements. `args` is host memory, read before the call returns (here and
 * below). */
int lamq_norm_forward(const lamq_norm_args *args, lamq_stream_t stream);

/*
 * The gradients, from dh and dy (data NULL: zero; the norm alone has a dy) and from `residual`, which here holds the forward's
 * h (the norm alone: its input), the statistics being computed again. d_residual is always written (whoever wants the others alone
 * pays for it, too); d_branch (NULL: not wanted, as where it equals d_residual), d_weight, d_post and d_gate where they are not
 * NULL. The gradient of a weight or of a shared gate is
 * summed in fp32 in a fixed order: equal calls give equal bits. Workspace: lamq_norm_backward_workspace_size(args) bytes,
 * 32-byte aligned (0 where no such sum is wanted).
 */
size_t lamq_norm_backward_workspace_size(const lamq_norm_args *args);
int lamq_norm_backward(const lamq_norm_args *args, void *workspace, size_t workspace_bytes, lamq_stream_t stream);

/*
 * One tensor of a list: n contiguous elements of dtype (LAMQ_F32 or LAMQ_BF16), and where its clipped values go
 * (out_dtype; data itself, in its own type, to clip in place). 32 bytes, no padding.
 */
typedef struct lamq_gradient {
    void *data, *out;
    int64_t n;
    int dtype, out_dtype;
} lamq_gradient;

/*
 * *norm (fp32) = the square root of the sum of squares over all `count` tensors (host array, read before the call
 * returns). Squares are summed in fp64 where fp32 could lose or overflow, in a fixed order. Workspace:
 * lamq_gradient_workspace_size(count) bytes, 8-byte aligned.
 */
size_t lamq_gradient_workspace_size(int64_t count);
int lamq_gradient_norm(const lamq_gradient *list, int64_t count, float *norm, void *workspace, size_t workspace_bytes,
                       lamq_stream_t stream);

/*
 * The same, and out = data · min(1, max_norm / (norm + eps)), the factor in fp64. Tensors that are clipped in place are
 * not written where the factor is 1; a norm of NaN gives NaN everywhere, an infinite one zeros (NaN where an element is
 * infinite). No two tensors of the list may share memory, nor an `out` any memory but its own `data`.
 */
int lamq_gradient_clip(const lamq_gradient *list, int64_t count, double max_norm, double eps, float *norm, void *workspace,
                       size_t workspace_bytes, lamq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* LAMQ_B200_STEP_H */
