/*
 * lamq_b200 training operators — the part of liblamq_b200.so's C ABI that a fine-tuning step around the quantized
 * matrices runs: attention forwards and backwards, the scaled embedding lookup and its gradient, and the Newton-Schulz
 * orthogonalisation of an update. The conventions are lamq_b200.h's: plain device pointers and sizes, asynchronous on
 * the given stream, an int status, buffers and workspaces owned by the caller, nothing allocated by a call.
 * `status` arguments are a device int, 0 at first, that kernels raise to an error code (the greater where there are two).
 * They do not read it: calls may share one, and an error that is still in it affects none of them.
 */
#ifndef LAMQ_B200_TRAIN_H
#define LAMQ_B200_TRAIN_H

#include "lamq_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * out[t] = scale · table[ids[t]] for t < n: rows of d values (table: rows x d, leading dimension ldt; out: n x d, ldo;
 * dtype LAMQ_F32 or LAMQ_BF16, the product in fp32 rounded once). ids are int64 (ids64 != 0) or int32. A token with
 * id == padding (-1: none) gets a zero row; an id outside [0, rows) gets a zero row and sets *status to
 * LAMQ_ERR_INVALID. Any d and alignment; rows that are 16-byte aligned move in 16-byte pieces.
 */
int lamq_embedding_lookup(const void *table, int dtype, int64_t ldt, int64_t rows, int d, const void *ids, int ids64,
                          int64_t n, float scale, int64_t padding, void *out, int64_t ldo, int *status,
                          lamq_stream_t stream);

/*
 * The lookup's gradient: dE[v] = scale · Σ_{t: ids[t] = v} dy[t] for every v < rows (dE: rows x d, lde, of dy's dtype),
 * or dE[v] += that with accumulate != 0 (rows without a token are then left alone). Tokens with id == padding or an
 * invalid id (which sets *status to LAMQ_ERR_INVALID) add nothing. Sums are fp32 in the order of the tokens (above 2048
 * tokens, within fixed chunks of the sorted tokens, then chunk by chunk): equal calls give equal bits. Workspace:
 * lamq_embedding_gradient_workspace_size(n, d) bytes, 16-byte aligned (0, and NULL allowed, up to 2048 tokens). *status
 * becomes LAMQ_ERR_TIMEOUT if a bounded device wait gives up: no sums are written then.
 */
size_t lamq_embedding_gradient_workspace_size(int64_t n, int d);
int lamq_embedding_gradient(const void *dy, int dtype, int64_t ldy, const void *ids, int ids64, int64_t n, int64_t rows,
                            int d, float scale, int64_t padding, int accumulate, void *dE, int64_t lde, void *workspace,
                            size_t workspace_bytes, int *status, lamq_stream_t stream);

/*
 * A (batch, heads, length, head_dim) bf16 tensor: its first element (16-byte aligned) and the strides in elements of
 * the first three axes (positive multiples of 8 where the axis has more than one entry; head_dim is contiguous).
 */
typedef struct lamq_heads {
    void *data;
    int64_t batch, head, row;
} lamq_heads;

/*
 * The operands of an attention call. Query head h reads key head h / (heads / kv_heads). Query i of text b sees the
 * keys j with key_start[b] <= j < key_end[b] (device int32 arrays of `batch` entries, clamped to [0, kv_len); NULL:
 * from 0, to kv_len) and, with causal != 0, j <= i + kv_len − q_len (the last query sees the last key). head_dim is a
 * multiple of 8 up to 128; lengths are arbitrary, zero included. q, k, v: read. o and lse (batch x heads x q_len fp32,
 * contiguous): written by the forward, read by the backward. d_o is read and dq, dk, dv are written by the backward
 * only. Outputs are written whole (with no query heads at all nothing is: the call is a no-op) and overlap no input.
 * 328 bytes, no padding (`reserved` is ignored).
 */
typedef struct lamq_attention_args {
    int64_t batch;
    int heads, kv_heads, head_dim, causal;
    int64_t q_len, kv_len;
    float scale;
    int reserved;
    const int32_t *key_start, *key_end;
    lamq_heads q, k, v, o;
    float *lse;
    lamq_heads d_o, dq, dk, dv;
} lamq_attention_args;

/*
 * o = softmax(scale·q·kᵀ)·v over each query's allowed keys (bf16, the softmax in fp32) and lse, the natural logarithm
 * of the sum of exponentials. A query without a key gets o = 0 and lse = −inf. Keys outside a text's range are not
 * used, whatever they hold; a NaN or infinity inside it spreads to the queries of its tile, as in a matrix product.
 * *status becomes LAMQ_ERR_TIMEOUT if a bounded device wait gives up. `args` is host memory, read before the call
 * returns.
 */
int lamq_attention_forward(const lamq_attention_args *args, int *status, lamq_stream_t stream);

/*
 * The gradients of lamq_attention_forward from d_o, recomputing the probabilities from q, k and lse (o and lse as the
 * forward wrote them): dq, dk, dv (bf16, summed in fp32; a key head's gradient is the sum over its query heads).
 * Queries without a key get a zero gradient and add none, whatever their rows of q and d_o hold; keys that no query
 * sees get zeros. Every sum has a fixed order: equal calls give equal bits. Workspace:
 * lamq_attention_backward_workspace_size(batch, heads, q_len) bytes, 16-byte aligned.
 */
size_t lamq_attention_backward_workspace_size(int64_t batch, int heads, int64_t q_len);
int lamq_attention_backward(const lamq_attention_args *args, void *workspace, size_t workspace_bytes, int *status,
                            lamq_stream_t stream);

/*
 * The orthogonalised update of each of `batch` matrices G (m x n, leading dimension ldg, batch_stride elements apart;
 * dtype LAMQ_F32 or LAMQ_BF16): X = G / (|G|_F + eps), then for each of `steps` (1..16) steps, with (a, b, c) the
 * step's coefficients (host memory, 3·steps floats, read before the call returns), X <- (aI + bA + cA²)·X, A = X·Xᵀ
 * (on the smaller side of G: for m > n, X <- X·(aI + bA + cA²), A = Xᵀ·X). out: batch x m x n bf16, contiguous.
 * X, A and B are held in 22 bits, products take fp16 operands where their rounding cannot grow, fp16 pairs elsewhere,
 * with fp32 accumulation: the relative error is about the bf16 output's rounding (2^-9) again. (Coefficients whose steps are
 * steeper than 9 anywhere take pairs everywhere, 2.6 times the work.) Coefficients that take singular values of [0, 1]
 * above 5, or the polynomial of A above 32, are rejected. A zero matrix gives zeros; a matrix with a NaN or an infinity
 * gives NaN. Workspace: lamq_newton_schulz_workspace_size(batch, m, n) bytes, 16-byte aligned. One cooperative kernel; *status becomes
 * LAMQ_ERR_TIMEOUT if a bounded device wait gives up. Equal calls give equal bits.
 */
size_t lamq_newton_schulz_workspace_size(int batch, int m, int n);
int lamq_newton_schulz(const void *G, int dtype, int64_t ldg, int64_t batch_stride, int batch, int m, int n, int steps,
                       const float *coefficients, float eps, uint16_t *out, void *workspace, size_t workspace_bytes,
                       int *status, lamq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* LAMQ_B200_TRAIN_H */
