/*
 * lamq_b200 training operators — the part of liblamq_b200.so's C ABI that a fine-tuning step around the quantized
 * matrices runs: attention forwards and backwards, the scaled embedding lookup and its gradient, and the Newton-Schulz
 * orthogonalisation of an update. The conventions are lamq_b200.h's: plain device pointers and sizes, asynchronous on
 * the given stream, an int status, buffers and workspaces owned by the caller, nothing allocated by a call.
 * `status` arguments are a device int, 0 before the call, that a kernel sets to an error code.
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
 * invalid id (which sets *status to LAMQ_ERR_INVALID) add nothing. Sums are fp32 in the order of the tokens within
 * fixed chunks of the sorted tokens: equal calls give equal bits. Workspace:
 * lamq_embedding_gradient_workspace_size(n, d) bytes, 16-byte aligned.
 */
size_t lamq_embedding_gradient_workspace_size(int64_t n, int d);
int lamq_embedding_gradient(const void *dy, int dtype, int64_t ldy, const void *ids, int ids64, int64_t n, int64_t rows,
                            int d, float scale, int64_t padding, int accumulate, void *dE, int64_t lde, void *workspace,
                            size_t workspace_bytes, int *status, lamq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* LAMQ_B200_TRAIN_H */
