// The norms' backward call: its plan, the kernels for aligned rows (norm_backward.cuh), and the sums of the partial rows.
#include "norm_backward.cuh"

namespace lamq {
namespace {

// How the rows are dealt out, and what a call's workspace holds: partial rows of d_weight, d_post and d_gate.
struct Plan {
    NormLayout layout;
    int per, grid, gate_mode, columns;
    int64_t g_rows;
    size_t w_at, u_at, g_at, bytes;
};

Plan plan_of(const lamq_norm_args &a) {
    Plan q{};
    q.layout = norm_layout(a, true, a.d_weight || a.d_post || a.d_gate, a.d_gate);
    const NormShape &shape = q.layout.shape;
    const int slots = q.layout.slots;
    const int64_t most = (int64_t)kSMs * q.layout.blocks * slots;  // workers
    int64_t per = std::max<int64_t>(1, (a.rows + most - 1) / most);
    q.gate_mode = kGateNone;
    if (a.d_gate) {
        if (a.gate_span == a.rows && a.rows > 1) {
            q.gate_mode = kGateOne;
        } else if (a.gate_span == 1) {
            q.gate_mode = kGateInside;
        } else if (a.gate_span <= per) {
            q.gate_mode = kGateInside;
            per = (per + a.gate_span - 1) / a.gate_span * a.gate_span;
        } else {
            q.gate_mode = kGateAcross;
        }
    }
    q.per = (int)per;
    const int64_t workers = (a.rows + per - 1) / per;
    q.grid = (int)((workers + slots - 1) / slots);
    q.columns = (a.d + 7) / 8 * 8;
    // the wide kernels sum every gate row in memory: one row for each block, where no worker shares a gate row
    const bool block_rows = q.gate_mode == kGateOne || (q.gate_mode == kGateInside && shape.kernel == kWide && a.gate_span > 1);
    q.g_rows = block_rows ? q.grid : q.gate_mode == kGateAcross ? (int64_t)q.grid * slots + a.rows / a.gate_span : 0;
    const size_t row = (size_t)q.columns * sizeof(float);
    q.w_at = 0;
    q.u_at = q.w_at + (a.d_weight ? (size_t)q.grid * row : 0);
    q.g_at = q.u_at + (a.d_post ? (size_t)q.grid * row : 0);
    q.bytes = q.g_at + (size_t)q.g_rows * row;
    return q;
}

// Each output row is the sum of some partial rows: a block adds 32 columns of them, its warps every 32nd row in order, then
// the warps in order. Bound by the latency of its few loads, which are all on their way at once for up to 512 rows.
struct ReduceParams {
    const float *w_part, *u_part, *g_part;
    void *d_weight, *d_post, *d_gate;
    int weight_dtype, post_dtype, gate_dtype;
    int d, columns, grid;
    int gate_one, gate_span, per;
};

constexpr int kReduceWarps = 32;

__global__ void __launch_bounds__(kReduceWarps * 32) norm_reduce_kernel(const __grid_constant__ ReduceParams p) {
    __shared__ float sums[kReduceWarps][32];
    await_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int blocks = (p.d + 31) / 32;  // of 32 columns each
    int job = blockIdx.x / blocks;
    const int col = (blockIdx.x - job * blocks) * 32 + lane;
    const float *part;
    void *dst;
    int dtype, count = p.grid;
    int64_t at = 0;
    if (p.d_weight && job-- == 0) {
        part = p.w_part, dst = p.d_weight, dtype = p.weight_dtype;
    } else if (p.d_post && job-- == 0) {
        part = p.u_part, dst = p.d_post, dtype = p.post_dtype;
    } else {
        part = p.g_part, dst = p.d_gate, dtype = p.gate_dtype;
        if (!p.gate_one) {  // gate row `job`: of the workers that hold rows of it
            const int64_t r0 = (int64_t)job * p.gate_span;
            const int64_t k0 = r0 / p.per, k1 = (r0 + p.gate_span - 1) / p.per;
            part += (k0 + job) * p.columns;
            count = (int)(k1 - k0 + 1);
            at = (int64_t)job * p.d;
        }
    }
    float s = 0.f;
    if (col < p.d) {
        const float *src = part + col;
#pragma unroll 16
        for (int k = warp; k < count; k += kReduceWarps) s += __ldcg(src + (int64_t)k * p.columns);
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || col >= p.d) return;
    for (int w = 1; w < kReduceWarps; ++w) s += sums[w][lane];
    const float one[1] = {s};
    store_typed<1>(dst, dtype, at + col, one);
}

}  // namespace
}  // namespace lamq

using namespace lamq;

extern "C" size_t lamq_norm_backward_workspace_size(const lamq_norm_args *a) {
    if (norm_args_status(a, true) != LAMQ_OK || a->rows == 0 || a->d == 0) return 0;
    return plan_of(*a).bytes;
}

extern "C" int lamq_norm_backward(const lamq_norm_args *a, void *workspace, size_t workspace_bytes, lamq_stream_t stream) {
    if (const int st = norm_args_status(a, true)) return st;
    if (a->rows == 0 || a->d == 0) return LAMQ_OK;
    const Plan q = plan_of(*a);
    LAMQ_REQUIRE(workspace_bytes >= q.bytes, "a workspace of %zu bytes is needed", q.bytes);
    LAMQ_REQUIRE(q.bytes == 0 || workspace, "null pointer (workspace)");
    LAMQ_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 31) == 0, "the workspace must be 32-byte aligned");
    const NormLayout &l = q.layout;
    const int mode = l.mode;
    const bool sums = a->d_weight || a->d_post || a->d_gate;
    BackwardParams p;
    p.in = present(*a, true);
    p.d_residual = a->d_residual, p.d_branch = a->d_branch, p.d_gate = a->d_gate;
    char *const ws = reinterpret_cast<char *>(workspace);
    p.w_part = a->d_weight ? reinterpret_cast<float *>(ws + q.w_at) : nullptr;
    p.u_part = a->d_post ? reinterpret_cast<float *>(ws + q.u_at) : nullptr;
    p.g_part = q.g_rows ? reinterpret_cast<float *>(ws + q.g_at) : nullptr;
    p.rows = (int)a->rows, p.d = a->d;
    p.scale = a->scale, p.eps = a->eps, p.offset = a->offset, p.inv_d = 1.f / (float)a->d;
    p.team = l.shape.team, p.slots = l.slots, p.packs = l.shape.packs, p.columns = q.columns;
    p.per = q.per, p.gate_mode = q.gate_mode;
    const cudaStream_t st = (cudaStream_t)stream;
    p.ring = l.ring;
    p.sums_at = l.ring.ring_bytes;
    const int shared = l.shared;
    const NormKernel kernel = l.shape.kernel;
    const int launched = kernel == kVectors       ? launch_backward<kVectors>(*a, p, q.grid, mode, sums, shared, st)
                         : kernel == kVectors8    ? launch_backward<kVectors8>(*a, p, q.grid, mode, sums, shared, st)
                         : kernel == kVectorsWide ? launch_backward<kVectorsWide>(*a, p, q.grid, mode, sums, shared, st)
                         : kernel == kVectorsWidest
                             ? launch_backward<kVectorsWidest>(*a, p, q.grid, mode, sums, shared, st)
                             : launch_backward_elements(kernel, *a, &p, q.grid, mode, sums, shared, st);
    if (launched) return launched;
    LAMQ_CHECK_LAUNCH("lamq_norm_backward");
    if (!q.bytes) return LAMQ_OK;
    const bool gates = q.gate_mode == kGateOne || q.gate_mode == kGateAcross;
    ReduceParams sum;
    sum.w_part = p.w_part, sum.u_part = p.u_part, sum.g_part = p.g_part;
    sum.d_weight = a->d_weight, sum.d_post = a->d_post, sum.d_gate = gates ? a->d_gate : nullptr;
    sum.weight_dtype = a->weight_dtype, sum.post_dtype = a->post_dtype, sum.gate_dtype = a->gate_dtype;
    sum.d = a->d, sum.columns = q.columns, sum.grid = q.grid;
    sum.gate_one = q.gate_mode == kGateOne, sum.gate_span = p.in.gate_span, sum.per = q.per;
    const int64_t jobs = (a->d_weight ? 1 : 0) + (a->d_post ? 1 : 0) +
                         (q.gate_mode == kGateOne ? 1 : q.gate_mode == kGateAcross ? a->rows / a->gate_span : 0);
    if (jobs == 0) return LAMQ_OK;
    launch_following(norm_reduce_kernel, (unsigned)(jobs * ((a->d + 31) / 32)), kReduceWarps * 32, st, sum);
    LAMQ_CHECK_LAUNCH("lamq_norm_backward (sums)");
    return LAMQ_OK;
}
