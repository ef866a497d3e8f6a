// The norms' backward kernels for rows that may begin anywhere, an element at a time: by teams (norm_backward.cuh), and, for
// more than 4096 of them, by blocks (norm_wide.cuh).
#include "norm_backward.cuh"

namespace lamq {
namespace {

template <typename R, typename B>
__global__ void __launch_bounds__(kWideThreads, 1) norm_backward_wide_kernel(const __grid_constant__ BackwardParams p, int mode) {
    __shared__ alignas(16) float scratch[Team::kScratch];
    let_follow();
    Team team(kWideThreads, scratch);
    const int64_t block_row = (int64_t)blockIdx.x * p.columns;
    const bool full = mode == kJoinFull;
    for (int j = threadIdx.x; j < p.d; j += kWideThreads) {
        if (p.w_part) p.w_part[block_row + j] = 0.f;
        if (p.u_part) p.u_part[block_row + j] = 0.f;
    }
    const int first = blockIdx.x * p.per, end = min(p.rows, first + p.per);
    for (int row = first; row < end; ++row) {
        const int64_t out = (int64_t)row * p.d;
        const R *const h = row_at<R>(p.in.h, row), *const dh = row_at<R>(p.in.dh, row);
        const B *const dy = row_at<B>(p.in.dy, row), *const branch = row_at<B>(p.in.branch, row);
        const bool pre = (p.in.has & kHasDy);
        float f = 0.f, shrunk = 1.f, r = 0.f, c = 0.f;
        const auto t = [&](int j) { return load_one(dy + j) * (p.offset + value_at(p.in.weight, p.in.weight_dtype, j)); };
        const auto unit = [&](int j) { return load_one(h + j) * shrunk * f; };
        if (pre) {
            f = wide_factor(team, p.d, [&](int j) { return load_one(h + j); }, p.inv_d, p.eps, shrunk);
            r = f * shrunk;
            c = wide_sum(team, p.d, [&](int j) { return t(j) * unit(j); }) * p.inv_d;
        }
        const auto g = [&](int j) {
            const float x = (p.in.has & kHasDh) ? load_one(dh + j) : 0.f;
            return pre ? fmaf(r, fmaf(-unit(j), c, t(j)), x) : x;
        };
        for (int j = threadIdx.x; j < p.d; j += kWideThreads) {
            const float x[1] = {g(j)};
            Raw<R, 1>::store(reinterpret_cast<R *>(p.d_residual) + out + j, x);
            if (p.w_part && pre) p.w_part[block_row + j] = fmaf(load_one(dy + j), unit(j), p.w_part[block_row + j]);
        }
        if (mode == kNormAlone || (!p.d_branch && !full)) continue;
        const int64_t gate_row = row / p.in.gate_span;
        float fb = 1.f, less = 1.f, cb = 0.f;
        if (full && (p.in.has & kHasPost))
            fb = wide_factor(team, p.d, [&](int j) { return load_one(branch + j); }, p.inv_d, p.eps, less);
        const auto b = [&](int j) { return load_one(branch + j) * less * fb; };
        const auto u = [&](int j) { return p.offset + value_at(p.in.post, p.in.post_dtype, j); };
        const auto back = [&](int j) {
            const float x = p.scale * g(j);
            return full && (p.in.has & kHasGate) ? x * value_at(p.in.gate, p.in.gate_dtype, gate_row * p.d + j) : x;
        };
        if (full && p.gate_mode != kGateNone) {
            // one gate row for all: the block's partial row; else the pair's (a gate row of its own: written at once)
            const bool begins = row == first || (p.gate_mode != kGateOne && row % p.in.gate_span == 0);
            float *const part = p.g_part + (p.gate_mode == kGateOne ? (int64_t)blockIdx.x : blockIdx.x + gate_row) * p.columns;
            for (int j = threadIdx.x; j < p.d; j += kWideThreads) {
                const float x[1] = {p.scale * g(j) * (p.in.has & kHasPost ? b(j) * u(j) : b(j))};
                if (p.gate_mode == kGateInside)
                    store_typed<1>(p.d_gate, p.in.gate_dtype, gate_row * p.d + j, x);
                else
                    part[j] = begins ? x[0] : part[j] + x[0];
            }
        }
        if (full && (p.in.has & kHasPost)) cb = wide_sum(team, p.d, [&](int j) { return back(j) * u(j) * b(j); }) * p.inv_d;
        for (int j = threadIdx.x; j < p.d; j += kWideThreads) {
            float x[1] = {back(j)};
            if (full && (p.in.has & kHasPost)) {
                if (p.u_part) p.u_part[block_row + j] = fmaf(x[0], b(j), p.u_part[block_row + j]);
                x[0] = fb * less * fmaf(-b(j), cb, x[0] * u(j));
            }
            if (p.d_branch) Raw<B, 1>::store(reinterpret_cast<B *>(p.d_branch) + out + j, x);
        }
    }
}

int launch_wide(const lamq_norm_args &a, const BackwardParams &p, int grid, int mode, cudaStream_t stream) {
    if (a.residual_dtype == LAMQ_BF16)
        norm_backward_wide_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, kWideThreads, 0, stream>>>(p, mode);
    else if (a.branch_dtype == LAMQ_BF16)
        norm_backward_wide_kernel<float, __nv_bfloat16><<<grid, kWideThreads, 0, stream>>>(p, mode);
    else
        norm_backward_wide_kernel<float, float><<<grid, kWideThreads, 0, stream>>>(p, mode);
    return LAMQ_OK;
}

}  // namespace

int launch_backward_elements(int kernel, const lamq_norm_args &a, const void *params, int grid, int mode, bool sums, int shared,
                             cudaStream_t stream) {
    const BackwardParams &p = *reinterpret_cast<const BackwardParams *>(params);
    return kernel == kElements    ? launch_backward<kElements>(a, p, grid, mode, sums, shared, stream)
           : kernel == kElements8 ? launch_backward<kElements8>(a, p, grid, mode, sums, shared, stream)
                                  : launch_wide(a, p, grid, mode, stream);
}

}  // namespace lamq
