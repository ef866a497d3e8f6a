// The norms' backward kernels for rows that may begin anywhere, an element at a time: by teams (norm_backward.cuh), and, for
// wide rows, by blocks (norm_wide.cuh).
#include "norm_backward.cuh"

namespace lamq {
namespace {

template <typename R, typename B>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(const __grid_constant__ BackwardParams p, int mode) {
    extern __shared__ float row_of_t[];  // the gradient that comes to the post norm
    __shared__ float scratch[3 * 32];
    let_follow();
    const int64_t block_row = (int64_t)blockIdx.x * p.columns;
    const bool full = mode == kJoinFull, pre = p.in.has & kHasDy, post = full && (p.in.has & kHasPost),
               gate = full && (p.in.has & kHasGate), gate_sums = full && p.gate_mode != kGateNone;
    wide_each(p.d, [&](int j) {
        if (p.w_part) p.w_part[block_row + j] = 0.f;
        if (p.u_part) p.u_part[block_row + j] = 0.f;
    });
    const int first = blockIdx.x * p.per, end = min(p.rows, first + p.per);
    for (int row = first; row < end; ++row) {
        const int64_t out = (int64_t)row * p.d;
        const R *const h = row_at<R>(p.in.h, row), *const dh = row_at<R>(p.in.dh, row);
        const B *const dy = row_at<B>(p.in.dy, row), *const branch = row_at<B>(p.in.branch, row);
        const auto weight = [&](int j) { return p.offset + value_at(p.in.weight, p.in.weight_dtype, j); };
        const auto after = [&](int j) { return p.offset + value_at(p.in.post, p.in.post_dtype, j); };
        float s[3] = {0.f, 0.f, 0.f};  // Σ h², Σ t h, Σ b²
        wide_each(p.d, [&](int j) {
            if (pre) {
                const float x = load_one(h + j);
                s[0] = fmaf(x, x, s[0]);
                s[1] = fmaf(load_one(dy + j) * weight(j), x, s[1]);
            }
            if (post) {
                const float b = load_one(branch + j);
                s[2] = fmaf(b, b, s[2]);
            }
        });
        if (pre || post) wide_sum(s, scratch);
        float f = 0.f, shrunk = 1.f, fb = 1.f, less = 1.f, c = 0.f;
        if (pre) {
            f = wide_factor(s[0], p.d, [&](int j) { return load_one(h + j); }, p.inv_d, p.eps, shrunk, scratch);
            c = s[1] * f;
            if (sums_lost(s[0], s[1], p.eps)) {
                float unit[1] = {0.f};
                wide_each(p.d, [&](int j) { unit[0] = fmaf(load_one(dy + j) * weight(j), load_one(h + j) * shrunk * f, unit[0]); });
                wide_sum(unit, scratch);
                c = unit[0];
            }
            c *= p.inv_d;
        }
        if (post) fb = wide_factor(s[2], p.d, [&](int j) { return load_one(branch + j); }, p.inv_d, p.eps, less, scratch);
        const float r = f * shrunk;
        const int gate_row = p.in.by_span.of(row);
        // a gate row is summed in the block's partial row, one that spans blocks in the pair's
        const bool begins = row == first || (p.gate_mode != kGateOne && row == gate_row * p.in.gate_span);
        const bool done = p.gate_mode == kGateInside && row + 1 == (gate_row + 1) * p.in.gate_span;
        float *const part = p.g_part + (p.gate_mode == kGateAcross ? (int64_t)blockIdx.x + gate_row : (int64_t)blockIdx.x) * p.columns;
        float cb[1] = {0.f};
        wide_each(p.d, [&](int j) {
            float g[1] = {(p.in.has & kHasDh) ? load_one(dh + j) : 0.f};
            if (pre) {
                const float unit = load_one(h + j) * shrunk * f, y = load_one(dy + j);
                g[0] = fmaf(r, fmaf(-unit, c, y * weight(j)), g[0]);
                if (p.w_part) p.w_part[block_row + j] = fmaf(y, unit, own_at(p.w_part + block_row + j));
            }
            Raw<R, 1>::store(reinterpret_cast<R *>(p.d_residual) + out + j, g);
            float t[1] = {g[0] * p.scale};
            if (full) {
                const float b = post || gate_sums ? load_one(branch + j) * less * fb : 0.f, u = post ? after(j) : 1.f;
                if (gate_sums) {
                    float to[1] = {t[0] * (b * u)};
                    if (!begins) to[0] += own_at(part + j);
                    if (done)
                        store_typed<1>(p.d_gate, p.in.gate_dtype, (int64_t)gate_row * p.d + j, to);
                    else
                        part[j] = to[0];
                }
                if (gate) t[0] *= value_at(p.in.gate, p.in.gate_dtype, (int64_t)gate_row * p.d + j);
                if (post) {
                    if (p.u_part) p.u_part[block_row + j] = fmaf(t[0], b, own_at(p.u_part + block_row + j));
                    t[0] *= u;
                    cb[0] = fmaf(t[0], b, cb[0]);
                    row_of_t[j] = t[0];
                }
            }
            if (p.d_branch && !post) Raw<B, 1>::store(reinterpret_cast<B *>(p.d_branch) + out + j, t);
        });
        if (!post) continue;
        wide_sum(cb, scratch);
        cb[0] *= p.inv_d;
        if (p.d_branch)
            wide_each(p.d, [&](int j) {
                const float t[1] = {fb * less * fmaf(-load_one(branch + j) * less * fb, cb[0], row_of_t[j])};
                Raw<B, 1>::store(reinterpret_cast<B *>(p.d_branch) + out + j, t);
            });
    }
}

template <typename R, typename B>
int launch_wide(const BackwardParams &p, int grid, int mode, int shared, cudaStream_t stream) {
    const auto kernel = norm_backward_wide_kernel<R, B>;
    if (const int st = allow_shared(reinterpret_cast<const void *>(kernel), shared)) return st;
    kernel<<<grid, kWideThreads, shared, stream>>>(p, mode);
    return LAMQ_OK;
}

int launch_wide(const lamq_norm_args &a, const BackwardParams &p, int grid, int mode, int shared, cudaStream_t stream) {
    if (a.residual_dtype == LAMQ_BF16) return launch_wide<__nv_bfloat16, __nv_bfloat16>(p, grid, mode, shared, stream);
    if (a.branch_dtype == LAMQ_BF16) return launch_wide<float, __nv_bfloat16>(p, grid, mode, shared, stream);
    return launch_wide<float, float>(p, grid, mode, shared, stream);
}

}  // namespace

int launch_backward_elements(int kernel, const lamq_norm_args &a, const void *params, int grid, int mode, bool sums, int shared,
                             cudaStream_t stream) {
    const BackwardParams &p = *reinterpret_cast<const BackwardParams *>(params);
    return kernel == kElements    ? launch_backward<kElements>(a, p, grid, mode, sums, shared, stream)
           : kernel == kElements8 ? launch_backward<kElements8>(a, p, grid, mode, sums, shared, stream)
                                  : launch_wide(a, p, grid, mode, shared, stream);
}

}  // namespace lamq
