// The norms before and after a block, joined with the block's gate, its scale and the residual addition, forwards:
//
//   p = N(branch; post) or branch,   h = residual + scale · gate ⊙ p,   y = N(h; weight)
//   N(x; w) = x · (mean(x²) + eps)^-1/2 · (offset + w)
//
// and N(x; w) alone. Bound by memory: each row is read once into registers and written once; a norm is one exchange among
// the row's threads. y is made from h in fp32, before h is rounded to its type: one rounding fewer than a norm that reads
// the stored h.
#include "norm_wide.cuh"

namespace lamq {
namespace {

struct ForwardParams {
    lamq_rows residual;
    Present in;
    void *h, *y;
    int rows, d;
    float scale, eps, offset, inv_d;
    int team, slots, packs;
};

// kBranch: a join; else the norm alone (of `residual`).
template <typename R, typename B, int V, int P, bool kBranch>
__global__ void __launch_bounds__(kNormThreads, 1) norm_forward_kernel(const __grid_constant__ ForwardParams p) {
    __shared__ float scratch[2 * (kNormThreads / 32) * kNormSums];
    Team team(p.team, scratch);
    // Teams of a warp take steps together: the loop ends when the first of them has no row.
    const int ahead = p.team < 32 ? team.slot % (32 / p.team) : 0;
    for (int row0 = blockIdx.x * p.slots + team.slot - ahead; row0 < p.rows; row0 += gridDim.x * p.slots) {
        const int row = row0 + ahead;
        const bool live = row < p.rows;
        const int at = live ? row : 0;
        const R *const src = row_at<R>(p.residual, at);
        float x[P][V];
        Raw<R, V> r[P];
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const int pack = team.t + q * p.team;
            r[q].zero();
            if (live && pack < p.packs) r[q].load(src + pack * V);
        }
        if constexpr (kBranch) {
            const B *const add = row_at<B>(p.in.branch, at);
            Raw<B, V> b[P];
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                b[q].zero();
                if (live && pack < p.packs) b[q].load(add + pack * V);
            }
#pragma unroll
            for (int q = 0; q < P; ++q) b[q].get(x[q]);
            if (p.in.has & kHasPost) {
                float ss[1] = {0.f}, shrunk;
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) ss[0] = fmaf(x[q][e], x[q][e], ss[0]);
                team.sum(ss);
                const float f = unit_factor(team, x, ss[0], p.inv_d, p.eps, shrunk);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float u[V];
                    load_typed<V>(p.in.post, p.in.post_dtype, pack * V, u);
#pragma unroll
                    for (int e = 0; e < V; ++e) x[q][e] *= f * (p.offset + u[e]);
                }
            }
            if (p.in.has & kHasGate) {
                const int64_t g = (int64_t)(at / p.in.gate_span) * p.d;
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float u[V];
                    load_typed<V>(p.in.gate, p.in.gate_dtype, g + pack * V, u);
#pragma unroll
                    for (int e = 0; e < V; ++e) x[q][e] *= u[e];
                }
            }
            R *const out = reinterpret_cast<R *>(p.h) + (int64_t)at * p.d;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                float add_to[V];
                r[q].get(add_to);
#pragma unroll
                for (int e = 0; e < V; ++e) x[q][e] = fmaf(p.scale, x[q][e], add_to[e]);
                if (live && pack < p.packs) Raw<R, V>::store(out + pack * V, x[q]);
            }
        } else {
#pragma unroll
            for (int q = 0; q < P; ++q) r[q].get(x[q]);
        }
        if (p.in.has & kHasWeight) {
            float ss[1] = {0.f}, shrunk;
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int e = 0; e < V; ++e) ss[0] = fmaf(x[q][e], x[q][e], ss[0]);
            team.sum(ss);
            const float f = unit_factor(team, x, ss[0], p.inv_d, p.eps, shrunk);
            B *const out = reinterpret_cast<B *>(p.y) + (int64_t)at * p.d;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                if (pack >= p.packs) break;
                float w[V];
                load_typed<V>(p.in.weight, p.in.weight_dtype, pack * V, w);
#pragma unroll
                for (int e = 0; e < V; ++e) w[e] = x[q][e] * f * (p.offset + w[e]);
                if (live) Raw<B, V>::store(out + pack * V, w);
            }
        }
    }
}

template <typename R, typename B, bool kBranch>
__global__ void __launch_bounds__(kWideThreads, 1) norm_forward_wide_kernel(const __grid_constant__ ForwardParams p) {
    __shared__ float scratch[2 * (kNormThreads / 32) * kNormSums];
    Team team(kWideThreads, scratch);
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const R *const src = row_at<R>(p.residual, row);
        const B *const add = row_at<B>(p.in.branch, kBranch ? row : 0);
        const int64_t g = (int64_t)(row / p.in.gate_span) * p.d;
        float shrunk, f = 1.f;
        if (kBranch && (p.in.has & kHasPost)) {
            f = wide_factor(team, p.d, [&](int j) { return load_one(add + j); }, p.inv_d, p.eps, shrunk);
        } else {
            shrunk = 1.f;
        }
        const auto h = [&](int j) {
            const float r = load_one(src + j);
            if (!kBranch) return r;
            float x = load_one(add + j);
            if (p.in.has & kHasPost) x = x * shrunk * (f * (p.offset + value_at(p.in.post, p.in.post_dtype, j)));
            if (p.in.has & kHasGate) x *= value_at(p.in.gate, p.in.gate_dtype, g + j);
            return fmaf(p.scale, x, r);
        };
        if (kBranch)
            for (int j = threadIdx.x; j < p.d; j += kWideThreads) {
                const float x[1] = {h(j)};
                Raw<R, 1>::store(reinterpret_cast<R *>(p.h) + (int64_t)row * p.d + j, x);
            }
        if (p.in.has & kHasWeight) {
            float less;
            const float factor = wide_factor(team, p.d, h, p.inv_d, p.eps, less);
            for (int j = threadIdx.x; j < p.d; j += kWideThreads) {
                const float y[1] = {h(j) * less * factor * (p.offset + value_at(p.in.weight, p.in.weight_dtype, j))};
                Raw<B, 1>::store(reinterpret_cast<B *>(p.y) + (int64_t)row * p.d + j, y);
            }
        }
    }
}

template <typename R, typename B>
void launch_wide(const ForwardParams &p, int grid, bool branch, cudaStream_t stream) {
    if (branch)
        norm_forward_wide_kernel<R, B, true><<<grid, kWideThreads, 0, stream>>>(p);
    else if constexpr (std::is_same_v<R, B>)
        norm_forward_wide_kernel<R, B, false><<<grid, kWideThreads, 0, stream>>>(p);
}

template <typename R, typename B, int V, int P>
void launch_forward(const ForwardParams &p, int grid, bool branch, cudaStream_t stream) {
    if (branch)
        norm_forward_kernel<R, B, V, P, true><<<grid, p.team * p.slots, 0, stream>>>(p);
    else if constexpr (std::is_same_v<R, B>)
        norm_forward_kernel<R, B, V, P, false><<<grid, p.team * p.slots, 0, stream>>>(p);
}

template <typename R, typename B>
void launch_forward(const NormShape &s, const ForwardParams &p, int grid, bool branch, cudaStream_t stream) {
    if (s.V == 8)
        s.P == 1   ? launch_forward<R, B, 8, 1>(p, grid, branch, stream)
        : s.P == 2 ? launch_forward<R, B, 8, 2>(p, grid, branch, stream)
                   : launch_forward<R, B, 8, 4>(p, grid, branch, stream);
    else
        s.P == 1   ? launch_forward<R, B, 1, 1>(p, grid, branch, stream)
        : s.P == 8 ? launch_forward<R, B, 1, 8>(p, grid, branch, stream)
                   : launch_wide<R, B>(p, grid, branch, stream);
}

}  // namespace

int norm_args_status(const lamq_norm_args *a, bool backward) {
    LAMQ_REQUIRE(a, "null pointer (args)");
    const bool join = a->branch.data != nullptr;
    LAMQ_REQUIRE(a->rows >= 0 && a->d >= 0 && a->rows <= 1 << 30, "bad shape: %lld rows of %d",
                 (long long)a->rows, a->d);
    LAMQ_REQUIRE(a->d <= kNormMaxD, "rows of %d elements: up to %d", a->d, kNormMaxD);
    const int types[] = {a->residual_dtype, a->branch_dtype, a->weight_dtype, a->post_dtype, a->gate_dtype};
    for (int t : types) LAMQ_REQUIRE(t == LAMQ_F32 || t == LAMQ_BF16, "dtype %d: LAMQ_F32 or LAMQ_BF16", t);
    LAMQ_REQUIRE(a->residual_dtype == a->branch_dtype || (join && a->residual_dtype == LAMQ_F32),
                 "dtype: a bf16 residual takes a bf16 branch (the norm alone: one type)");
    LAMQ_REQUIRE(std::isfinite(a->eps) && a->eps >= 0x1p-126f, "eps must be a positive normal number");
    LAMQ_REQUIRE(std::isfinite(a->scale) && std::isfinite(a->offset), "scale and offset must be finite");
    if (a->rows == 0 || a->d == 0) return LAMQ_OK;
    LAMQ_REQUIRE(!a->gate || (a->gate_span >= 1 && a->gate_span <= INT_MAX && a->rows % a->gate_span == 0),
                 "gate_span %lld must divide the %lld rows", (long long)a->gate_span, (long long)a->rows);
    LAMQ_REQUIRE(join || (a->weight && !a->post && !a->gate), "null pointer: the norm alone has a weight, no post and no gate");
    const lamq_rows *rows[] = {&a->residual, &a->branch, &a->dh, &a->dy};
    for (int i = 0; i < (backward ? 4 : 2); ++i)
        LAMQ_REQUIRE(!rows[i]->data || (rows[i]->inner >= 1 && rows[i]->inner <= INT_MAX), "rows: an inner count of 1 to 2^31 - 1");
    LAMQ_REQUIRE(a->residual.data, "null pointer (residual)");
    if (!backward) {
        LAMQ_REQUIRE(!join || a->h, "null pointer (h)");
        LAMQ_REQUIRE(!a->weight || a->y, "null pointer (y)");
    } else {
        LAMQ_REQUIRE(a->d_residual, "null pointer (d_residual)");
        LAMQ_REQUIRE(join || !a->dh.data, "the norm alone has no dh");
        LAMQ_REQUIRE(join || !a->d_branch, "the norm alone has no d_branch");
        LAMQ_REQUIRE(a->weight || (!a->d_weight && !a->dy.data), "dy and d_weight belong to a weight");
        LAMQ_REQUIRE(a->post || !a->d_post, "d_post belongs to a post weight");
        LAMQ_REQUIRE(a->gate || !a->d_gate, "d_gate belongs to a gate");
    }
    return LAMQ_OK;
}

}  // namespace lamq

using namespace lamq;

extern "C" int lamq_norm_forward(const lamq_norm_args *a, lamq_stream_t stream) {
    if (const int st = norm_args_status(a, false)) return st;
    if (a->rows == 0 || a->d == 0) return LAMQ_OK;
    const bool join = a->branch.data != nullptr;
    const NormShape s = norm_shape(*a, false);
    ForwardParams p;
    p.residual = a->residual, p.in = present(*a, false);
    p.h = a->h, p.y = a->y;
    p.rows = (int)a->rows, p.d = a->d;
    p.scale = a->scale, p.eps = a->eps, p.offset = a->offset, p.inv_d = 1.f / (float)a->d;
    p.team = s.team, p.slots = norm_slots(s, a->rows, 256), p.packs = s.packs;
    const int64_t blocks = (a->rows + p.slots - 1) / p.slots;
    const int grid = (int)std::min<int64_t>(blocks, kSMs * (2048 / (p.team * p.slots)));
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->residual_dtype == LAMQ_BF16)
        launch_forward<__nv_bfloat16, __nv_bfloat16>(s, p, grid, join, st);
    else if (a->branch_dtype == LAMQ_BF16)
        launch_forward<float, __nv_bfloat16>(s, p, grid, join, st);
    else
        launch_forward<float, float>(s, p, grid, join, st);
    LAMQ_CHECK_LAUNCH("lamq_norm_forward");
    return LAMQ_OK;
}
