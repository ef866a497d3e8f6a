// The gradients of the norms around a block, from dh and dy, the gradients of h and y. With x̂ = x·r(x), r the norm's
// factor:
//
//   t = dy ⊙ (offset + weight)        g = dh + r(h)·(t − ĥ·mean(t ⊙ ĥ))        d_weight = Σ_rows dy ⊙ ĥ
//   d_residual = g                    d_gate = scale · Σ g ⊙ p, over the rows that share the gate's row
//   t = scale · gate ⊙ g              d_branch = r(b)·(t ⊙ u − b̂·mean(t ⊙ u ⊙ b̂)),  u = offset + post;  d_post = Σ t ⊙ b̂
//
// Bound by memory. The statistics of h and b are computed again: their rows are read whole anyway, and nothing has to be
// kept from the forward. The sums over rows stay in the registers of the threads that own the columns: a worker (a team)
// takes the rows of one range, blocks write one partial row each, and a second kernel adds the partials in order.
#pragma once

#include "norm_wide.cuh"

namespace lamq {
namespace {

struct BackwardParams {
    lamq_rows h;
    Present in;
    void *d_residual, *d_branch, *d_gate;
    float *w_part, *u_part, *g_part;  // partial sums of d_weight, d_post and a shared d_gate (NULL: not wanted)
    int rows, d;
    float scale, eps, offset, inv_d;
    int team, slots, packs, columns;  // columns: of a partial row
    int per;        // rows of a worker
    int gate_mode;  // kGate*: where the sums of d_gate go
};

// d_gate is not wanted; one gate row for all rows (summed like a weight's gradient); its rows are whole inside a worker's
// range (written at once); its rows span workers (a partial for each worker and gate row that meet).
enum { kGateNone, kGateOne, kGateInside, kGateAcross };
enum { kNormAlone, kJoinPlain, kJoinFull };  // the norm alone; a join without post and gate; any join

// What a thread has summed of its columns: in registers where these are few, else in shared memory that no other thread
// touches (three sums of 16384 columns take 196608 bytes).
template <int P, int V, bool kRegisters = P * V <= kNormShared>
struct Columns {
    float v[P][V];
    __device__ __forceinline__ Columns(float *) { clear(); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) v[q][e] = 0.f;
    }
    __device__ __forceinline__ void add(int q, int e, float a, float b) { v[q][e] = fmaf(a, b, v[q][e]); }
    __device__ __forceinline__ void get(int q, float (&f)[V]) const {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = v[q][e];
    }
};

template <int P, int V>
struct Columns<P, V, false> {
    float *at;
    __device__ __forceinline__ Columns(float *shared) : at(shared + threadIdx.x) { clear(); }
    __device__ __forceinline__ float &of(int q, int e) { return at[(q * V + e) * blockDim.x]; }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) of(q, e) = 0.f;
    }
    __device__ __forceinline__ void add(int q, int e, float a, float b) { of(q, e) = fmaf(a, b, of(q, e)); }
    __device__ __forceinline__ void get(int q, float (&f)[V]) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = of(q, e);
    }
};

// The block's teams' sums added in order and written as the block's partial row.
template <int P, int V>
__device__ __forceinline__ void write_partial(const BackwardParams &p, const Team &team, Columns<P, V> &sums, float *part,
                                              float *shared) {
    float acc[P][V];
#pragma unroll
    for (int q = 0; q < P; ++q) sums.get(q, acc[q]);
    if constexpr (P * V <= kNormShared) {
        if (p.slots > 1) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int e = 0; e < V; ++e) shared[(q * V + e) * kNormThreads + threadIdx.x] = acc[q][e];
            __syncthreads();
            if (team.slot != 0) return;
            for (int s = 1; s < p.slots; ++s)
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[q][e] += shared[(q * V + e) * kNormThreads + s * p.team + team.t];
        }
    }
    float *const row = part + (int64_t)blockIdx.x * p.columns;
#pragma unroll
    for (int q = 0; q < P; ++q) {
        const int pack = team.t + q * p.team;
        if (pack < p.packs) Raw<float, V>::store(row + pack * V, acc[q]);
    }
}

template <typename R, typename B, int V, int P, int kMode, bool kSums>
__global__ void __launch_bounds__(kNormThreads, 1) norm_backward_kernel(const __grid_constant__ BackwardParams p) {
    __shared__ float scratch[2 * (kNormThreads / 32) * kNormSums];
    __shared__ float shared[kSums && P * V <= kNormShared ? kNormThreads * P * V : 1];
    extern __shared__ float columns[];  // of the sums that registers do not hold (backward_shared)
    Team team(p.team, scratch);
    constexpr bool kEarly = P * V <= 16;
    constexpr int kStep = kSums && P * V > kNormShared ? P * V : 0;
    Columns<P, V, !kStep> dw(columns), du(columns + (kMode == kJoinFull ? 1 : 0) * kStep * p.team),
        dg(columns + (kMode == kJoinFull ? 2 : 0) * kStep * p.team);
    const int worker = blockIdx.x * p.slots + team.slot;
    const bool ranges = kMode == kJoinFull && p.gate_mode >= kGateInside;  // each team its own range of rows
    const int first = ranges ? worker * p.per : blockIdx.x * p.slots * p.per + team.slot, step = ranges ? 1 : p.slots;
    for (int k = 0; k < p.per; ++k) {
        const int row = first + k * step;
        const bool live = row < p.rows;
        if (p.team < 32 ? !__any_sync(0xffffffffu, live) : !live) break;
        const int at = live ? row : 0;
        const R *const dh = row_at<R>(p.in.dh, at);
        const bool has_dh = kMode != kNormAlone && (p.in.has & kHasDh);
        Raw<R, V> early[kEarly ? P : 1];
        if (kEarly && has_dh)
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                early[q].zero();
                if (live && pack < p.packs) early[q].load(dh + pack * V);
            }
        // dh, a pack at a time: loaded before the row's sums, or where registers are short behind them
        const auto add_dh = [&](int q, int pack, float (&f)[V]) {
            if (!has_dh) return;
            float x[V];
            if (kEarly) {
                early[kEarly ? q : 0].get(x);
            } else {
                Raw<R, V> late;
                late.zero();
                if (live) late.load(dh + pack * V);
                late.get(x);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] += x[e];
        };
        float g[P][V];  // dy, then the gradient at h, then at the branch
        if (p.in.has & kHasDy) {
            float x[P][V], s[2] = {0.f, 0.f}, shrunk;
            const R *const src = row_at<R>(p.h, at);
            const B *const grad = row_at<B>(p.in.dy, at);
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                Raw<R, V> a;
                Raw<B, V> b;
                a.zero(), b.zero();
                if (live && pack < p.packs) a.load(src + pack * V), b.load(grad + pack * V);
                a.get(x[q]), b.get(g[q]);
            }
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                if (pack >= p.packs) break;
                float w[V];
                load_typed<V>(p.in.weight, p.in.weight_dtype, pack * V, w);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    s[0] = fmaf(x[q][e], x[q][e], s[0]);
                    s[1] = fmaf(g[q][e] * (p.offset + w[e]), x[q][e], s[1]);
                }
            }
            team.sum(s);
            const float f = unit_factor(team, x, s[0], p.inv_d, p.eps, shrunk);
            if (p.team < 32 ? __any_sync(0xffffffffu, shrunk != 1.f) : shrunk != 1.f) {
                float again[1] = {0.f};  // x changed, and the sum may have overflowed
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float w[V];
                    load_typed<V>(p.in.weight, p.in.weight_dtype, pack * V, w);
#pragma unroll
                    for (int e = 0; e < V; ++e) again[0] = fmaf(g[q][e] * (p.offset + w[e]), x[q][e], again[0]);
                }
                team.sum(again);
                s[1] = again[0];
            }
            // f is the factor of x as it stands, f · shrunk that of x as it was
            const float r = f * shrunk, c = s[1] * f * p.inv_d;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                if (pack >= p.packs) break;
                float w[V];
                load_typed<V>(p.in.weight, p.in.weight_dtype, pack * V, w);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float unit = x[q][e] * f;
                    if (kSums) dw.add(q, e, g[q][e], unit);
                    g[q][e] = r * fmaf(-unit, c, g[q][e] * (p.offset + w[e]));
                }
                add_dh(q, pack, g[q]);
            }
        } else {
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
#pragma unroll
                for (int e = 0; e < V; ++e) g[q][e] = 0.f;
                if (pack < p.packs) add_dh(q, pack, g[q]);
            }
        }
        {
            R *const out = reinterpret_cast<R *>(p.d_residual) + (int64_t)at * p.d;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                if (live && pack < p.packs) Raw<R, V>::store(out + pack * V, g[q]);
            }
        }
        if (kMode == kNormAlone) continue;
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) g[q][e] *= p.scale;
        if (kMode == kJoinFull) {
            float x[P][V], f = 1.f, shrunk = 1.f;  // the branch
            if ((p.in.has & kHasPost) || p.gate_mode != kGateNone) {
                const B *const src = row_at<B>(p.in.branch, at);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    Raw<B, V> a;
                    a.zero();
                    if (live && pack < p.packs) a.load(src + pack * V);
                    a.get(x[q]);
                }
            }
            if (p.in.has & kHasPost) {
                float ss[1] = {0.f};
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) ss[0] = fmaf(x[q][e], x[q][e], ss[0]);
                team.sum(ss);
                f = unit_factor(team, x, ss[0], p.inv_d, p.eps, shrunk);
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) x[q][e] *= f;
            }
            if (p.in.has & kHasGate) {
                const int64_t gate_row = at / p.in.gate_span;
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float u[V], v[V];
                    load_typed<V>(p.in.gate, p.in.gate_dtype, gate_row * p.d + pack * V, u);
                    if (kSums && p.gate_mode != kGateNone) {
                        if (p.in.has & kHasPost) load_typed<V>(p.in.post, p.in.post_dtype, pack * V, v);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float b = p.in.has & kHasPost ? x[q][e] * (p.offset + v[e]) : x[q][e];
                            dg.add(q, e, g[q][e], live ? b : 0.f);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) g[q][e] *= u[e];
                }
                if (kSums && p.gate_mode >= kGateInside && live && (k + 1 == p.per || (at + 1) % p.in.gate_span == 0 || at + 1 == p.rows)) {
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        const int pack = team.t + q * p.team;
                        if (pack >= p.packs) break;
                        float sum[V];
                        dg.get(q, sum);
                        if (p.gate_mode == kGateInside)
                            store_typed<V>(p.d_gate, p.in.gate_dtype, gate_row * p.d + pack * V, sum);
                        else  // a worker and a gate row, both growing row by row: their sum names the pair
                            Raw<float, V>::store(p.g_part + (worker + gate_row) * p.columns + pack * V, sum);
                    }
                    dg.clear();
                }
            }
            if (p.in.has & kHasPost) {
                float s[1] = {0.f};
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float u[V];
                    load_typed<V>(p.in.post, p.in.post_dtype, pack * V, u);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        if (kSums) du.add(q, e, g[q][e], x[q][e]);
                        g[q][e] *= p.offset + u[e];
                        s[0] = fmaf(g[q][e], x[q][e], s[0]);
                    }
                }
                team.sum(s);
                const float r = f * shrunk, c = s[0] * p.inv_d;
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) g[q][e] = r * fmaf(-x[q][e], c, g[q][e]);
            }
        }
        if (p.d_branch) {
            B *const out = reinterpret_cast<B *>(p.d_branch) + (int64_t)at * p.d;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int pack = team.t + q * p.team;
                if (live && pack < p.packs) Raw<B, V>::store(out + pack * V, g[q]);
            }
        }
    }
    if constexpr (kSums) {
        if (p.w_part) write_partial(p, team, dw, p.w_part, shared);
        if (kMode == kJoinFull && p.u_part) write_partial(p, team, du, p.u_part, shared);
        if (kMode == kJoinFull && p.gate_mode == kGateOne) write_partial(p, team, dg, p.g_part, shared);
    }
}

// Dynamic shared memory of a block.
template <int V, int P>
int backward_shared(int mode, bool sums, int team) {
    return sums && P * V > kNormShared ? (mode == kJoinFull ? 3 : 1) * P * V * team * (int)sizeof(float) : 0;
}

template <typename R, typename B, int V, int P, int kMode, bool kSums>
int launch_backward(const BackwardParams &p, int grid, cudaStream_t stream) {
    const auto kernel = norm_backward_kernel<R, B, V, P, kMode, kSums>;
    const int shared = backward_shared<V, P>(kMode, kSums, p.team);
    if (shared) {
        const cudaError_t e = smem_limit_max_once(reinterpret_cast<const void *>(kernel));
        if (e != cudaSuccess) {
            set_error("lamq_norm_backward: %s", cudaGetErrorString(e));
            return LAMQ_ERR_CUDA;
        }
    }
    kernel<<<grid, p.team * p.slots, shared, stream>>>(p);
    return LAMQ_OK;
}

template <typename R, typename B, int V, int P>
int launch_backward(const BackwardParams &p, int grid, int mode, bool sums, cudaStream_t stream) {
    if constexpr (P * V <= kNormFull)
        if (mode == kJoinFull)
            return sums ? launch_backward<R, B, V, P, kJoinFull, true>(p, grid, stream)
                        : launch_backward<R, B, V, P, kJoinFull, false>(p, grid, stream);
    if (mode == kJoinPlain)
        return sums ? launch_backward<R, B, V, P, kJoinPlain, true>(p, grid, stream)
                    : launch_backward<R, B, V, P, kJoinPlain, false>(p, grid, stream);
    if constexpr (std::is_same_v<R, B>)
        return sums ? launch_backward<R, B, V, P, kNormAlone, true>(p, grid, stream)
                    : launch_backward<R, B, V, P, kNormAlone, false>(p, grid, stream);
    return LAMQ_ERR_INVALID;  // no such call: the checks refuse a norm of two types, the shape a wider full join
}

// By the call's types.
template <int V, int P>
int launch_backward(const lamq_norm_args &a, const BackwardParams &p, int grid, int mode, bool sums, cudaStream_t stream) {
    if (a.residual_dtype == LAMQ_BF16)
        return launch_backward<__nv_bfloat16, __nv_bfloat16, V, P>(p, grid, mode, sums, stream);
    if (a.branch_dtype == LAMQ_BF16) return launch_backward<float, __nv_bfloat16, V, P>(p, grid, mode, sums, stream);
    return launch_backward<float, float, V, P>(p, grid, mode, sums, stream);
}

}  // namespace

// The kernels for rows that may begin anywhere (norm_backward_elements.cu). `params`: a BackwardParams.
int launch_backward_elements(int P, const lamq_norm_args &a, const void *params, int grid, int mode, bool sums,
                             cudaStream_t stream);

}  // namespace lamq
