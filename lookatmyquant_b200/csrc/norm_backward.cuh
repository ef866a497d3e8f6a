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
    int sums_at;    // of the dynamic shared memory: where the sums that registers do not hold begin
    RingParams ring;
};

// d_gate is not wanted; one gate row for all rows (summed like a weight's gradient); its rows are whole inside a worker's
// range (written at once); its rows span workers (a partial for each worker and gate row that meet).
enum { kGateNone, kGateOne, kGateInside, kGateAcross };


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

// Threads that hold few packs keep the weights and gates of their columns in registers.
template <typename R, typename B, int V, int P, int kMode, bool kSums>
__global__ void __launch_bounds__(kNormThreads, kMode != kJoinFull && P * V <= kNormShared ? 2 : 1)
    norm_backward_kernel(const __grid_constant__ BackwardParams p) {
    extern __shared__ uint4 stages[];
    __shared__ alignas(16) float scratch[Team::kScratch];
    __shared__ float shared[kSums && P * V <= kNormShared ? kNormThreads * P * V : 1];
    constexpr bool kFull = kMode == kJoinFull, kJoin = kMode != kNormAlone, kHold = P * V <= kNormShared;
    Team team(p.team, scratch);
    const Ring<V, P> ring(stages, p.ring, team, p.packs);
    float *const columns = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(stages) + p.sums_at);
    constexpr int kStep = kSums && !kHold ? P * V : 0;
    Columns<P, V, !kStep> dw(columns), du(columns + (kFull ? 1 : 0) * kStep * p.team), dg(columns + (kFull ? 2 : 0) * kStep * p.team);

    const bool has_dy = p.in.has & kHasDy, has_dh = kJoin && (p.in.has & kHasDh), post = kFull && (p.in.has & kHasPost),
               gate = kFull && (p.in.has & kHasGate), gates = gate && p.in.gate_span == 1,
               gate_sums = kSums && kFull && p.gate_mode != kGateNone, branch = post || gate_sums;
    const auto weight = [&](const void *from, int dtype, int pack, float (&w)[V]) {
        load_typed<V>(from, dtype, pack * V, w);
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] += p.offset;
    };
    float w_held[kHold ? P : 1][V], u_held[kHold && kFull ? P : 1][V], gate_held[kHold && kFull ? P : 1][V];
    int gate_of = -1;  // the gate row that is held
    if constexpr (kHold)
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const int pack = team.t + q * p.team;
            if (pack >= p.packs) break;
            if (has_dy) weight(p.in.weight, p.in.weight_dtype, pack, w_held[q]);
            if constexpr (kFull)
                if (post) weight(p.in.post, p.in.post_dtype, pack, u_held[q]);
        }
    // a pack's weights: held, or loaded into `w`
    const auto w_of = [&](int q, int pack, float (&w)[V]) {
        if constexpr (kHold)
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = w_held[q][e];
        else
            weight(p.in.weight, p.in.weight_dtype, pack, w);
    };
    const auto u_of = [&](int q, int pack, float (&u)[V]) {
        if constexpr (kHold && kFull)
#pragma unroll
            for (int e = 0; e < V; ++e) u[e] = u_held[q][e];
        else
            weight(p.in.post, p.in.post_dtype, pack, u);
    };
    const auto gate_at = [&](int row) {
        return reinterpret_cast<const unsigned char *>(p.in.gate) +
               (int64_t)(row / p.in.gate_span) * p.d * (p.in.gate_dtype == LAMQ_F32 ? 4 : 2);
    };

    const int worker = blockIdx.x * p.slots + team.slot;
    const bool ranges = kFull && p.gate_mode >= kGateInside;  // each team its own range of rows
    const int first = ranges ? worker * p.per : blockIdx.x * p.slots * p.per + team.slot, step = ranges ? 1 : p.slots;
    const auto fetch = [&](int k, int stage) {
        const int row = first + k * step;
        if (k < p.per && row < p.rows) {
            if (has_dy) {
                ring.fetch(stage, kTensorH, row_at<R>(p.h, row));
                ring.fetch(stage, kTensorDy, row_at<B>(p.in.dy, row));
            }
            if (has_dh) ring.fetch(stage, kTensorDh, row_at<R>(p.in.dh, row));
            if (branch) ring.fetch(stage, kTensorBranch, row_at<B>(p.in.branch, row));
            if (gates) ring.fetch_typed(stage, kTensorGate, gate_at(row), p.in.gate_dtype);
        }
        ring.commit();
    };
    int stage = 0, to = 0;
    for (int i = 1; i < p.ring.stages; ++i, to = ring.after(to)) fetch(i - 1, to);
    for (int k = 0; k < p.per; ++k, stage = ring.after(stage), to = ring.after(to)) {
        const int row = first + k * step;
        const bool live = row < p.rows;
        if (p.team < 32 ? !__any_sync(0xffffffffu, live) : !live) break;
        if (p.ring.stages == 1) {
            fetch(k, 0);
            ring.wait();
        } else if (V == 1) {  // all have read the stage that is filled next
            ring.wait();
            fetch(k + p.ring.stages - 1, to);
        } else {
            fetch(k + p.ring.stages - 1, to);
            ring.wait();
        }
        const int at = live ? row : 0;
        float g[P][V], b[kFull ? P : 1][V];  // dy, then the gradient at h, then at the branch; the branch
        float s[kFull ? 3 : 2] = {};         // Σ h², Σ t h, Σ b²
        float x[P][V];
        const R *const h_row = row_at<R>(p.h, at), *const dh_row = row_at<R>(p.in.dh, at);
        const B *const dy_row = row_at<B>(p.in.dy, at), *const b_row = row_at<B>(p.in.branch, at);
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const int pack = team.t + q * p.team;
            const bool in = live && pack < p.packs;
#pragma unroll
            for (int e = 0; e < V; ++e) x[q][e] = g[q][e] = 0.f;
            if (has_dy && in) {
                float w[V];
                ring.read(stage, kTensorH, h_row, q, x[q]);
                ring.read(stage, kTensorDy, dy_row, q, g[q]);
                w_of(q, pack, w);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    s[0] = fmaf(x[q][e], x[q][e], s[0]);
                    s[1] = fmaf(g[q][e] * w[e], x[q][e], s[1]);
                }
            }
            if constexpr (kFull) {
#pragma unroll
                for (int e = 0; e < V; ++e) b[q][e] = 0.f;
                if (branch && in) ring.read(stage, kTensorBranch, b_row, q, b[q]);
#pragma unroll
                for (int e = 0; e < V; ++e) s[2] = fmaf(b[q][e], b[q][e], s[2]);
            }
        }
        if (has_dy || post) team.sum(s);
        if (has_dy) {
            float shrunk;
            const float f = unit_factor(team, x, s[0], p.inv_d, p.eps, shrunk);
            if (p.team < 32 ? __any_sync(0xffffffffu, shrunk != 1.f) : shrunk != 1.f) {
                float again[1] = {0.f};  // x changed, and the sum may have overflowed
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float w[V];
                    w_of(q, pack, w);
#pragma unroll
                    for (int e = 0; e < V; ++e) again[0] = fmaf(g[q][e] * w[e], x[q][e], again[0]);
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
                w_of(q, pack, w);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float unit = x[q][e] * f;
                    if (kSums) dw.add(q, e, g[q][e], unit);
                    g[q][e] = r * fmaf(-unit, c, g[q][e] * w[e]);
                }
            }
        }
        R *const out = reinterpret_cast<R *>(p.d_residual) + (int64_t)at * p.d;
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const int pack = team.t + q * p.team;
            if (pack >= p.packs || !live) break;
            if (has_dh) {
                float x[V];
                ring.read(stage, kTensorDh, dh_row, q, x);
#pragma unroll
                for (int e = 0; e < V; ++e) g[q][e] += x[e];
            }
            Raw<R, V>::store(out + pack * V, g[q]);
        }
        if (!kJoin) continue;
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) g[q][e] *= p.scale;
        if constexpr (kFull) {
            float f = 1.f, shrunk = 1.f;
            if (post) {
                f = unit_factor(team, b, s[2], p.inv_d, p.eps, shrunk);
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) b[q][e] *= f;
            }
            if (gate) {
                const int gate_row = at / p.in.gate_span;
                const unsigned char *const from = gate_at(at);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs || !live) break;
                    float v[V];
                    if (gates)
                        ring.read_typed(stage, kTensorGate, from, p.in.gate_dtype, q, v);
                    else if (!kHold)
                        load_typed<V>(from, p.in.gate_dtype, pack * V, v);
                    else if (gate_row != gate_of)
                        load_typed<V>(from, p.in.gate_dtype, pack * V, gate_held[kHold ? q : 0]);
                    if (gate_sums) {
                        float u[V];
                        if (post) u_of(q, pack, u);
#pragma unroll
                        for (int e = 0; e < V; ++e) dg.add(q, e, g[q][e], post ? b[q][e] * u[e] : b[q][e]);
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) g[q][e] *= kHold && !gates ? gate_held[kHold ? q : 0][e] : v[e];
                }
                if (live) gate_of = gate_row;
                if (gate_sums && p.gate_mode >= kGateInside && live &&
                    (k + 1 == p.per || (at + 1) % p.in.gate_span == 0 || at + 1 == p.rows)) {
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        const int pack = team.t + q * p.team;
                        if (pack >= p.packs) break;
                        float sum[V];
                        dg.get(q, sum);
                        if (p.gate_mode == kGateInside)
                            store_typed<V>(p.d_gate, p.in.gate_dtype, (int64_t)gate_row * p.d + pack * V, sum);
                        else  // a worker and a gate row, both growing row by row: their sum names the pair
                            Raw<float, V>::store(p.g_part + (int64_t)(worker + gate_row) * p.columns + pack * V, sum);
                    }
                    dg.clear();
                }
            }
            if (post) {
                float t[1] = {0.f};
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const int pack = team.t + q * p.team;
                    if (pack >= p.packs) break;
                    float u[V];
                    u_of(q, pack, u);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        if (kSums) du.add(q, e, g[q][e], b[q][e]);
                        g[q][e] *= u[e];
                        t[0] = fmaf(g[q][e], b[q][e], t[0]);
                    }
                }
                team.sum(t);
                const float r = f * shrunk, c = t[0] * p.inv_d;
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) g[q][e] = r * fmaf(-b[q][e], c, g[q][e]);
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
        if (kFull && p.u_part) write_partial(p, team, du, p.u_part, shared);
        if (kFull && p.gate_mode == kGateOne) write_partial(p, team, dg, p.g_part, shared);
    }
}

template <typename R, typename B, int V, int P, int kMode, bool kSums>
int launch_backward(const BackwardParams &p, int grid, int shared, cudaStream_t stream) {
    const auto kernel = norm_backward_kernel<R, B, V, P, kMode, kSums>;
    if (const int st = allow_shared(reinterpret_cast<const void *>(kernel), shared)) return st;
    kernel<<<grid, p.team * p.slots, shared, stream>>>(p);
    return LAMQ_OK;
}

template <typename R, typename B, int V, int P>
int launch_backward(const BackwardParams &p, int grid, int mode, bool sums, int shared, cudaStream_t stream) {
    if constexpr (P * V <= kNormFull)
        if (mode == kJoinFull)
            return sums ? launch_backward<R, B, V, P, kJoinFull, true>(p, grid, shared, stream)
                        : launch_backward<R, B, V, P, kJoinFull, false>(p, grid, shared, stream);
    if (mode == kJoinPlain)
        return sums ? launch_backward<R, B, V, P, kJoinPlain, true>(p, grid, shared, stream)
                    : launch_backward<R, B, V, P, kJoinPlain, false>(p, grid, shared, stream);
    if constexpr (std::is_same_v<R, B>)
        return sums ? launch_backward<R, B, V, P, kNormAlone, true>(p, grid, shared, stream)
                    : launch_backward<R, B, V, P, kNormAlone, false>(p, grid, shared, stream);
    return LAMQ_ERR_INVALID;  // no such call: the checks refuse a norm of two types, the shape a wider full join
}

// By the call's types.
template <int V, int P>
int launch_backward(const lamq_norm_args &a, const BackwardParams &p, int grid, int mode, bool sums, int shared,
                    cudaStream_t stream) {
    if (a.residual_dtype == LAMQ_BF16)
        return launch_backward<__nv_bfloat16, __nv_bfloat16, V, P>(p, grid, mode, sums, shared, stream);
    if (a.branch_dtype == LAMQ_BF16) return launch_backward<float, __nv_bfloat16, V, P>(p, grid, mode, sums, shared, stream);
    return launch_backward<float, float, V, P>(p, grid, mode, sums, shared, stream);
}

}  // namespace

// The kernels for rows that may begin anywhere (norm_backward_elements.cu). `params`: a BackwardParams.
int launch_backward_elements(int P, const lamq_norm_args &a, const void *params, int grid, int mode, bool sums, int shared,
                             cudaStream_t stream);

}  // namespace lamq
