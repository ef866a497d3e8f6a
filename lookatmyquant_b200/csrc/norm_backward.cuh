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
//
// Measured (us; bytes at 6551 GB/s in brackets): the norm alone, 16384 x 2560 bf16 53 (38); a plain join of that size 63 (51); a
// join with both norms and a gate for all, 8192 x 4096 bf16 125 (62): 520 instructions a warp and row of 8 elements a thread at
// 2.0 a cycle, 122 registers, 16 warps; the same with a gate of its own for each element, 3335 x 1337 fp32, rows that begin
// anywhere, 55 (22).
#pragma once

#include "dependent.cuh"
#include "norm_wide.cuh"

namespace lamq {
namespace {

struct BackwardParams {
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
template <int E, bool kRegisters>
struct Columns {
    Vec<E> v;
    __device__ __forceinline__ Columns(float *) { v.clear(); }
    __device__ __forceinline__ void clear() { v.clear(); }
    __device__ __forceinline__ void add(const Vec<E> &a, const Vec<E> &b) { v.add(a, b); }
    __device__ __forceinline__ Vec<E> all() const { return v; }
};

template <int E>
struct Columns<E, false> {
    float2 *at;  // pair i of this thread: at[i * blockDim.x]
    __device__ __forceinline__ Columns(float *shared) : at(reinterpret_cast<float2 *>(shared) + threadIdx.x) { clear(); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < Vec<E>::kPairs; ++i) at[i * blockDim.x] = make_float2(0.f, 0.f);
    }
    __device__ __forceinline__ void add(const Vec<E> &a, const Vec<E> &b) {
#pragma unroll
        for (int i = 0; i < Vec<E>::kPairs; ++i) at[i * blockDim.x] = fma2(a.v[i], b.v[i], at[i * blockDim.x]);
    }
    __device__ __forceinline__ Vec<E> all() const {
        Vec<E> x;
#pragma unroll
        for (int i = 0; i < Vec<E>::kPairs; ++i) x.v[i] = at[i * blockDim.x];
        return x;
    }
};

// The block's teams' sums added in order and written as the block's partial row.
template <int P, int V, bool kHold, bool kSub>
__device__ __forceinline__ void write_partial(const BackwardParams &p, const Team<kSub> &team, Vec<P * V> acc, float *part,
                                              float2 *shared) {
    if constexpr (kHold) {
        constexpr int kPairs = Vec<P * V>::kPairs, kThreads = 4096 / (P * V);
        if (p.slots > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPairs; ++i) shared[i * kThreads + threadIdx.x] = acc.v[i];
            __syncthreads();
            if (team.slot != 0) return;
            for (int s = 1; s < p.slots; ++s)
#pragma unroll
                for (int i = 0; i < kPairs; ++i) acc.v[i] = add2(acc.v[i], shared[i * kThreads + s * p.team + team.t]);
        }
    }
    float *const row = part + (int64_t)blockIdx.x * p.columns;
#pragma unroll
    for (int q = 0; q < P; ++q) {
        const int pack = team.pack(q);
        float f[V];
        acc.get(q * V, f);
        if (pack < p.packs) Raw<float, V>::store(row + pack * V, f);
    }
}

// Threads of blocks that are not too large (kHold) keep the weights and the gate of their columns in registers.
template <typename R, typename B, NormKernel kKernel, int kMode, bool kSums, bool kSub>
__global__ void __launch_bounds__(resident(kKernel, kMode, true), 1)
    norm_backward_kernel(const __grid_constant__ BackwardParams p) {
    extern __shared__ uint4 stages[];
    __shared__ alignas(16) float scratch[Team<false>::kScratch];
    constexpr int V = NormSizes<kKernel>::V, P = NormSizes<kKernel>::P;
    constexpr bool kFull = kMode == kJoinFull, kJoin = kMode != kNormAlone, kHold = NormSizes<kKernel>::kHold;
    using Row = Vec<P * V>;
    __shared__ float2 shared[kSums && kHold ? NormSizes<kKernel>::kThreads * Row::kPairs : 1];
    if (kSums) let_follow();
    Team<kSub> team(p.team, P, scratch);
    const Ring<V, P, kSub> ring(stages, p.ring, team, p.packs);
    float *const columns = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(stages) + p.sums_at);
    constexpr int kStep = kSums && !kHold ? P * V : 0;
    Columns<P * V, !kStep> dw(columns), du(columns + (kFull ? 1 : 0) * kStep * p.team),
        dg(columns + (kFull ? 2 : 0) * kStep * p.team);

    const bool has_dy = kMode == kNormAlone || (p.in.has & kHasDy), has_dh = kJoin && (p.in.has & kHasDh), post = kFull && (p.in.has & kHasPost),
               gate = kFull && (p.in.has & kHasGate), gates = gate && p.in.gate_span == 1,
               gate_sums = kSums && kFull && p.gate_mode != kGateNone, branch = post || gate_sums;
    const auto each = [&](auto f) {  // this thread's packs
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const int pack = team.pack(q);
            if (pack < p.packs) f(q, pack);
        }
    };
    const auto load = [&](const void *from, int dtype, float add, Row &w) {  // a weight, or a row of the gate
        w.clear();
        each([&](int q, int pack) {
            float f[V];
            load_typed<V>(from, dtype, pack * V, f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] += add;
            w.set(q * V, f);
        });
    };
    const auto gate_at = [&](int row) {
        return reinterpret_cast<const unsigned char *>(p.in.gate) +
               (int64_t)p.in.by_span.of(row) * p.d * (p.in.gate_dtype == LAMQ_F32 ? 4 : 2);
    };
    Row w, u, held;
    int gate_of = -1;  // the gate row that is held
    if (kHold) {
        if (has_dy) load(p.in.weight, p.in.weight_dtype, p.offset, w);
        if (kFull && post) load(p.in.post, p.in.post_dtype, p.offset, u);
    }

    const int worker = blockIdx.x * p.slots + team.slot;
    const bool ranges = kFull && p.gate_mode >= kGateInside;  // each team its own range of rows
    const int first = ranges ? worker * p.per : blockIdx.x * p.slots * p.per + team.slot, step = ranges ? 1 : p.slots;
    int fetched = 0;
    const auto fetch = [&](uint32_t stage) {
        const int row = first + fetched * step;
        const bool there = fetched < p.per && row < p.rows;
        if (there || kSub) {  // a team that has no row beside others of its warp that do: zeros
            const int at = there ? row : 0, bytes = there ? 16 : 0;
            if (has_dy) {
                ring.fetch(stage, kTensorH, row_at<R, kJoin>(p.in.h, at), bytes);
                ring.fetch(stage, kTensorDy, row_at<B, kJoin>(p.in.dy, at), bytes);
            }
            if (has_dh) ring.fetch(stage, kTensorDh, row_at<R, kJoin>(p.in.dh, at), bytes);
            if (branch) ring.fetch(stage, kTensorBranch, row_at<B, kJoin>(p.in.branch, at), bytes);
            if (gates) ring.fetch_typed(stage, kTensorGate, gate_at(at), p.in.gate_dtype, bytes);
        }
        ++fetched;
        ring.commit();
    };
    uint32_t stage = ring.first(), to = stage;
    for (int i = 1; i < p.ring.stages; ++i, to = ring.after(to)) fetch(to);
    for (int k = 0; k < p.per; ++k) {
        const int row = first + k * step;
        const bool live = row < p.rows;
        if (!team.any(live)) break;
        if (V == 1 && p.ring.stages > 1) {  // all have read the stage that is filled next
            ring.wait();
            fetch(to);
        } else {
            __syncwarp();  // all of the warp have read the stage that is filled next
            fetch(to);
            ring.wait();
        }
        const int at = live ? row : 0;
        Row g, x, b;  // dy, then the gradient at h, then at the branch; h; the branch
        if (has_dy) {
            ring.read(stage, kTensorH, row_at<R, kJoin>(p.in.h, at), x);
            ring.read(stage, kTensorDy, row_at<B, kJoin>(p.in.dy, at), g);
        } else {
            x.clear(), g.clear();
        }
        if constexpr (kFull) {
            if (branch)
                ring.read(stage, kTensorBranch, row_at<B, kJoin>(p.in.branch, at), b);
            else
                b.clear();
        }
        Row t = g;
        if (!kHold && has_dy) load(p.in.weight, p.in.weight_dtype, p.offset, w);
        if (has_dy) t *= w;
        float s[kFull ? 3 : 2];  // Σ h², Σ t h, Σ b²
        s[0] = x.dot(x), s[1] = t.dot(x);
        if constexpr (kFull) s[2] = b.dot(b);
        if (has_dy || post) team.sum(s);
        if (has_dy) {
            const bool lost = sums_lost(s[0], s[1], p.eps);
            // f: the factor of x as it stands, f · shrunk that of h
            float shrunk = 1.f, f = reciprocal_root(fmaf(s[0], p.inv_d, p.eps)), c = s[1] * f, by = f;
            if (team.any(lost)) {
                f = unit_factor(team, x, s[0], p.inv_d, p.eps, shrunk);
                x *= f, by = 1.f;
                float unit[1] = {t.dot(x)};
                team.sum(unit);
                if (lost) c = unit[0];
            }
            x *= by;
            if (kSums) dw.add(g, x);
            t.take(c * p.inv_d, x, f * shrunk);
            g = t;
        }
        if (has_dh) {
            ring.read(stage, kTensorDh, row_at<R, kJoin>(p.in.dh, at), x);
            g += x;
        }
        if (live) {
            R *const out = reinterpret_cast<R *>(p.d_residual) + (int64_t)row * p.d;
            each([&](int q, int pack) {
                float f[V];
                g.get(q * V, f);
                Raw<R, V>::store(out + pack * V, f);
            });
        }
        if constexpr (kJoin) {
            g *= p.scale;
            if constexpr (kFull) {
                float f = 1.f, shrunk = 1.f;
                if (post) {
                    f = unit_factor(team, b, s[2], p.inv_d, p.eps, shrunk);
                    b *= f;
                    if (!kHold) load(p.in.post, p.in.post_dtype, p.offset, u);
                }
                if (gate && live) {
                    const int gate_row = p.in.by_span.of(row);
                    if (gates) {
                        ring.read_typed(stage, kTensorGate, gate_at(row), p.in.gate_dtype, held);
                    } else if (gate_row != gate_of) {
                        gate_of = gate_row;
                        load(gate_at(row), p.in.gate_dtype, 0.f, held);
                    }
                    if (gate_sums) {
                        Row q = b;
                        if (post) q *= u;
                        dg.add(g, q);
                    }
                    g *= held;
                    if (gate_sums && p.gate_mode >= kGateInside &&
                        (k + 1 == p.per || row + 1 == (gate_row + 1) * p.in.gate_span)) {
                        const Row sums = dg.all();
                        each([&](int q, int pack) {
                            float f[V];
                            sums.get(q * V, f);
                            if (p.gate_mode == kGateInside)
                                store_typed<V>(p.d_gate, p.in.gate_dtype, (int64_t)gate_row * p.d + pack * V, f);
                            else  // a worker and a gate row, both growing row by row: their sum names the pair
                                Raw<float, V>::store(p.g_part + (int64_t)(worker + gate_row) * p.columns + pack * V, f);
                        });
                        dg.clear();
                    }
                }
                if (post) {
                    if (kSums) du.add(g, b);
                    g *= u;
                    float c[1] = {g.dot(b)};
                    team.sum(c);
                    g.take(c[0] * p.inv_d, b, f * shrunk);
                }
            }
            if (p.d_branch && live) {
                B *const out = reinterpret_cast<B *>(p.d_branch) + (int64_t)row * p.d;
                each([&](int q, int pack) {
                    float f[V];
                    g.get(q * V, f);
                    Raw<B, V>::store(out + pack * V, f);
                });
            }
        }
        stage = ring.after(stage), to = ring.after(to);
    }
    if constexpr (kSums) {
        if (p.w_part) write_partial<P, V, kHold>(p, team, dw.all(), p.w_part, shared);
        if (kFull && p.u_part) write_partial<P, V, kHold>(p, team, du.all(), p.u_part, shared);
        if (kFull && p.gate_mode == kGateOne) write_partial<P, V, kHold>(p, team, dg.all(), p.g_part, shared);
    }
}

template <typename R, typename B, NormKernel kKernel, int kMode, bool kSums>
int launch_backward(const BackwardParams &p, int grid, int shared, cudaStream_t stream) {
    const bool sub = NormSizes<kKernel>::kHold && p.team < 32;
    const auto kernel = sub ? norm_backward_kernel<R, B, kKernel, kMode, kSums, NormSizes<kKernel>::kHold>
                            : norm_backward_kernel<R, B, kKernel, kMode, kSums, false>;
    if (const int st = allow_shared(reinterpret_cast<const void *>(kernel), shared)) return st;
    kernel<<<grid, p.team * p.slots, shared, stream>>>(p);
    return LAMQ_OK;
}

template <typename R, typename B, NormKernel kKernel>
int launch_backward(const BackwardParams &p, int grid, int mode, bool sums, int shared, cudaStream_t stream) {
    constexpr bool k8 = kKernel == kVectors8 || kKernel == kElements8;  // for full joins only
    if constexpr (k8 || kKernel == kVectorsWide)
        if (mode == kJoinFull)
            return sums ? launch_backward<R, B, kKernel, kJoinFull, true>(p, grid, shared, stream)
                        : launch_backward<R, B, kKernel, kJoinFull, false>(p, grid, shared, stream);
    if constexpr (!k8)
        if (mode == kJoinPlain)
            return sums ? launch_backward<R, B, kKernel, kJoinPlain, true>(p, grid, shared, stream)
                        : launch_backward<R, B, kKernel, kJoinPlain, false>(p, grid, shared, stream);
    if constexpr (!k8 && std::is_same_v<R, B>)
        return sums ? launch_backward<R, B, kKernel, kNormAlone, true>(p, grid, shared, stream)
                    : launch_backward<R, B, kKernel, kNormAlone, false>(p, grid, shared, stream);
    return LAMQ_ERR_INVALID;  // no such call: the checks refuse a norm of two types, the shapes are chosen by the mode
}

// By the call's types.
template <NormKernel kKernel>
int launch_backward(const lamq_norm_args &a, const BackwardParams &p, int grid, int mode, bool sums, int shared,
                    cudaStream_t stream) {
    if (a.residual_dtype == LAMQ_BF16)
        return launch_backward<__nv_bfloat16, __nv_bfloat16, kKernel>(p, grid, mode, sums, shared, stream);
    if (a.branch_dtype == LAMQ_BF16)
        return launch_backward<float, __nv_bfloat16, kKernel>(p, grid, mode, sums, shared, stream);
    return launch_backward<float, float, kKernel>(p, grid, mode, sums, shared, stream);
}

}  // namespace

// The kernels for rows that may begin anywhere (norm_backward_elements.cu). `params`: a BackwardParams.
int launch_backward_elements(int kernel, const lamq_norm_args &a, const void *params, int grid, int mode, bool sums, int shared,
                             cudaStream_t stream);

}  // namespace lamq
