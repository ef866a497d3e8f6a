// The norms before and after a block, joined with the block's gate, its scale and the residual addition, forwards:
//
//   p = N(branch; post) or branch,   h = residual + scale · gate ⊙ p,   y = N(h; weight)
//   N(x; w) = x · (mean(x²) + eps)^-1/2 · (offset + w)
//
// and N(x; w) alone. Bound by memory: each row is read once into registers and written once; a norm is one exchange among
// the row's threads. Measured (us; bytes at 6551 GB/s in brackets): 262144 heads of 128 out of a wider projection, bf16, 28 (20);
// a join with both norms, a gate for each text and an fp32 stream, 8192 x 2560, 57 (38); a plain join, 16384 x 2560 bf16 62 (51).
// y is made from h in fp32, before h is rounded to its type: one rounding fewer than a norm that reads the stored h.
#include <cstddef>

#include "norm_wide.cuh"

namespace lamq {
namespace {

struct ForwardParams {
    Present in;
    void *h, *y;
    int rows, d;
    float scale, eps, offset, inv_d;
    int team, slots, packs;
    RingParams ring;
};

// Threads of blocks that are not too large (kHold) keep the weights and the gate of their columns in registers.
template <typename R, typename B, NormKernel kKernel, int kMode, bool kSub>
__global__ void __launch_bounds__(resident(kKernel, kMode, false), 1) norm_forward_kernel(const __grid_constant__ ForwardParams p) {
    extern __shared__ uint4 stages[];
    __shared__ alignas(16) float scratch[Team<false>::kScratch];
    constexpr int V = NormSizes<kKernel>::V, P = NormSizes<kKernel>::P;
    constexpr bool kBranch = kMode != kNormAlone, kFull = kMode == kJoinFull, kHold = NormSizes<kKernel>::kHold;
    using Row = Vec<P * V>;
    Team<kSub> team(p.team, P, scratch);
    const Ring<V, P, kSub> ring(stages, p.ring, team, p.packs);
    const bool post = kFull && (p.in.has & kHasPost), gate = kFull && (p.in.has & kHasGate), pre = p.in.has & kHasWeight;
    const bool gates = gate && p.in.gate_span == 1;  // a gate row for each row
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
    int gate_row = -1;  // the gate row that is held
    if (kHold) {
        if (pre) load(p.in.weight, p.in.weight_dtype, p.offset, w);
        if (kFull && post) load(p.in.post, p.in.post_dtype, p.offset, u);
    }
    const int step = gridDim.x * p.slots, first = blockIdx.x * p.slots + team.slot;
    const auto fetch = [&](int row, uint32_t stage) {
        if (row < p.rows || kSub) {  // a team that has no row beside others of its warp that do: zeros
            const int at = row < p.rows ? row : 0, bytes = row < p.rows ? 16 : 0;
            ring.fetch(stage, kTensorH, row_at<R, kBranch>(p.in.h, at), bytes);
            if (kBranch) ring.fetch(stage, kTensorBranch, row_at<B, true>(p.in.branch, at), bytes);
            if (gates) ring.fetch_typed(stage, kTensorGate, gate_at(at), p.in.gate_dtype, bytes);
        }
        ring.commit();
    };
    uint32_t stage = ring.first(), to = stage;
    int ahead = first;
    for (int i = 1; i < p.ring.stages; ++i, ahead += step, to = ring.after(to)) fetch(ahead, to);
    // Teams of a warp take steps together: the loop ends when the first of them has no row.
    const int lead = kSub ? team.slot % (32 / p.team) : 0;
    for (int row = first; row - lead < p.rows; row += step, ahead += step) {
        if (V == 1 && p.ring.stages > 1) {  // all have read the stage that is filled next
            ring.wait();
            fetch(ahead, to);
        } else {
            __syncwarp();  // all of the warp have read the stage that is filled next
            fetch(ahead, to);
            ring.wait();
        }
        const bool live = row < p.rows;
        const int at = live ? row : 0;
        Row x;
        if constexpr (kBranch) ring.read(stage, kTensorBranch, row_at<B, true>(p.in.branch, at), x);
        if constexpr (kFull) {
            if (post) {
                float ss[1] = {x.dot(x)}, shrunk;
                team.sum(ss);
                const float f = unit_factor(team, x, ss[0], p.inv_d, p.eps, shrunk);
                if (!kHold) load(p.in.post, p.in.post_dtype, p.offset, u);
                x *= f;
                x *= u;
            }
            if (gate && live) {
                const unsigned char *const from = gate_at(row);
                if (gates) {
                    ring.read_typed(stage, kTensorGate, from, p.in.gate_dtype, held);
                } else if (p.in.by_span.of(row) != gate_row) {
                    gate_row = p.in.by_span.of(row);
                    load(from, p.in.gate_dtype, 0.f, held);
                }
                x *= held;
            }
        }
        if constexpr (kBranch) {
            Row r;
            ring.read(stage, kTensorH, row_at<R, kBranch>(p.in.h, at), r);
            x.scale_add(p.scale, r);
        } else {
            ring.read(stage, kTensorH, row_at<R, kBranch>(p.in.h, at), x);
        }
        if (kBranch && live) {
            R *const out = reinterpret_cast<R *>(p.h) + (int64_t)row * p.d;
            each([&](int q, int pack) {
                float f[V];
                x.get(q * V, f);
                Raw<R, V>::store(out + pack * V, f);
            });
        }
        if (pre) {
            float ss[1] = {x.dot(x)}, shrunk;
            team.sum(ss);
            const float f = unit_factor(team, x, ss[0], p.inv_d, p.eps, shrunk);
            if (!kHold) load(p.in.weight, p.in.weight_dtype, p.offset, w);
            x *= f;
            x *= w;
            if (live) {
                B *const out = reinterpret_cast<B *>(p.y) + (int64_t)row * p.d;
                each([&](int q, int pack) {
                    float f[V];
                    x.get(q * V, f);
                    Raw<B, V>::store(out + pack * V, f);
                });
            }
        }
        stage = ring.after(stage), to = ring.after(to);
    }
}

template <typename R, typename B, bool kBranch>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(const __grid_constant__ ForwardParams p) {
    extern __shared__ float row_of_h[];
    __shared__ float scratch[32];
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const R *const src = row_at<R>(p.in.h, row);
        const B *const add = row_at<B>(p.in.branch, kBranch ? row : 0);
        const int64_t g = (int64_t)p.in.by_span.of(row) * p.d, out = (int64_t)row * p.d;
        const bool post = kBranch && (p.in.has & kHasPost), gate = kBranch && (p.in.has & kHasGate);
        float shrunk = 1.f, f = 1.f, s[1] = {0.f};
        if (post) {
            wide_each(p.d, [&](int j) {
                const float b = load_one(add + j);
                s[0] = fmaf(b, b, s[0]);
            });
            wide_sum(s, scratch);
            f = wide_factor(s[0], p.d, [&](int j) { return load_one(add + j); }, p.inv_d, p.eps, shrunk, scratch);
            s[0] = 0.f;
        }
        wide_each(p.d, [&](int j) {
            float h = load_one(src + j);
            if (kBranch) {
                float x = load_one(add + j);
                if (post) x = x * shrunk * (f * (p.offset + value_at(p.in.post, p.in.post_dtype, j)));
                if (gate) x *= value_at(p.in.gate, p.in.gate_dtype, g + j);
                const float to[1] = {fmaf(p.scale, x, h)};
                Raw<R, 1>::store(reinterpret_cast<R *>(p.h) + out + j, to);
                h = to[0];
            }
            row_of_h[j] = h;
            s[0] = fmaf(h, h, s[0]);
        });
        if (p.in.has & kHasWeight) {
            wide_sum(s, scratch);
            const float factor = wide_factor(s[0], p.d, [&](int j) { return row_of_h[j]; }, p.inv_d, p.eps, shrunk, scratch);
            wide_each(p.d, [&](int j) {
                const float y[1] = {row_of_h[j] * shrunk * factor * (p.offset + value_at(p.in.weight, p.in.weight_dtype, j))};
                Raw<B, 1>::store(reinterpret_cast<B *>(p.y) + out + j, y);
            });
        }
    }
}

template <typename R, typename B, bool kBranch>
int launch_wide(const ForwardParams &p, int grid, int shared, cudaStream_t stream) {
    const auto kernel = norm_forward_wide_kernel<R, B, kBranch>;
    if (const int st = allow_shared(reinterpret_cast<const void *>(kernel), shared)) return st;
    kernel<<<grid, kWideThreads, shared, stream>>>(p);
    return LAMQ_OK;
}

template <typename R, typename B, NormKernel kKernel, int kMode>
int launch_forward(const ForwardParams &p, int grid, int shared, cudaStream_t stream) {
    const bool sub = NormSizes<kKernel>::kHold && p.team < 32;
    const auto kernel = sub ? norm_forward_kernel<R, B, kKernel, kMode, NormSizes<kKernel>::kHold>
                            : norm_forward_kernel<R, B, kKernel, kMode, false>;
    if (const int st = allow_shared(reinterpret_cast<const void *>(kernel), shared)) return st;
    kernel<<<grid, p.team * p.slots, shared, stream>>>(p);
    return LAMQ_OK;
}

template <typename R, typename B, NormKernel kKernel>
int launch_forward(const ForwardParams &p, int grid, int mode, int shared, cudaStream_t stream) {
    if (mode == kJoinFull) return launch_forward<R, B, kKernel, kJoinFull>(p, grid, shared, stream);
    if (mode == kJoinPlain) return launch_forward<R, B, kKernel, kJoinPlain>(p, grid, shared, stream);
    if constexpr (std::is_same_v<R, B>) return launch_forward<R, B, kKernel, kNormAlone>(p, grid, shared, stream);
    return LAMQ_ERR_INVALID;  // the checks refuse a norm of two types
}

template <typename R, typename B>
int launch_forward(NormKernel kernel, const ForwardParams &p, int grid, int mode, int shared, cudaStream_t stream) {
    switch (kernel) {
        case kVectors: return launch_forward<R, B, kVectors>(p, grid, mode, shared, stream);
        case kElements: return launch_forward<R, B, kElements>(p, grid, mode, shared, stream);
        case kVectorsWide: return launch_forward<R, B, kVectorsWide>(p, grid, mode, shared, stream);
        case kVectorsWidest: return launch_forward<R, B, kVectorsWidest>(p, grid, mode, shared, stream);
        case kVectors8:
        case kElements8: return LAMQ_ERR_INVALID;  // backward only
        case kWide:
            if (mode != kNormAlone) return launch_wide<R, B, true>(p, grid, shared, stream);
            if constexpr (std::is_same_v<R, B>) return launch_wide<R, B, false>(p, grid, shared, stream);
    }
    return LAMQ_ERR_INVALID;  // the checks refuse a norm of two types
}

}  // namespace

static_assert(sizeof(lamq_norm_args) == 264 && sizeof(lamq_rows) == 32, "the bindings pack 264 bytes");
static_assert(offsetof(lamq_norm_args, d) == 16 && offsetof(lamq_norm_args, scale) == 40 && offsetof(lamq_norm_args, residual) == 56 &&
                  offsetof(lamq_norm_args, weight) == 120 && offsetof(lamq_norm_args, dh) == 160 &&
                  offsetof(lamq_norm_args, d_residual) == 224,
              "the header's field order, without padding");

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
    for (int i = 0; join && i < (backward ? 4 : 2); ++i)
        LAMQ_REQUIRE(!rows[i]->data || (one_stride(*rows[i], a->rows) && rows[i]->row <= INT_MAX / 4),
                     "rows: a join's lie at one stride, below 2^29");
    if (!backward) {
        LAMQ_REQUIRE(!join || a->h, "null pointer (h)");
        LAMQ_REQUIRE(!a->weight || a->y, "null pointer (y)");
    } else {
        LAMQ_REQUIRE(a->d_residual, "null pointer (d_residual)");
        LAMQ_REQUIRE(join || !a->dh.data, "the norm alone has no dh");
        LAMQ_REQUIRE(join || a->dy.data, "null pointer (dy)");
        LAMQ_REQUIRE(join || !a->d_branch, "the norm alone has no d_branch");
        LAMQ_REQUIRE(a->weight || (!a->d_weight && !a->dy.data), "dy and d_weight belong to a weight");
        LAMQ_REQUIRE(a->post || !a->d_post, "d_post belongs to a post weight");
        LAMQ_REQUIRE(a->gate || !a->d_gate, "d_gate belongs to a gate");
    }
    const struct {
        const char *what;
        const void *at;
        int dtype;
        bool used;
    } pointers[] = {{"residual", a->residual.data, a->residual_dtype, true}, {"branch", a->branch.data, a->branch_dtype, true},
                    {"weight", a->weight, a->weight_dtype, true}, {"post", a->post, a->post_dtype, true},
                    {"gate", a->gate, a->gate_dtype, true}, {"h", a->h, a->residual_dtype, !backward},
                    {"y", a->y, a->branch_dtype, !backward}, {"dh", a->dh.data, a->residual_dtype, backward},
                    {"dy", a->dy.data, a->branch_dtype, backward}, {"d_residual", a->d_residual, a->residual_dtype, backward},
                    {"d_branch", a->d_branch, a->branch_dtype, backward}, {"d_weight", a->d_weight, a->weight_dtype, backward},
                    {"d_post", a->d_post, a->post_dtype, backward}, {"d_gate", a->d_gate, a->gate_dtype, backward}};
    for (const auto &p : pointers)
        LAMQ_REQUIRE(!p.used || aligned_to(p.at, element_size(p.dtype)), "%s: not aligned to its elements", p.what);
    return LAMQ_OK;
}

}  // namespace lamq

using namespace lamq;

extern "C" int lamq_norm_forward(const lamq_norm_args *a, lamq_stream_t stream) {
    if (const int st = norm_args_status(a, false)) return st;
    if (a->rows == 0 || a->d == 0) return LAMQ_OK;
    const NormLayout l = norm_layout(*a, false, false, false);
    const NormShape &s = l.shape;
    const int mode = l.mode, shared = l.shared;
    ForwardParams p;
    p.in = present(*a, false);
    p.h = a->h, p.y = a->y;
    p.rows = (int)a->rows, p.d = a->d;
    p.scale = a->scale, p.eps = a->eps, p.offset = a->offset, p.inv_d = 1.f / (float)a->d;
    p.team = s.team, p.slots = l.slots, p.packs = s.packs;
    p.ring = l.ring;
    const int grid = (int)std::min<int64_t>((a->rows + p.slots - 1) / p.slots, kSMs * l.blocks);
    const cudaStream_t st = (cudaStream_t)stream;
    const int launched = a->residual_dtype == LAMQ_BF16
                             ? launch_forward<__nv_bfloat16, __nv_bfloat16>(s.kernel, p, grid, mode, shared, st)
                         : a->branch_dtype == LAMQ_BF16 ? launch_forward<float, __nv_bfloat16>(s.kernel, p, grid, mode, shared, st)
                                                        : launch_forward<float, float>(s.kernel, p, grid, mode, shared, st);
    if (launched) return launched;
    LAMQ_CHECK_LAUNCH("lamq_norm_forward");
    return LAMQ_OK;
}
