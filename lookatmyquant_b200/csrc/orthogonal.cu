// Newton-Schulz orthogonalisation of an update on tcgen05 (the Muon optimiser's step): with X_0 = G / (|G|_F + eps),
//
//   A = X·Xᵀ,   B = aI + bA + cA²,   X ← B·X          (steps times; for a tall G, A = Xᵀ·X and X ← X·B)
//
// an odd polynomial in X that takes every singular value towards 1 and leaves the singular vectors alone.
//
// Precision. A singular value near zero grows by a = 3.4445 a step, and the rounding of an early step would grow with it:
// bf16 operands leave several percent of error. So X, A and B are held as fp16 pairs hi + lo (22 bits), aX is added
// exactly (from hi + lo, outside the product), and what is left to the products, X's rounding in A and in B·X with B
// without its a, moves singular vectors by 2^-12 relative where singular values have already reached 1 and nothing
// where they have not. Single products (hi·hi) are therefore enough for A in every step and for B·X in all but the last;
// A·A and the last B·X take three (hi·hi + hi·lo + lo·hi), and so does everything after a fifth step, where the roundings
// of saturated directions would go on adding up. In simulation (64 x 2000 .. 500 x 520; Gaussian, low-rank,
// power-law, row-scaled updates) this leaves 2e-4 .. 1.8e-3 of relative error, against 1.65e-3 of the bf16 output's
// rounding; three products everywhere leave 1e-5 for 2.6 times the work, single ones 4e-3. Everything is held times
// kScale = 2^10, which keeps entries of order 1/max(m, n) clear of fp16's subnormals and the largest (singular values
// up to 5, B up to 32) below its maximum. Accumulation is fp32 in TMEM.
//
// One persistent cooperative kernel runs all phases (sum of squares, X_0, then A, B, X per step) with a grid barrier
// between two of them: a small matrix would otherwise spend its time in launches. A phase's products are tiles of
// 128 x 256, or of 128 x 64 where the wider ones would leave SMs idle, handed out over the CTAs; A and B are symmetric,
// so only the tiles that reach the diagonal are computed and each is also written mirrored. Operands are read by TMA in the major order in which they lie, so nothing is
// transposed in memory.
//
// Warp roles (320 threads): warp 0 issues TMA loads, warp 1 the MMAs into two TMEM accumulators, warps 2-9 drain one
// while the next fills.
#include <algorithm>
#include <climits>
#include <mutex>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/lamq_b200_train.h"
#include "lamq_common.cuh"
#include "sm100.cuh"

namespace lamq {
namespace {

using namespace sm100;

constexpr int BM = 128, BK = 64;
constexpr int BOX = 64 * 128;                    // bytes of a 64 x 64 fp16 box

template <int BN>
struct Tile {
    static constexpr int A_BYTES = 2 * BOX, B_BYTES = BN / 64 * BOX;
    static constexpr int SLOT = A_BYTES + B_BYTES;       // the hi (or the lo) operands of 64 entries of K
    static constexpr int SLOTS = BN == 256 ? 4 : 8;      // the ring; split products take two slots a step
    static constexpr size_t SMEM = 1024 + SLOTS * SLOT + 512;
    static constexpr int EPI = BN / 2;                   // columns per epilogue warp
};

constexpr int kThreads = 320;
constexpr uint32_t kTmemCols = 512;
constexpr float kScale = 1024.f;
constexpr int kMaxSteps = 16;
constexpr int kParts = 296;                      // parts of a matrix in the sum of squares (fewer for a batch)

struct Maps {
    CUtensorMap x[2][2];  // X of even and odd steps, hi and lo
    CUtensorMap gram[2], poly[2];
};

struct Params {
    const void *G;
    int64_t ldg, gbatch;
    int g_bf16, g_vec;    // g_vec: rows of G are whole 16-byte pieces
    int out_vec;          // so are those of out
    __nv_bfloat16 *out;
    int batch, m, n;      // G is batch x m x n
    int s, l, tall;       // the smaller and the larger side
    int64_t ldx, lds;     // leading dimensions of X (m x n) and of A and B (s x s)
    __half *x[2][2], *gram[2], *poly[2];
    double *partial;      // batch x parts sums of squares
    int parts;
    float eps;
    int steps;
    float coef[kMaxSteps][3];
    unsigned *barrier;    // zero before the launch
    int *status;
};

enum { kGram, kPoly, kApply };

// One phase's products: C (M x N) over K; a_mn, b_mn: the operand lies with M (N) along its rows.
struct Phase {
    int kind, M, N, K, a_mn, b_mn, split, last;
    int tm, tn, tiles;    // tiles per matrix (of A and B: those that reach the diagonal)
};

// The row tiles of column tile tj of a symmetric C that reach the diagonal: those that start at or before its last column.
template <int BN>
__host__ __device__ __forceinline__ int column_tiles(int tm, int tj) {
    const int c = ((tj + 1) * BN - 1) / BM + 1;
    return c < tm ? c : tm;
}

template <int BN>
__host__ __device__ __forceinline__ int symmetric_tiles(int tm, int tn) {
    int t = 0;
    for (int j = 0; j < tn; ++j) t += column_tiles<BN>(tm, j);
    return t;
}

template <int BN>
__device__ __forceinline__ Phase phase_of(const Params &p, int index) {
    Phase f;
    const int step = index / 3;
    f.kind = index % 3;
    f.last = step == p.steps - 1;
    f.split = f.kind == kPoly || step > 4 || (f.kind == kApply && (step == 4 || f.last));
    f.M = f.kind == kApply && p.tall ? p.l : p.s;
    f.N = f.kind == kApply && !p.tall ? p.l : p.s;
    f.K = f.kind == kGram ? p.l : p.s;
    f.a_mn = f.kind == kGram && p.tall;
    f.b_mn = (f.kind == kGram && p.tall) || (f.kind == kApply && !p.tall);
    f.tm = (f.M + BM - 1) / BM;
    f.tn = (f.N + BN - 1) / BN;
    f.tiles = f.kind == kApply ? f.tm * f.tn : symmetric_tiles<BN>(f.tm, f.tn);
    return f;
}

// Unit u: matrix z, tile (ti, tj). The tiles that share rows or columns of X follow one another.
template <int BN>
__device__ __forceinline__ void tile_of(const Params &p, const Phase &f, int64_t u, int &z, int &ti, int &tj) {
    z = (int)(u / f.tiles);
    int t = (int)(u - (int64_t)z * f.tiles);
    if (f.kind == kApply) {
        if (p.tall) {
            ti = t / f.tn;
            tj = t - ti * f.tn;
        } else {
            tj = t / f.tm;
            ti = t - tj * f.tm;
        }
        return;
    }
    for (tj = 0;; ++tj) {
        const int c = column_tiles<BN>(f.tm, tj);
        if (t < c) break;
        t -= c;
    }
    ti = t;
}

// Every CTA has finished the phase and what it wrote is visible to all, to TMA too. Bounded: false when it gives up or
// an error has been recorded.
__device__ __forceinline__ bool grid_barrier(const Params &p, unsigned target, int *shared_ok) {
    asm volatile("fence.proxy.async.global;" ::: "memory");  // this thread's writes before other SMs' TMA reads
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(p.barrier, 1u);
        const unsigned long long t0 = globaltimer();
        int ok = 1;
        for (unsigned it = 1;; ++it) {
            unsigned v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p.barrier) : "memory");
            if (v >= target) break;
            if ((it & 255u) == 0u) {
                if (*reinterpret_cast<volatile int *>(p.status) != 0) ok = 0;
                else if (globaltimer() - t0 > kWaitTimeoutNs) {
                    atomicCAS(p.status, 0, LAMQ_ERR_TIMEOUT);
                    ok = 0;
                }
                if (!ok) break;
            }
        }
        __threadfence();
        *shared_ok = ok;
    }
    __syncthreads();
    asm volatile("fence.proxy.async.global;" ::: "memory");
    return *shared_ok != 0;
}

// Eight entries of G's row r from column c (zero past the end).
__device__ __forceinline__ void load_g8(const Params &p, int z, int r, int c, float (&v)[8]) {
    const int64_t at = z * p.gbatch + (int64_t)r * p.ldg + c;
    if (p.g_vec && c + 8 <= p.n) {
        if (p.g_bf16) {
            const uint4 q = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(p.G) + at));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __uint_as_float(w[e] << 16);
                v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        } else {
            const float4 *q = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.G) + at);
            const float4 a = __ldg(q), b = __ldg(q + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = c + e >= p.n  ? 0.f
               : p.g_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p.G)[at + e])
                          : reinterpret_cast<const float *>(p.G)[at + e];
}

// Sum over the block of one double per thread, in a fixed order, to every thread.
__device__ __forceinline__ double block_sum(double v, double *red) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) t += red[w];
    return t;
}

// v as hi + lo, both fp16.
__device__ __forceinline__ void split8(const float (&v)[8], __half (&h)[8], __half (&l)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        h[e] = __float2half_rn(v[e]);
        l[e] = __float2half_rn(v[e] - __half2float(h[e]));
    }
}

// Eight (or, at a row's end, `left`) fp16 values to p; rows start at multiples of 16 bytes.
__device__ __forceinline__ void store8(__half *p, const __half (&h)[8], int left) {
    if (left >= 8) {
        union { __half h[8]; uint4 q; } u;
#pragma unroll
        for (int e = 0; e < 8; ++e) u.h[e] = h[e];
        *reinterpret_cast<uint4 *>(p) = u.q;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < left) p[e] = h[e];
}

// hi + lo of eight (or `left`) values.
__device__ __forceinline__ void load8(const __half *hi, const __half *lo, int left, float (&v)[8]) {
    if (left >= 8) {
        union { uint4 q; __half h[8]; } a, b;
        a.q = *reinterpret_cast<const uint4 *>(hi);
        b.q = *reinterpret_cast<const uint4 *>(lo);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __half2float(a.h[e]) + __half2float(b.h[e]);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? __half2float(hi[e]) + __half2float(lo[e]) : 0.f;
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
    newton_schulz_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
    using Z = Tile<BN>;
    constexpr int SLOT = Z::SLOT, SLOTS = Z::SLOTS, A_BYTES = Z::A_BYTES, EPI = Z::EPI;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + SLOTS * SLOT);
    double *red = reinterpret_cast<double *>(bars + 2 * SLOTS + 6);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(red + kThreads / 32);
    int *shared_ok = reinterpret_cast<int *>(tmem_holder + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + SLOTS);
    const uint32_t tfull0 = smem_u32(bars + 2 * SLOTS), tempty0 = tfull0 + 16, drain = tfull0 + 32;
    const uint32_t ring = smem_u32(smem);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * SLOTS; ++i) mbar_init(full0 + 8 * i, 1);
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull0 + 8 * a, 1);
            mbar_init(tempty0 + 8 * a, 8);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_holder), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    unsigned target = 0;

    // ---- |G|_F: fixed parts of each matrix, summed in 64 bits; then X_0 by the same parts
    const int row_groups = (p.n + 7) / 8;
    const int64_t groups = (int64_t)p.m * row_groups;
    for (int64_t u = blockIdx.x; u < (int64_t)p.batch * p.parts; u += gridDim.x) {
        const int z = (int)(u / p.parts), part = (int)(u % p.parts);
        const int64_t g1 = groups * (part + 1) / p.parts;
        double acc = 0.0;
        for (int64_t g = groups * part / p.parts + threadIdx.x; g < g1; g += kThreads) {
            const int r = (int)(g / row_groups);
            float v[8];
            load_g8(p, z, r, (int)(g - (int64_t)r * row_groups) * 8, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc += (double)v[e] * (double)v[e];
        }
        acc = block_sum(acc, red);
        if (threadIdx.x == 0) p.partial[u] = acc;
    }
    bool go = grid_barrier(p, target += gridDim.x, shared_ok);
    for (int64_t u = blockIdx.x; go && u < (int64_t)p.batch * p.parts; u += gridDim.x) {
        const int z = (int)(u / p.parts), part = (int)(u % p.parts);
        double acc = 0.0;
        for (int i = threadIdx.x; i < p.parts; i += kThreads)
            acc += *reinterpret_cast<volatile double *>(p.partial + (int64_t)z * p.parts + i);
        const float inv = (float)((double)kScale / (sqrt(block_sum(acc, red)) + (double)p.eps));
        const int64_t g1 = groups * (part + 1) / p.parts;
        for (int64_t g = groups * part / p.parts + threadIdx.x; g < g1; g += kThreads) {
            const int r = (int)(g / row_groups), c = (int)(g - (int64_t)r * row_groups) * 8;
            float v[8];
            load_g8(p, z, r, c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= inv;
            __half h[8], l[8];
            split8(v, h, l);
            const int64_t at = ((int64_t)z * p.m + r) * p.ldx + c;
            store8(p.x[0][0] + at, h, p.n - c);
            store8(p.x[0][1] + at, l, p.n - c);
        }
    }
    if (go) go = grid_barrier(p, target += gridDim.x, shared_ok);

    // ---- the products. Ring slots and accumulators are counted through all phases, by each role alike
    int64_t slots = 0;
    int accs = 0;
    bool ok = true;
    for (int ph = 0; go && ph < 3 * p.steps; ++ph) {
        const Phase f = phase_of<BN>(p, ph);
        const int step = ph / 3, cur = step & 1, parts = f.split ? 2 : 1;
        const int kblocks = (f.K + BK - 1) / BK;
        const int64_t units = (int64_t)p.batch * f.tiles;
        if (warp == 0) {
            if (lane == 0) {  // ---- TMA producer
                const CUtensorMap *ma = f.kind == kGram || (f.kind == kApply && p.tall) ? maps.x[cur]
                                        : f.kind == kPoly                               ? maps.gram
                                                                                        : maps.poly;
                const CUtensorMap *mb = f.kind == kGram || (f.kind == kApply && !p.tall) ? maps.x[cur]
                                        : f.kind == kPoly                                ? maps.gram
                                                                                         : maps.poly;
                for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
                    int z, ti, tj;
                    tile_of<BN>(p, f, u, z, ti, tj);
                    for (int kb = 0; ok && kb < kblocks; ++kb)
                        for (int q = 0; q < parts; ++q, ++slots) {
                            const int st = (int)(slots % SLOTS);
                            ok = mbar_wait(empty0 + 8 * st, (uint32_t)((slots / SLOTS) & 1) ^ 1, p.status);
                            if (!ok) break;
                            const uint32_t bar = full0 + 8 * st, sa = ring + st * SLOT, sb = sa + A_BYTES;
                            const int k = kb * BK;
                            mbar_expect_tx(bar, SLOT);
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int mn = ti * BM + 64 * c;
                                tma_load_3d(sa + c * BOX, ma + q, f.a_mn ? mn : k, f.a_mn ? k : mn, z, bar);
                            }
#pragma unroll
                            for (int c = 0; c < BN / 64; ++c) {
                                const int mn = tj * BN + 64 * c;
                                tma_load_3d(sb + c * BOX, mb + q, f.b_mn ? mn : k, f.b_mn ? k : mn, z, bar);
                            }
                        }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            if (lane == 0) {  // ---- MMA issuer
                const uint32_t idesc = idesc_f16_f32(BM, BN, f.a_mn, f.b_mn);
                const uint32_t a_step = f.a_mn ? 2048 : 32, b_step = f.b_mn ? 2048 : 32;
                const uint32_t a_lbo = f.a_mn ? BOX : 16, b_lbo = f.b_mn ? BOX : 16;
                for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x, ++accs) {
                    const int acc = accs & 1;
                    ok = mbar_wait(tempty0 + 8 * acc, (uint32_t)((accs >> 1) & 1) ^ 1, p.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + acc * BN;
                    for (int kb = 0; ok && kb < kblocks; ++kb, slots += parts) {
                        uint32_t sa[2];
                        for (int q = 0; q < parts; ++q) {
                            const int64_t i = slots + q;
                            ok = ok && mbar_wait(full0 + 8 * (int)(i % SLOTS), (uint32_t)((i / SLOTS) & 1), p.status);
                            sa[q] = ring + (int)(i % SLOTS) * SLOT;
                        }
                        if (!ok) break;
                        tc_fence_after();
                        const int products = f.split ? 3 : 1;  // hi·hi, hi·lo, lo·hi
                        for (int q = 0; q < products; ++q) {
                            const uint32_t at = sa[q == 2 ? 1 : 0], bt = sa[q == 1 ? 1 : 0] + A_BYTES;
#pragma unroll
                            for (int kk = 0; kk < BK / 16; ++kk)
                                mma_f16_ss(d, smem_desc_sw128(at + kk * a_step, a_lbo, 1024),
                                           smem_desc_sw128(bt + kk * b_step, b_lbo, 1024), idesc,
                                           (kb > 0 || kk > 0 || q > 0) ? 1u : 0u);
                        }
                        for (int q = 0; q < parts; ++q) mma_commit(empty0 + 8 * (int)((slots + q) % SLOTS));
                    }
                    if (ok) mma_commit(tfull0 + 8 * acc);
                }
            }
            __syncwarp();
        } else {  // ---- epilogue: two warps per TMEM lane quadrant, half of the columns each
            const int quad = warp & 3, half = (warp - 2) >> 2;
            const float *coef = p.coef[step];
            // the exact terms: aX of B·X, bA of B (and a on its diagonal is left out of B)
            const __half *const *old = f.kind == kApply ? p.x[cur] : p.gram;
            __half *const *dst = f.kind == kApply ? p.x[cur ^ 1] : f.kind == kGram ? p.gram : p.poly;
            const float f_old = f.kind == kApply ? coef[0] : coef[1];
            const float f_acc = (f.kind == kPoly ? coef[2] : 1.f) / kScale;
            const int64_t ld = f.kind == kApply ? p.ldx : p.lds;
            for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x, ++accs) {
                int z, ti, tj;
                tile_of<BN>(p, f, u, z, ti, tj);
                const int acc = accs & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * acc, (uint32_t)((accs >> 1) & 1), p.status));
                if (!ok) break;
                tc_fence_after();
                const int i0 = ti * BM + 32 * quad, i = i0 + lane, j0 = tj * BN + EPI * half;
                // (j, i) lies in no computed tile (EPI columns share a row tile, a warp's rows a column tile)
                const bool mirror = f.kind != kApply && j0 / BM >= column_tiles<BN>(f.tm, i0 / BN);
                const uint32_t t = tmem + ((uint32_t)(32 * quad) << 16) + acc * BN + EPI * half;
#pragma unroll 1
                for (int c = 0; c < EPI; c += 32) {
                    if (j0 + c >= f.N) break;
                    const int64_t at0 = ((int64_t)z * f.M + i) * ld + j0 + c;
                    const bool live = i < f.M;
                    float o[32];
                    if (f.kind != kGram && live) {
#pragma unroll
                        for (int e0 = 0; e0 < 32; e0 += 8) {
                            float v[8];
                            load8(old[0] + at0 + e0, old[1] + at0 + e0, f.N - j0 - c - e0, v);
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e0 + e] = v[e];
                        }
                    }
                    uint32_t r[32];
                    tmem_load32(t + c, r);
                    tmem_ld_wait();
                    if (!live) continue;
#pragma unroll
                    for (int e0 = 0; e0 < 32; e0 += 8) {
                        const int j = j0 + c + e0, left = f.N - j;
                        if (left <= 0) break;
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r[e0 + e]) * f_acc;
                        if (f.kind != kGram) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = fmaf(f_old, o[e0 + e], v[e]);
                        }
                        if (f.kind == kApply && f.last) {
                            __nv_bfloat16 *to = p.out + ((int64_t)z * p.m + i) * p.n + j;
                            if (p.out_vec && left >= 8) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e] * (1.f / kScale),
                                                                                   v[2 * e + 1] * (1.f / kScale));
                                    w[e] = *reinterpret_cast<const uint32_t *>(&b);
                                }
                                *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    if (e < left) to[e] = __float2bfloat16_rn(v[e] * (1.f / kScale));
                            }
                            continue;
                        }
                        __half h[8], l[8];
                        split8(v, h, l);
                        store8(dst[0] + at0 + e0, h, left);
                        store8(dst[1] + at0 + e0, l, left);
                        if (mirror) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                if (e >= left) break;
                                const int64_t back = ((int64_t)z * f.M + j + e) * ld + i;
                                dst[0][back] = h[e];
                                dst[1][back] = l[e];
                            }
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty0 + 8 * acc);
            }
        }
        go = grid_barrier(p, target += gridDim.x, shared_ok);
    }
    if (warp == 0 && lane == 0) {  // after an error, copies may still be in flight: they land before the CTA exits
        for (int64_t i = slots > SLOTS ? slots - SLOTS : 0; i < slots; ++i) {
            const unsigned long long t0 = globaltimer();
            while (!mbar_try_wait(full0 + 8 * (int)(i % SLOTS), (uint32_t)((i / SLOTS) & 1)) &&
                   globaltimer() - t0 < kWaitTimeoutNs) {
            }
        }
    }
    if (warp == 1 && lane == 0) {  // every MMA completes before TMEM is released
        mma_commit(drain);
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(drain, 0) && globaltimer() - t0 < kWaitTimeoutNs) {
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// --------------------------------------------------------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn() {
    static std::once_flag once;
    static EncodeTiled fn = nullptr;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(ptr);
    });
    return fn;
}

// A batch of rows x cols fp16 matrices in boxes of 64 x 64, 128-byte swizzle, zero outside each matrix.
int matrix_map(CUtensorMap *m, const __half *base, int batch, int rows, int cols, int64_t ld) {
    EncodeTiled enc = encode_fn();
    if (enc == nullptr) {
        set_error("lamq_newton_schulz: cuTensorMapEncodeTiled is unavailable");
        return LAMQ_ERR_CUDA;
    }
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * (cuuint64_t)rows};
    const cuuint32_t box[3] = {64, 64, 1}, step[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(base), dims, strides, box, step,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("lamq_newton_schulz: cuTensorMapEncodeTiled failed (%d)", (int)r);
        return LAMQ_ERR_CUDA;
    }
    return LAMQ_OK;
}

int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

int parts_of(int batch) { return std::max(1, kParts / batch); }

struct Layout {
    size_t x, square, partial, total;  // bytes of one X, of one A or B, of the partial sums, and of all
};

Layout layout_of(int batch, int m, int n) {
    Layout L;
    const int s = std::min(m, n);
    L.x = up256((size_t)batch * m * up8(n) * 2);
    L.square = up256((size_t)batch * s * up8(s) * 2);
    L.partial = up256((size_t)batch * parts_of(batch) * 8);
    L.total = 4 * L.x + 4 * L.square + L.partial + 256;
    return L;
}

int cuda_failed(cudaError_t e) {
    set_error("lamq_newton_schulz: %s", cudaGetErrorString(e));
    return LAMQ_ERR_CUDA;
}

template <int BN>
int launch(Maps &maps, Params &p, int grid, cudaStream_t s) {
    const void *k = (const void *)newton_schulz_kernel<BN>;
    cudaError_t e = smem_limit_once(k, (int)Tile<BN>::SMEM);
    void *args[] = {&maps, &p};
    if (e == cudaSuccess) e = cudaLaunchCooperativeKernel(k, dim3(grid), dim3(kThreads), args, Tile<BN>::SMEM, s);
    if (e != cudaSuccess) return cuda_failed(e);
    LAMQ_CHECK_LAUNCH("lamq_newton_schulz");
    return LAMQ_OK;
}

}  // namespace
}  // namespace lamq

using namespace lamq;

extern "C" size_t lamq_newton_schulz_workspace_size(int batch, int m, int n) {
    if (batch <= 0 || m <= 0 || n <= 0) return 0;
    return layout_of(batch, m, n).total;
}

extern "C" int lamq_newton_schulz(const void *G, int dtype, int64_t ldg, int64_t batch_stride, int batch, int m, int n,
                                  int steps, const float *coefficients, float eps, uint16_t *out, void *workspace,
                                  size_t workspace_bytes, int *status, lamq_stream_t stream) {
    LAMQ_REQUIRE(batch >= 0 && m >= 0 && n >= 0 && ldg >= n, "lamq_newton_schulz: bad shape");
    LAMQ_REQUIRE(dtype == LAMQ_F32 || dtype == LAMQ_BF16, "lamq_newton_schulz: dtype must be LAMQ_F32 or LAMQ_BF16");
    LAMQ_REQUIRE(steps >= 1 && steps <= kMaxSteps, "lamq_newton_schulz: 1 to %d steps (got %d)", kMaxSteps, steps);
    LAMQ_REQUIRE(eps >= 0.f && eps < INFINITY, "lamq_newton_schulz: eps must not be negative");
    LAMQ_REQUIRE(batch <= 65535 && m <= (1 << 24) && n <= (1 << 24) && (double)batch * m * n <= 1e10,
                 "lamq_newton_schulz: the batch is too large");
    if (batch == 0 || m == 0 || n == 0) return LAMQ_OK;
    LAMQ_REQUIRE(batch == 1 || batch_stride >= (int64_t)(m - 1) * ldg + n, "lamq_newton_schulz: matrices overlap");
    LAMQ_REQUIRE(G && coefficients && out && status, "lamq_newton_schulz: null pointer");
    const Layout L = layout_of(batch, m, n);
    LAMQ_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= L.total,
                 "lamq_newton_schulz: workspace of %zu bytes (16-byte aligned) needed, %zu given", L.total,
                 workspace_bytes);
    Params p{};
    // singular values start within [0, 1]: the polynomials must keep them, and B, within what fp16 holds
    double top = 1.0;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0, big = 0.0;
        for (int e = 0; e < 3; ++e) p.coef[k][e] = coefficients[3 * k + e];
        for (int i = 0; i <= 1024; ++i) {
            const double x = top * i / 1024, q = p.coef[k][0] + x * x * (p.coef[k][1] + x * x * p.coef[k][2]);
            big = std::max(big, q < 0 ? -q : q);
            next = std::max(next, (q < 0 ? -q : q) * x);
        }
        LAMQ_REQUIRE(p.coef[k][0] + p.coef[k][1] + p.coef[k][2] == p.coef[k][0] + p.coef[k][1] + p.coef[k][2] &&
                         big <= 32.0 && next <= 5.0,
                     "lamq_newton_schulz: the coefficients of step %d leave the range (singular values up to 5, the "
                     "polynomial of A up to 32)", k);
        top = std::max(1.0, next);
    }
    cudaStream_t s = (cudaStream_t)stream;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);  // binds the context for the driver call that makes the tensor maps
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_failed(e);
    p.G = G;
    p.ldg = ldg;
    p.gbatch = batch_stride;
    p.g_bf16 = dtype == LAMQ_BF16;
    const int64_t piece = p.g_bf16 ? 8 : 4;
    p.g_vec = (uintptr_t)G % 16 == 0 && ldg % piece == 0 && (batch == 1 || batch_stride % piece == 0);
    p.out = reinterpret_cast<__nv_bfloat16 *>(out);
    p.out_vec = (uintptr_t)out % 16 == 0 && n % 8 == 0;
    p.batch = batch;
    p.m = m;
    p.n = n;
    p.tall = m > n;
    p.s = std::min(m, n);
    p.l = std::max(m, n);
    p.ldx = up8(n);
    p.lds = up8(p.s);
    p.parts = parts_of(batch);
    p.eps = eps;
    p.steps = steps;
    p.status = status;
    char *ws = reinterpret_cast<char *>(workspace);
    Maps maps;
    for (int i = 0; i < 2; ++i) {
        for (int q = 0; q < 2; ++q) {
            p.x[i][q] = reinterpret_cast<__half *>(ws + (2 * i + q) * L.x);
            if (int st = matrix_map(&maps.x[i][q], p.x[i][q], batch, m, n, p.ldx)) return st;
        }
        p.gram[i] = reinterpret_cast<__half *>(ws + 4 * L.x + i * L.square);
        p.poly[i] = reinterpret_cast<__half *>(ws + 4 * L.x + (2 + i) * L.square);
        if (int st = matrix_map(&maps.gram[i], p.gram[i], batch, p.s, p.s, p.lds)) return st;
        if (int st = matrix_map(&maps.poly[i], p.poly[i], batch, p.s, p.s, p.lds)) return st;
    }
    p.partial = reinterpret_cast<double *>(ws + 4 * L.x + 4 * L.square);
    p.barrier = reinterpret_cast<unsigned *>(ws + 4 * L.x + 4 * L.square + L.partial);
    e = cudaMemsetAsync(p.barrier, 0, sizeof(unsigned), s);
    if (e != cudaSuccess) return cuda_failed(e);
    // The wide tiles have the better ratio of products to operand bytes; the narrow ones a quarter of the latency. Wide
    // ones as soon as the larger phase (B·X) fills the device with them.
    const int64_t ts = (p.s + BM - 1) / BM, tl = (p.l + BM - 1) / BM;
    const bool wide = (int64_t)batch * (p.tall ? tl * ((p.s + 255) / 256) : ts * ((p.l + 255) / 256)) >= sms;
    // a CTA per tile of the phase with the most of them, at most one per SM
    const int grid = (int)std::min<int64_t>(sms, std::max<int64_t>((int64_t)batch * ts * tl * 2,
                                                                  std::min<int64_t>(sms, (int64_t)m * n / 4096 + 1)));
    return wide ? launch<256>(maps, p, grid, s) : launch<64>(maps, p, grid, s);
}
