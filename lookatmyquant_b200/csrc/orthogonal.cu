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
// of saturated directions would go on adding up, and everything where the shorter side is 128 at most: with few directions
// single products came to 2.7e-3 (198 x 21), and those products are short (70 x 458: 154 us so, 140 with single ones). In
// simulation (64 x 2000 .. 500 x 520; Gaussian, low-rank, power-law, row-scaled updates) this leaves 2e-4 .. 1.8e-3 of
// relative error beside 1.65e-3 of the bf16 output's
// rounding; three products everywhere leave 1e-5 for 2.6 times the work, single ones 4e-3. That is for steps that multiply a
// rounding by 4 (Muon's, the largest derivative of the step's polynomial) to 8. Steeper schedules take three products
// everywhere: for one that begins with (8.287, -23.596, 17.3), a derivative of 24, the model gives 2.1e-3 to 5.2e-3 otherwise
// (150 x 2000 the worst). Everything is held times
// kScale = 2^10, which keeps entries of order 1/max(m, n) clear of fp16's subnormals and the largest (singular values
// up to 5, B up to 32) below its maximum. Accumulation is fp32 in TMEM.
//
// One persistent cooperative kernel runs all phases (sum of squares, X_0, then A, B, X per step) with a grid barrier
// between two of them: a small matrix would otherwise spend its time in launches. A phase's products are tiles of
// 256 x 256 on pairs of CTAs, or of 128 x 128 on single ones where the larger would leave SMs idle, handed out over the
// device. A and B are symmetric: of the large tiles only those that reach the diagonal are computed, and each is also
// written mirrored. Operands are read by TMA in the major order in which they lie, so nothing is transposed in memory.
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
#include "give_up.cuh"
#include "lamq_common.cuh"
#include "sm100.cuh"

namespace lamq {
namespace {

using namespace sm100;

constexpr int BM = 128, BK = 64;
constexpr int BOX = 64 * 128;                    // bytes of a 64 x 64 fp16 box

template <int BN>
struct Tile {
    static constexpr bool PAIR = BN == 256;              // two CTAs (a cluster) compute 256 x 256 with cta_group::2 MMAs
    static constexpr int ROWS = PAIR ? 256 : 128;        // of a tile
    static constexpr int A_BYTES = 2 * BOX, B_BYTES = 2 * BOX;  // a CTA loads 128 rows of either operand
    static constexpr int SLOT = A_BYTES + B_BYTES;       // the hi (or the lo) operands of 64 entries of K
    static constexpr int SLOTS = 6;                      // the ring; split products take two slots a step
    static constexpr int STAGING = 8 * 32 * 128;         // the epilogue warps': 32 rows of 64 fp16 each
    static constexpr size_t SMEM = SLOTS * SLOT + STAGING + 512;
    static constexpr int EPI = BN / 2;                   // columns per epilogue warp
    static constexpr bool HALF = PAIR;                   // of A and B only the tiles that reach the diagonal (the narrow
                                                         // tiles leave SMs idle: mirroring would cost more than it saves)
};

constexpr int kThreads = 320;
constexpr uint32_t kTmemCols = 512;
constexpr float kScale = 1024.f;
constexpr int kMaxSteps = 16;
constexpr double kSteep = 9.0;                   // the derivative of a step's polynomial from which single products are too few
constexpr int kParts = 296;                      // parts of a batch in the sum of squares, at most
constexpr int kSplitUnits = 148;                 // pieces of A's products over all of K, at most

struct Maps {
    CUtensorMap x[2][2];     // X of even and odd steps, hi and lo: boxes of 128 rows by 64 columns
    CUtensorMap xt[2][2];    // the same in boxes of 64 rows by two blocks of 64 columns: X as the transposed operand
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
    int64_t ldx, lds;     // leading dimensions of X (m x n) and of A and B (s x s): whole 64s, zeros past the end
    __half *x[2][2], *gram[2], *poly[2];
    double *partial;      // batch x parts sums of squares
    int parts;
    float *pieces;        // A's tiles over a part of K each (ksplit > 1), columns of 128 rows
    int ksplit;
    float eps;
    int steps;
    float coef[kMaxSteps][3];
    int exact;            // three products everywhere
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
    const int c = ((tj + 1) * BN - 1) / Tile<BN>::ROWS + 1;
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
    f.split = f.kind == kPoly || step > 4 || p.s <= BM || p.exact || (f.kind == kApply && (step == 4 || f.last));
    f.M = f.kind == kApply && p.tall ? p.l : p.s;
    f.N = f.kind == kApply && !p.tall ? p.l : p.s;
    f.K = f.kind == kGram ? p.l : p.s;
    f.a_mn = f.kind == kGram && p.tall;
    f.b_mn = (f.kind == kGram && p.tall) || (f.kind == kApply && !p.tall);
    f.tm = (f.M + Tile<BN>::ROWS - 1) / Tile<BN>::ROWS;
    f.tn = (f.N + BN - 1) / BN;
    f.tiles = f.kind == kApply || !Tile<BN>::HALF ? f.tm * f.tn : symmetric_tiles<BN>(f.tm, f.tn);
    return f;
}

// Unit u: matrix z, tile (ti, tj). The tiles that share rows or columns of X follow one another.
template <int BN>
__device__ __forceinline__ void tile_of(const Params &p, const Phase &f, int u, int &z, int &ti, int &tj) {
    z = u / f.tiles;
    int t = u - z * f.tiles;
    if (f.kind == kApply || !Tile<BN>::HALF) {
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

// Every CTA has finished the phase and what it wrote is visible to all, to TMA too. Bounded: false when it or
// another wait of the launch gives up.
__device__ __forceinline__ bool grid_barrier(const Params &p, unsigned target, int *shared_ok) {
    asm volatile("fence.proxy.async.global;" ::: "memory");  // this thread's writes before other SMs' TMA reads
    __syncthreads();
    if (threadIdx.x == 0) {
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.barrier) : "memory");
        const unsigned long long t0 = globaltimer();
        int ok = 1;
        for (unsigned it = 1;; ++it) {
            unsigned v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p.barrier) : "memory");
            if (v >= target) break;
            if (it % LAMQ_GIVE_UP_POLLS == 0u) {
                if (launch_gave_up()) ok = 0;
                else if (globaltimer() - t0 > LAMQ_GIVE_UP_NS) {
                    give_up(p.status);
                    ok = 0;
                }
                if (!ok) break;
            }
        }
        *shared_ok = ok;
    }
    __syncthreads();
    asm volatile("fence.proxy.async.global;" ::: "memory");
    return *shared_ok != 0;
}

// A word of another CTA's shared memory.
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
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
__device__ __forceinline__ void split8(const float *v, uint4 &hi, uint4 &lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __half2 a = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
        const float2 f = __half22float2(a);
        const __half2 b = __floats2half2_rn(v[2 * e] - f.x, v[2 * e + 1] - f.y);
        h[e] = *reinterpret_cast<const uint32_t *>(&a);
        l[e] = *reinterpret_cast<const uint32_t *>(&b);
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// v[e] += the eight fp16 of q.
__device__ __forceinline__ void add8(uint4 q, float *v) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
        v[2 * e] += f.x;
        v[2 * e + 1] += f.y;
    }
}

// A warp's 32 x 64 block of 16-bit values between rows (a lane holds a row) and pieces of 16 bytes in memory order (a
// warp's access covers whole 128-byte rows: a lane's own row in 16-byte stores took 14,000 cycles a tile). Piece c of
// row r lies at c ^ (r mod 8).
__device__ __forceinline__ uint4 *staged(uint8_t *buf, int row, int c) {
    return reinterpret_cast<uint4 *>(buf + row * 128 + ((c ^ (row & 7)) << 4));
}

// Rows [0, rows) of the block at `base` into the lanes' pieces (piece i of a lane: row 4i + lane / 8, piece lane % 8).
__device__ __forceinline__ void load_block(const __half *base, int64_t ld, int rows, uint4 (&q)[8]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        q[i] = r < rows ? *reinterpret_cast<const uint4 *>(base + r * ld + 8 * (lane & 7)) : make_uint4(0, 0, 0, 0);
    }
}

__device__ __forceinline__ void pieces_to_rows(uint8_t *buf, const uint4 (&q)[8], float (&v)[64]) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) *staged(buf, 4 * i + (lane >> 3), lane & 7) = q[i];
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) add8(*staged(buf, lane, c), v + 8 * c);
}

// The lanes' rows (8 pieces each) to the block at `base`.
template <typename T>
__device__ __forceinline__ void store_block(uint8_t *buf, const uint4 (&q)[8], T *base, int64_t ld, int rows) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) *staged(buf, lane, c) = q[c];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        if (r < rows) *reinterpret_cast<uint4 *>(base + r * ld + 8 * (lane & 7)) = *staged(buf, r, lane & 7);
    }
}

// The same block transposed: 64 rows (of which `rows` exist) of 32 values (pieces up to column `cols`).
__device__ __forceinline__ void store_transposed(uint8_t *buf, const uint4 (&q)[8], __half *base, int64_t ld, int rows,
                                                 int cols) {
    const int lane = threadIdx.x & 31;
    uint16_t *t = reinterpret_cast<uint16_t *>(buf) + lane;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            t[(8 * c + 2 * e) * 32] = (uint16_t)w[e];
            t[(8 * c + 2 * e + 1) * 32] = (uint16_t)(w[e] >> 16);
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 8 * i + (lane >> 2), c = 8 * (lane & 3);
        if (r < rows && c < cols)
            *reinterpret_cast<uint4 *>(base + r * ld + c) = *reinterpret_cast<const uint4 *>(buf + r * 64 + 2 * c);
    }
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
    newton_schulz_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
    using Z = Tile<BN>;
    constexpr int SLOT = Z::SLOT, SLOTS = Z::SLOTS, A_BYTES = Z::A_BYTES, EPI = Z::EPI;
    constexpr bool PAIR = Z::PAIR;
    const int rank = PAIR ? (int)cluster_rank() : 0, worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;  // what computes tiles: pairs, or CTAs
    extern __shared__ __align__(1024) uint8_t smem[];  // swizzled boxes start at multiples of 1024 bytes
    uint8_t *const staging = smem + SLOTS * SLOT;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + Z::STAGING);
    double *red = reinterpret_cast<double *>(bars + 2 * SLOTS + 6);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(red + kThreads / 32);
    int *shared_ok = reinterpret_cast<int *>(tmem_holder + 1);
    uint32_t *issued = tmem_holder + 2;  // slots that this CTA's loads have taken, at the end
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + SLOTS);
    const uint32_t tfull0 = smem_u32(bars + 2 * SLOTS), tempty0 = tfull0 + 16, drain = tfull0 + 32;
    const uint32_t ring = smem_u32(smem);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * SLOTS; ++i) mbar_init(full0 + 8 * i, 1);
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull0 + 8 * a, 1);
            mbar_init(tempty0 + 8 * a, PAIR ? 16 : 8);  // a pair's warps all arrive on the even CTA's
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        for (int i = 0; i < 2; ++i) {
            for (int q = 0; q < 2; ++q) {
                prefetch_tmap(&maps.x[i][q]);
                prefetch_tmap(&maps.xt[i][q]);
            }
            prefetch_tmap(&maps.gram[i]);
            prefetch_tmap(&maps.poly[i]);
        }
    }
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(smem_u32(tmem_holder), kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_holder), kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();  // both CTAs' barriers exist before either signals the other
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    unsigned target = 0;

    // ---- |G|_F: fixed parts of each matrix, summed in 64 bits; then X_0 by the same parts
    const uint32_t row_groups = (uint32_t)(p.ldx / 8), groups = (uint32_t)p.m * row_groups;
    for (int u = blockIdx.x; u < p.batch * p.parts; u += gridDim.x) {
        const int z = u / p.parts, part = u % p.parts;
        const uint32_t g1 = (uint32_t)((uint64_t)groups * (part + 1) / p.parts);
        double acc = 0.0;
        for (uint32_t g = (uint32_t)((uint64_t)groups * part / p.parts) + threadIdx.x; g < g1; g += kThreads) {
            const uint32_t r = g / row_groups;
            float v[8];
            load_g8(p, z, (int)r, (int)(g - r * row_groups) * 8, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc += (double)v[e] * (double)v[e];
        }
        acc = block_sum(acc, red);
        if (threadIdx.x == 0) p.partial[u] = acc;
    }
    bool go = grid_barrier(p, target += gridDim.x, shared_ok);
    for (int u = blockIdx.x; go && u < p.batch * p.parts; u += gridDim.x) {
        const int z = u / p.parts, part = u % p.parts;
        double acc = 0.0;
        for (int i = threadIdx.x; i < p.parts; i += kThreads)
            acc += *reinterpret_cast<volatile double *>(p.partial + (int64_t)z * p.parts + i);
        const double norm = sqrt(block_sum(acc, red)) + (double)p.eps;
        // in two factors where a tiny matrix's one is past fp32; a zero matrix without an eps stays zero
        const double factor = norm == 0.0 ? 0.0 : (double)kScale / norm;
        const float lift = factor > 1e38 ? 0x1p64f : 1.f, inv = (float)(factor / (double)lift);
        const uint32_t g1 = (uint32_t)((uint64_t)groups * (part + 1) / p.parts);
        for (uint32_t g = (uint32_t)((uint64_t)groups * part / p.parts) + threadIdx.x; g < g1; g += kThreads) {
            const uint32_t r = g / row_groups, c = (g - r * row_groups) * 8;
            float v[8];
            load_g8(p, z, (int)r, (int)c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * lift * inv;
            const int64_t at = ((int64_t)z * p.m + r) * p.ldx + c;
            split8(v, *reinterpret_cast<uint4 *>(p.x[0][0] + at), *reinterpret_cast<uint4 *>(p.x[0][1] + at));
        }
    }
    if (go) go = grid_barrier(p, target += gridDim.x, shared_ok);

    // ---- the products. Ring slots and accumulators are counted through all phases, by each role alike
    uint32_t slots = 0, accs = 0;
    bool ok = true;
    for (int ph = 0; go && ph < 3 * p.steps; ++ph) {
        const Phase f = phase_of<BN>(p, ph);
        const int step = ph / 3, cur = step & 1, parts = f.split ? 2 : 1;
        const int kblocks = (f.K + BK - 1) / BK;
        const int splits = !Z::HALF && f.kind == kGram ? p.ksplit : 1, units = p.batch * f.tiles * splits;
        const auto k_range = [&](int u, int &k0, int &k1) {
            const int part = Z::HALF ? 0 : u % splits;
            k0 = Z::HALF ? 0 : kblocks * part / splits;
            k1 = Z::HALF ? kblocks : kblocks * (part + 1) / splits;
        };
        if (warp == 0) {
            if (lane == 0) {  // ---- TMA producer
                const CUtensorMap *ma = f.a_mn                                          ? maps.xt[cur]
                                        : f.kind == kGram || (f.kind == kApply && p.tall) ? maps.x[cur]
                                        : f.kind == kPoly                               ? maps.gram
                                                                                        : maps.poly;
                const CUtensorMap *mb = f.b_mn                                          ? maps.xt[cur]
                                        : f.kind == kGram                               ? maps.x[cur]
                                        : f.kind == kPoly                               ? maps.gram
                                                                                        : maps.poly;
                for (int u = worker; ok && u < units; u += workers) {
                    int z, ti, tj, k0, k1;
                    tile_of<BN>(p, f, Z::HALF ? u : u / splits, z, ti, tj);
                    k_range(u, k0, k1);
                    for (int kb = k0; ok && kb < k1; ++kb)
                        for (int q = 0; q < parts; ++q, ++slots) {
                            const uint32_t st = slots % SLOTS;
                            ok = await(empty0 + 8 * st, ((slots / SLOTS) & 1) ^ 1, p.status);
                            if (!ok) break;
                            const uint32_t sa = ring + st * SLOT, sb = sa + A_BYTES, bar = full0 + 8 * st;
                            const int k = kb * BK, ra = ti * Z::ROWS + 128 * rank, rb = tj * BN + 128 * rank;
                            // two boxes of 16 KiB (six of 8 KiB kept the issuing thread behind the tensor core). A pair's
                            // loads all complete on the even CTA's barrier
                            if (PAIR) {
                                const uint32_t pb = map_to_rank(bar, 0);
                                if (rank == 0) mbar_expect_tx(bar, 2 * SLOT);
                                if (f.a_mn) tma_load_4d_pair(sa, ma + q, 0, k, ra / 64, z, pb);
                                else tma_load_3d_pair(sa, ma + q, k, ra, z, pb);
                                if (f.b_mn) tma_load_4d_pair(sb, mb + q, 0, k, rb / 64, z, pb);
                                else tma_load_3d_pair(sb, mb + q, k, rb, z, pb);
                            } else {
                                mbar_expect_tx(bar, SLOT);
                                if (f.a_mn) tma_load_4d(sa, ma + q, 0, k, ra / 64, z, bar);
                                else tma_load_3d(sa, ma + q, k, ra, z, bar);
                                if (f.b_mn) tma_load_4d(sb, mb + q, 0, k, rb / 64, z, bar);
                                else tma_load_3d(sb, mb + q, k, rb, z, bar);
                            }
                        }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            if (lane == 0 && rank == 0) {  // ---- MMA issuer (of a pair: the even CTA)
                const uint32_t idesc = idesc_f16_f32(Z::ROWS, BN, f.a_mn, f.b_mn);
                const uint32_t a_step = (f.a_mn ? 2048 : 32) >> 4, b_step = (f.b_mn ? 2048 : 32) >> 4;  // descriptor units
                const uint32_t a_lbo = f.a_mn ? BOX : 16, b_lbo = f.b_mn ? BOX : 16;
                for (int u = worker; ok && u < units; u += workers, ++accs) {
                    const int acc = accs & 1;
                    ok = await(tempty0 + 8 * acc, ((accs >> 1) & 1) ^ 1, p.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + acc * BN;
                    int k0, k1;
                    k_range(u, k0, k1);
                    for (int kb = k0; ok && kb < k1; ++kb, slots += parts) {
                        uint64_t da[2], db[2];
                        for (int q = 0; q < parts; ++q) {
                            const uint32_t st = (slots + q) % SLOTS;
                            ok = ok && await(full0 + 8 * st, ((slots + q) / SLOTS) & 1, p.status);
                            da[q] = smem_desc_sw128(ring + st * SLOT, a_lbo, 1024);
                            db[q] = smem_desc_sw128(ring + st * SLOT + A_BYTES, b_lbo, 1024);
                        }
                        if (!ok) break;
                        tc_fence_after();
                        const auto product = [&](int qa, int qb, bool first) {
#pragma unroll
                            for (int kk = 0; kk < BK / 16; ++kk) {
                                const uint64_t ad = da[qa] + kk * a_step, bd = db[qb] + kk * b_step;
                                const uint32_t add = first && kk == 0 ? 0u : 1u;
                                if (PAIR) mma_f16_ss_pair(d, ad, bd, idesc, add);
                                else mma_f16_ss(d, ad, bd, idesc, add);
                            }
                        };
                        product(0, 0, kb == k0);
                        if (f.split) {
                            product(0, 1, false);
                            product(1, 0, false);
                        }
                        for (int q = 0; q < parts; ++q) {
                            const uint32_t bar = empty0 + 8 * ((slots + q) % SLOTS);
                            if (PAIR) mma_commit_pair_multicast(bar, 0x3);
                            else mma_commit(bar);
                        }
                    }
                    if (ok) {
                        if (PAIR) mma_commit_pair_multicast(tfull0 + 8 * acc, 0x3);
                        else mma_commit(tfull0 + 8 * acc);
                    }
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
            for (int u = worker; ok && u < units; u += workers, ++accs) {
                int z, ti, tj;
                tile_of<BN>(p, f, Z::HALF ? u : u / splits, z, ti, tj);
                const int acc = accs & 1;
                const int i0 = ti * Z::ROWS + 128 * rank + 32 * quad, i = i0 + lane, j0 = tj * BN + EPI * half;
                const int rows = f.M - i0;  // of the warp's 32 that exist
                uint4 early_h[8], early_l[8];
                // the exact terms' operands come while the products run (a wide tile's warps are busy with the last tile)
                if (!Z::HALF && f.kind != kGram && rows > 0 && j0 < ld) {
                    const int64_t at0 = ((int64_t)z * f.M + i0) * ld + j0;
                    load_block(old[0] + at0, ld, rows, early_h);
                    load_block(old[1] + at0, ld, rows, early_l);
                }
                ok = __all_sync(0xffffffffu, await(tfull0 + 8 * acc, (accs >> 1) & 1, p.status));
                if (!ok) break;
                tc_fence_after();
                // (j, i) lies in no computed tile (EPI columns share a row tile, a warp's rows a column tile)
                const bool mirror = Z::HALF && f.kind != kApply && j0 / Z::ROWS >= column_tiles<BN>(f.tm, i0 / BN);
                const uint32_t t = tmem + ((uint32_t)(32 * quad) << 16) + acc * BN + EPI * half;
                if (!Z::HALF && splits > 1) {  // the piece as it is, column by column
                    float *const piece = p.pieces + ((int64_t)u * BN + EPI * half) * BM + 32 * quad + lane;
#pragma unroll 1
                    for (int c = 0; c < EPI; c += 32) {
                        uint32_t r[32];
                        tmem_load32(t + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) piece[(int64_t)(c + e) * BM] = __uint_as_float(r[e]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty0 + 8 * acc);
                    continue;
                }
                uint8_t *const buf = staging + (warp - 2) * 4096;
#pragma unroll 1
                for (int c = 0; c < EPI; c += 64) {
                    if (j0 + c >= ld || rows <= 0) break;
                    const int64_t at0 = ((int64_t)z * f.M + i0) * ld + j0 + c;
                    uint4 qh[8], ql[8];
                    float v[64];
#pragma unroll
                    for (int e = 0; e < 64; ++e) v[e] = 0.f;
                    if (f.kind != kGram) {
                        static_assert(Z::HALF || EPI == 64, "a narrow tile's warp has one block of columns");
                        if (Z::HALF) {
                            load_block(old[0] + at0, ld, rows, qh);
                            load_block(old[1] + at0, ld, rows, ql);
                        }
                        pieces_to_rows(buf, Z::HALF ? qh : early_h, v);
                        pieces_to_rows(buf, Z::HALF ? ql : early_l, v);
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t r[32];
                        tmem_load32(t + c + 32 * g, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            v[32 * g + e] = fmaf(f_old, v[32 * g + e], __uint_as_float(r[e]) * f_acc);
                    }
                    if (f.kind == kApply && f.last) {
                        __nv_bfloat16 *to = p.out + ((int64_t)z * p.m + i0) * p.n + j0 + c;
                        if (p.out_vec && j0 + c + 64 <= p.n) {
#pragma unroll
                            for (int g = 0; g < 8; ++g) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * g + 2 * e] * (1.f / kScale),
                                                                                   v[8 * g + 2 * e + 1] * (1.f / kScale));
                                    w[e] = *reinterpret_cast<const uint32_t *>(&b);
                                }
                                qh[g] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                            store_block(buf, qh, to, p.n, rows);
                        } else if (i < f.M) {
#pragma unroll
                            for (int e = 0; e < 64; ++e)
                                if (j0 + c + e < p.n) to[(int64_t)lane * p.n + e] = __float2bfloat16_rn(v[e] * (1.f / kScale));
                        }
                        continue;
                    }
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        split8(v + 8 * g, qh[g], ql[g]);
                    }
                    store_block(buf, qh, dst[0] + at0, ld, rows);
                    store_block(buf, ql, dst[1] + at0, ld, rows);
                    if (mirror) {
                        const int64_t back = ((int64_t)z * f.M + j0 + c) * ld + i0;
                        store_transposed(buf, qh, dst[0] + back, ld, f.M - j0 - c, (int)ld - i0);
                        store_transposed(buf, ql, dst[1] + back, ld, f.M - j0 - c, (int)ld - i0);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (rank) mbar_arrive_cluster(map_to_rank(tempty0 + 8 * acc, 0));
                    else mbar_arrive(tempty0 + 8 * acc);
                }
            }
        }
        if (!Z::HALF && splits > 1) {  // the pieces added in order; A is symmetric, so its columns are written as rows
            go = grid_barrier(p, target += gridDim.x, shared_ok);
            const int total = p.batch * f.tiles * BN * (BM / 4);
            for (int e = blockIdx.x * kThreads + threadIdx.x; go && e < total; e += gridDim.x * kThreads) {
                const int row = e % (BM / 4) * 4, col = e / (BM / 4) % BN, tile = e / (BM / 4 * BN);
                int z, ti, tj;
                tile_of<BN>(p, f, tile, z, ti, tj);
                const int i = ti * BM + row, j = tj * BN + col;
                if (j >= f.M || i >= p.lds) continue;  // (lds is a multiple of four)
                const float *piece = p.pieces + ((int64_t)tile * splits * BN + col) * BM + row;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                for (int q = 0; q < splits; ++q) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(piece + (int64_t)q * BN * BM));
                    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
                }
                const float v[8] = {acc.x / kScale, acc.y / kScale, acc.z / kScale, acc.w / kScale, 0.f, 0.f, 0.f, 0.f};
                uint4 hi, lo;
                split8(v, hi, lo);
                const int64_t at = ((int64_t)z * f.M + j) * p.lds + i;
                *reinterpret_cast<uint2 *>(p.gram[0] + at) = make_uint2(hi.x, hi.y);
                *reinterpret_cast<uint2 *>(p.gram[1] + at) = make_uint2(lo.x, lo.y);
            }
        }
        if (go) go = grid_barrier(p, target += gridDim.x, shared_ok);
    }
    // Copies that were issued land before their CTA leaves, also where an error, of any thread, ended a phase before they were
    // waited for.
    const auto landed = [&](uint32_t i) {
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(full0 + 8 * (i % SLOTS), (i / SLOTS) & 1) && globaltimer() - t0 < kWaitTimeoutNs) {
        }
    };
    if (threadIdx.x == 0) {
        *issued = slots;
        for (uint32_t i = slots > SLOTS ? slots - SLOTS : 0; !PAIR && i < slots; ++i) landed(i);
    }
    if (warp == 1 && lane == 0 && rank == 0) {  // every MMA completes before TMEM is released
        if (PAIR) mma_commit_pair(drain);
        else mma_commit(drain);
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(drain, 0) && globaltimer() - t0 < kWaitTimeoutNs) {
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (PAIR) {  // neither CTA leaves while the pair's MMAs, arrivals or copies may still touch it
        cluster_sync_all();
        if (rank == 0 && threadIdx.x == 0) {  // all copies are counted on this CTA's barriers, where both took part
            const uint32_t other = load_cluster(map_to_rank(smem_u32(issued), 1)), most = other > slots ? other : slots;
            for (uint32_t i = most > SLOTS ? most - SLOTS : 0; i < most; ++i) {
                const uint32_t bar = full0 + 8 * (i % SLOTS);
                if (i >= slots) mbar_expect_tx(bar, SLOT);        // the odd CTA's half alone
                else if (i >= other) mbar_complete_tx(bar, SLOT);  // this CTA's half alone
                landed(i);
            }
        }
        cluster_sync_all();
    }
    tc_fence_after();
    if (warp == 1) {
        if (PAIR) tmem_dealloc_pair(tmem, kTmemCols);
        else tmem_dealloc(tmem, kTmemCols);
    }
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

// A batch of rows x ld fp16 matrices, 128-byte swizzle, zero past the rows: boxes of 128 rows by 64 columns, or (blocks)
// of 64 rows by two blocks of 64 columns, one block after the other.
int matrix_map(CUtensorMap *m, const __half *base, int batch, int rows, int64_t ld, bool blocks) {
    EncodeTiled enc = encode_fn();
    if (enc == nullptr) {
        set_error("lamq_newton_schulz: cuTensorMapEncodeTiled is unavailable");
        return LAMQ_ERR_CUDA;
    }
    const cuuint64_t row = (cuuint64_t)ld * 2, all = row * (cuuint64_t)rows;
    const cuuint64_t dims3[3] = {(cuuint64_t)ld, (cuuint64_t)rows, (cuuint64_t)batch}, strides3[2] = {row, all};
    const cuuint64_t dims4[4] = {64, (cuuint64_t)rows, (cuuint64_t)ld / 64, (cuuint64_t)batch}, strides4[3] = {row, 128, all};
    const cuuint32_t box3[3] = {64, 128, 1}, box4[4] = {64, 64, 2, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, blocks ? 4 : 3, const_cast<__half *>(base),
                           blocks ? dims4 : dims3, blocks ? strides4 : strides3, blocks ? box4 : box3, step,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("lamq_newton_schulz: cuTensorMapEncodeTiled failed (%d)", (int)r);
        return LAMQ_ERR_CUDA;
    }
    return LAMQ_OK;
}

int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

int64_t tiles_of(int64_t n, int tile) { return (n + tile - 1) / tile; }

// How a batch of m x n matrices is cut up: by its sizes alone, so that equal calls sum in equal order everywhere.
struct Plan {
    bool wide;     // tiles of 256 x 256 on pairs of CTAs, else of 128 x 128
    int parts;     // of each matrix in the sum of squares
    int ksplit;    // parts of K in A's products
    size_t x, square, partial, pieces, total;  // bytes of one X, of one A or B, of the partial sums, the pieces, and all
};

Plan plan_of(int batch, int m, int n) {
    Plan L;
    const int s = std::min(m, n), l = std::max(m, n);
    // The wide tiles have the better ratio of products to operand bytes (single CTAs of 128 x 256 waited for L2: 9728 x
    // 2560 took 1.57 ms), the narrow ones half of the latency (narrower still would not: an MMA of 64 columns takes as
    // long as one of 128) and their sums for A can be cut. Wide ones where the larger phase (B·X) gives every pair of SMs a
    // tile, A has 15 of them or more, each of which sums over all of K on one pair, and s fills more than half of one.
    // Measured, us (narrow, wide): 2560 x 2560 1245, 695; 4 x 960 x 2560 681, 518; 1280 x 9728 915, 796; 80 x 130 x 200 286,
    // 245; and where A has few tiles 960 x 9728 621, 715; 512 x 9728 294, 579; 2 x 16 x 9728 159, 770; 64 x 131072 357, 8849;
    // or s is mostly padding 300 x 20 x 24 185, 239. (Near the rule's edges it is up to 8 % off: 2 x 960 x 2560 409, 428; 16 x
    // 320 x 960 243, 262; and 1600 x 1600, with 49 tiles in B·X, 582, 417.)
    const int64_t st = tiles_of(s, 256);
    L.wide = batch * tiles_of(l, 256) * st >= kSplitUnits / 2 && batch * st * (st + 1) / 2 >= 15 && s > BM;
    L.parts = (int)std::max<int64_t>(1, std::min<int64_t>(kParts / batch, (int64_t)m * up64(n) / 16384));
    // A is s x s over K = l: of a skinny matrix few tiles, each a long sum. Cut K, in parts of four steps or more, where
    // SMs would be idle (16 x 9728: 152 steps of some 700 cycles on one SM otherwise)
    const int64_t tiles = batch * tiles_of(s, BM) * tiles_of(s, 128), steps = tiles_of(l, BK);
    L.ksplit = L.wide ? 1 : (int)std::max<int64_t>(1, std::min(kSplitUnits / tiles, steps / 4));
    L.x = up256((size_t)batch * m * up64(n) * 2);
    L.square = up256((size_t)batch * s * up64(s) * 2);
    L.partial = up256((size_t)batch * L.parts * 8);
    L.pieces = L.ksplit > 1 ? (size_t)tiles * L.ksplit * BM * 128 * 4 : 0;
    L.total = 4 * L.x + 4 * L.square + L.partial + L.pieces + 256;
    return L;
}

int cuda_failed(cudaError_t e) {
    set_error("lamq_newton_schulz: %s", cudaGetErrorString(e));
    return LAMQ_ERR_CUDA;
}

template <int BN>
int launch(Maps &maps, Params &p, int grid, cudaStream_t s) {
    const auto k = newton_schulz_kernel<BN>;
    cudaError_t e = smem_limit_once((const void *)k, (int)Tile<BN>::SMEM);
    if (e != cudaSuccess) return cuda_failed(e);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Tile<BN>::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = Tile<BN>::PAIR ? 2 : 1;
    if (Tile<BN>::PAIR) {  // pairs that fit at once
        int pairs = 0;
        cfg.attrs = attr + 1;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&pairs, (const void *)k, &cfg);
        if (e != cudaSuccess) return cuda_failed(e);
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        cfg.gridDim = dim3((unsigned)std::min(grid / 2, pairs) * 2);
    }
    e = cudaLaunchKernelEx(&cfg, k, maps, p);
    if (e != cudaSuccess) return cuda_failed(e);
    LAMQ_CHECK_LAUNCH("lamq_newton_schulz");
    return LAMQ_OK;
}

}  // namespace
}  // namespace lamq

using namespace lamq;

extern "C" size_t lamq_newton_schulz_workspace_size(int batch, int m, int n) {
    if (batch <= 0 || m <= 0 || n <= 0) return 0;
    return plan_of(batch, m, n).total;
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
    const Plan L = plan_of(batch, m, n);
    LAMQ_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= L.total,
                 "lamq_newton_schulz: workspace of %zu bytes (16-byte aligned) needed, %zu given", L.total,
                 workspace_bytes);
    Params p{};
    // singular values start within [0, 1]: the polynomials must keep them, and B, within what fp16 holds
    double top = 1.0, steepest = 0.0;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0, big = 0.0;
        for (int e = 0; e < 3; ++e) p.coef[k][e] = coefficients[3 * k + e];
        for (int i = 0; i <= 1024; ++i) {
            const double x = top * i / 1024, q = p.coef[k][0] + x * x * (p.coef[k][1] + x * x * p.coef[k][2]);
            big = std::max(big, q < 0 ? -q : q);
            next = std::max(next, (q < 0 ? -q : q) * x);
            const double slope = p.coef[k][0] + x * x * (3.0 * p.coef[k][1] + x * x * 5.0 * p.coef[k][2]);
            steepest = std::max(steepest, slope < 0 ? -slope : slope);
        }
        LAMQ_REQUIRE(p.coef[k][0] + p.coef[k][1] + p.coef[k][2] == p.coef[k][0] + p.coef[k][1] + p.coef[k][2] &&
                         big <= 32.0 && next <= 5.0,
                     "lamq_newton_schulz: the coefficients of step %d leave the range (singular values up to 5, the "
                     "polynomial of A up to 32)", k);
        top = std::max(1.0, next);
    }
    p.exact = steepest > kSteep;
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
    p.ldx = up64(n);
    p.lds = up64(p.s);
    p.parts = L.parts;
    p.ksplit = L.ksplit;
    p.eps = eps;
    p.steps = steps;
    p.status = status;
    char *ws = reinterpret_cast<char *>(workspace);
    Maps maps;
    for (int i = 0; i < 2; ++i) {
        for (int q = 0; q < 2; ++q) {
            p.x[i][q] = reinterpret_cast<__half *>(ws + (2 * i + q) * L.x);
            if (int st = matrix_map(&maps.x[i][q], p.x[i][q], batch, m, p.ldx, false)) return st;
            if (int st = matrix_map(&maps.xt[i][q], p.x[i][q], batch, m, p.ldx, true)) return st;
        }
        p.gram[i] = reinterpret_cast<__half *>(ws + 4 * L.x + i * L.square);
        p.poly[i] = reinterpret_cast<__half *>(ws + 4 * L.x + (2 + i) * L.square);
        if (int st = matrix_map(&maps.gram[i], p.gram[i], batch, p.s, p.lds, false)) return st;
        if (int st = matrix_map(&maps.poly[i], p.poly[i], batch, p.s, p.lds, false)) return st;
    }
    p.partial = reinterpret_cast<double *>(ws + 4 * L.x + 4 * L.square);
    p.pieces = reinterpret_cast<float *>(ws + 4 * L.x + 4 * L.square + L.partial);
    p.barrier = reinterpret_cast<unsigned *>(ws + 4 * L.x + 4 * L.square + L.partial + L.pieces);
    e = cudaMemsetAsync(p.barrier, 0, sizeof(unsigned), s);
    if (e != cudaSuccess) return cuda_failed(e);
    // a CTA per unit of the phase with the most of them, at most one per SM
    const int bn = L.wide ? 256 : 128;
    const int64_t apply = batch * tiles_of(p.l, bn) * tiles_of(p.s, bn), gram = batch * tiles_of(p.s, bn) * tiles_of(p.s, bn);
    const int grid = (int)std::min<int64_t>(sms, std::max<int64_t>({apply * (L.wide ? 2 : 1), gram * L.ksplit,
                                                                   (int64_t)batch * L.parts, L.ksplit > 1 ? sms : 1}));
    return L.wide ? launch<256>(maps, p, grid, s) : launch<128>(maps, p, grid, s);
}
