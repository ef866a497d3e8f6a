// Attention of a training step on tcgen05: the forward, which keeps one number per query (lse), and the backward, which
// recomputes the probabilities from it.
//
//   S_ij = scale · q_i·k_j over the allowed pairs (keys of the text's range; j <= i + Lk − Lq when causal),
//   lse_i = log Σ_j exp S_ij,  P_ij = exp(S_ij − lse_i),  O = P·V          (a row without a key: O = 0, lse = −inf)
//   D_i = Σ_d dO_id·O_id,  dV = Pᵀ·dO,  dS = P ∘ (dO·Vᵀ − D),  dQ = scale·dS·K,  dK = scale·dSᵀ·Q
//
// Nothing of size Lq x Lk is written. bf16 operands, fp32 accumulators in TMEM; the softmax's maximum, sum, lse, D and
// dS are fp32, and P and dS are rounded to bf16 once, as operands of the second product (the precision of the inputs).
//
// forward: a CTA takes two tiles of 128 queries over the keys in tiles of 128; each tile has a warpgroup (a thread per
// query row), so one tile's softmax runs while the tensor core works for the other. P goes back to TMEM as the A operand
// of P·V. O is rescaled only when a row's maximum grows by more than 2^8. The (key tile, query tile) steps take turns in
// the S buffers; with head_dim 64 there is a third one, and a warpgroup finds its next S ready when it has stored P.
// backward: two kernels, so that every sum has one writer and one order (no atomics; equal calls give equal bits):
//   dq: a CTA per 128 queries walks the keys and sums dS·K in TMEM;
//   dkv: a CTA per 128 keys walks the queries of every head of its group and sums Pᵀ·dO and dSᵀ·Q in TMEM, so a shared
//        K/V head's gradient needs no join. It computes Sᵀ and dPᵀ (keys as rows): Pᵀ and dSᵀ come out as A operands.
//   The recomputation of S and dP in both costs two of seven products, against a dQ of fp32 sums in memory.
// The dq kernel, which holds dO's rows, also computes D and keeps lse and D by padded rows for the dkv kernel.
//
// Rows of K, V, Q or dO that no allowed pair touches (outside a text's key range; queries before its first key) are
// zeroed in shared memory before a product would sum over them, so what they hold (NaN included) reaches nothing.
//
// Warp roles (320 threads): warp 0 issues TMA loads, warp 1 the MMAs, warps 2-9 the elementwise work. One thread issues
// all MMAs of a CTA and the tensor core runs them in issue order, so a product may overwrite TMEM that the product
// issued before it reads. That thread does nothing else and waits alone: it runs hardly ahead of the tensor core, and
// where its warp takes part (a vote after each wait, MMAs predicated by lane) a group of 24 MMAs takes 2475 cycles
// instead of 1847. Two issuing warps were slower still (their MMAs alternate between accumulators). A wait takes it 70
// cycles and a commit 85, in which little is queued; releases by the elementwise warps instead cost those more.
//
// Measured and what bounds it (causal, no padding):
//   2 x 4096, 32/8 heads of 128: forward 278 us (983 TFLOP/s; the softmax warps, one S buffer a tile), dq 355 us (1160
//   TFLOP/s executed) and dkv 418 us (1320 executed; shared-memory bandwidth of products that read both operands from it,
//   and the elementwise steps between them).
//   8 x 2048, 15/5 heads of 64: forward 131 us, dq 170, dkv 182: an MMA of 64 columns takes as long as one of 128, so half
//   the tensor rate is lost; exponentials run at half of their rate.
//   A CTA's start and end cost as much as 3 to 5 of its tiles. CTAs that took over further units (cluster launch control)
//   made short rows 5 to 8 % faster (dq of 5 x 1337, 32/8 heads of 128: 174 -> 161 us) and long ones 3 to 6 % slower (2 x
//   8192, 15/5 of 64: 501 -> 528 us), and were left out.
#include <algorithm>
#include <climits>
#include <mutex>

#include <cuda.h>
#include <cuda_bf16.h>

#include "../../include/lamq_b200_train.h"
#include "attention_steps.cuh"
#include "give_up.cuh"
#include "lamq_common.cuh"
#include "sm100.cuh"

namespace lamq {
namespace {

using namespace sm100;

constexpr int kTile = 128;
constexpr int kThreads = 320;
constexpr int kFill = 148;  // CTAs that fill the device
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Rows {  // where a thread writes: element (b, h, row, 0) of a (B, H, L, D) tensor
    __nv_bfloat16 *p;
    int64_t batch, head, row;
};

// Division of 0 <= n < 2^31 by a number of the launch: a CTA's place takes several, of 100 cycles or more each as such.
struct Div {
    uint32_t d, m, shift;
    Div() = default;
    explicit Div(uint32_t by) : d(by), shift(0) {
        while ((1ull << shift) < by) ++shift;
        m = (uint32_t)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
    }
    __device__ __forceinline__ int of(int n, int &rest) const {
        const uint32_t q = (__umulhi((uint32_t)n, m) + (uint32_t)n) >> shift;
        rest = n - (int)(q * d);
        return (int)q;
    }
};

struct Shape {
    int B, Hq, Hkv, group, D;
    int Lq, Lk, off;  // off = Lk − Lq
    int lq_pad;       // Lq rounded up to whole tiles
    int causal;
    Div by_heads, by_kv_heads, by_q, by_kv, by_group;  // B·Hq, B·Hkv, Hq, Hkv, group
    float scale, sl;  // sl = scale·log2 e
    const int32_t *ks, *ke;
    int *status;
};

template <int HD>
struct Sizes {
    static constexpr int NC = HD / 64;                  // 64-wide chunks of a row
    static constexpr int CHUNK = kTile * 128;           // bytes of a chunk of 128 rows
    static constexpr int TILE = NC * CHUNK;             // bytes of a 128 x HD tile
    static constexpr int FWD_STAGES = HD == 128 ? 4 : 6;  // half of them K's, half V's
    static constexpr int FWD_S = HD == 128 ? 2 : 3;     // buffers of S in the forward: what TMEM holds beside O
    // backward: stages of the operand that two products read (K for dQ, Q for dK and dV) and of the one that the first
    // product alone reads early (V, dO). The former is released a whole tile later: with two stages for both, its next
    // load came a TMA latency too late and S waited 1100 of 3300 cycles a tile.
    static constexpr int LATE_STAGES = HD == 128 ? 3 : 4, EARLY_STAGES = HD == 128 ? 2 : 4;
    static constexpr int ROW = kTile * 4;               // bytes of lse (or D) of a query tile
    static constexpr size_t FWD_SMEM = 2 * TILE + FWD_STAGES * TILE + 256 + 4 * ROW;
    static constexpr size_t DQ_SMEM = 2 * TILE + (LATE_STAGES + EARLY_STAGES) * TILE + 256 + ROW;
    static constexpr size_t DKV_SMEM = 2 * TILE + (LATE_STAGES + EARLY_STAGES) * (TILE + ROW) + 256;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Pairs of fp32 operations in one instruction (each rounded as alone), and the maximum of three: the elementwise warps are
// bound by what they issue.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 2^x of a pair with x <= 1 or so, in fp32 instructions alone: x = n + f with n the nearest integer (from the low bits of x
// + 1.5·2^23), 2^f by the polynomial that meets it in the six Chebyshev points of [-1/2, 1/2] (2e-7 off with its roundings),
// times 2^n. Below -126 it stays at 2^-126; NaN stays NaN.
__device__ __forceinline__ float2 ex2_pair(float2 x) {
    constexpr float kMagic = 12582912.f;
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.x));
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.y));
    const float2 t = add2(x, make_float2(kMagic, kMagic)), n = add2(t, make_float2(-kMagic, -kMagic));
    const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 y = make_float2(0.00133908633f, 0.00133908633f);
    y = fma2(y, f, make_float2(0.00967603177f, 0.00967603177f));
    y = fma2(y, f, make_float2(0.0555035695f, 0.0555035695f));
    y = fma2(y, f, make_float2(0.240221068f, 0.240221068f));
    y = fma2(y, f, make_float2(0.693147182f, 0.693147182f));
    y = fma2(y, f, make_float2(1.00000012f, 1.00000012f));
    return mul2(y, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                               __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ float2 pair_of(const uint32_t *r) {
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void key_range(const Shape &s, int b, int &lo, int &hi) {
    lo = s.ks ? max(0, s.ks[b]) : 0;
    hi = s.ke ? min(s.Lk, s.ke[b]) : s.Lk;
    if (lo >= hi) lo = hi = 0;
}

// A tile of 128 rows from row `row` of head (b, h): NC boxes of 64 x 128, zero past the tensor's end.
template <int HD>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap *map, int row, int h, int b, uint32_t bar) {
#pragma unroll
    for (int c = 0; c < Sizes<HD>::NC; ++c) tma_load_4d(dst + c * Sizes<HD>::CHUNK, map, 64 * c, row, h, b, bar);
}

// Descriptors of a tile's first K step: K-major (rows as M or N) and as 128 rows of K by HD columns of N. Later steps add
// constants to them (a shared-memory address below 256 KiB never carries out of the address field): the issuing thread
// has a few cycles per MMA, and computing whole descriptors there held the tensor core up.
__device__ __forceinline__ uint64_t rows_desc(uint32_t tile) { return smem_desc_sw128(tile, 16, 1024); }

template <int HD>
__device__ __forceinline__ uint64_t cols_desc(uint32_t tile) { return smem_desc_sw128(tile, Sizes<HD>::CHUNK, 1024); }

// D (+)= A·Bᵀ over HD, both tiles 128 x HD (K-major).
template <int HD>
__device__ __forceinline__ void mma_rows_rows(uint32_t d, uint64_t a, uint64_t b) {
    constexpr uint32_t idesc = idesc_bf16_f32(kTile, kTile, false, false);
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
        const uint32_t at = ((kk / 4) * Sizes<HD>::CHUNK + (kk % 4) * 32) >> 4;
        mma_f16_ss(d, a + at, b + at, idesc, kk > 0);
    }
}

// D = A·Bᵀ over HD, A 128 x HD bf16 in TMEM, B a tile (K-major).
template <int HD>
__device__ __forceinline__ void mma_tmem_rows_t(uint32_t d, uint32_t a, uint64_t b) {
    constexpr uint32_t idesc = idesc_bf16_f32(kTile, kTile, false, false);
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
        mma_f16_ts(d, a + kk * 8, b + (((kk / 4) * Sizes<HD>::CHUNK + (kk % 4) * 32) >> 4), idesc, kk > 0);
}

// A thread's row of a tile's 64-wide chunk (swizzled: 16-byte piece c of row r lies at c ^ (r mod 8)) into 32 TMEM columns
// of its lane, as an A operand.
__device__ __forceinline__ void chunk_to_tmem(uint32_t chunk, int row, uint32_t taddr) {
    uint32_t r[32];
#pragma unroll
    for (int c = 0; c < 8; ++c)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[4 * c]), "=r"(r[4 * c + 1]), "=r"(r[4 * c + 2]), "=r"(r[4 * c + 3])
                     : "r"(chunk + row * 128 + ((c ^ (row & 7)) << 4)));
    tmem_store32(taddr, r);
}

// D (+)= A·B, A 128 x 128 bf16 in TMEM (its columns 64.. from a + hi_cols), B a tile of 128 rows x HD.
template <int HD>
__device__ __forceinline__ void mma_tmem_rows(uint32_t d, uint32_t a, uint32_t hi_cols, uint64_t b, bool accumulate) {
    constexpr uint32_t idesc = idesc_bf16_f32(kTile, HD, false, true);
#pragma unroll
    for (int kk = 0; kk < kTile / 16; ++kk)
        mma_f16_ts(d, a + (kk < 4 ? kk * 8 : hi_cols + (kk - 4) * 8), b + ((kk * 2048) >> 4), idesc,
                   kk > 0 ? 1u : (uint32_t)accumulate);
}

// Threads `me` of `threads` zero the rows of a tile outside [lo, hi) (whole rows: the swizzle stays inside a row), for
// products issued after the barrier on which they arrive next.
template <int HD>
__device__ __forceinline__ void zero_rows(uint32_t tile, int lo, int hi, int me, int threads) {
    for (int i = me; i < Sizes<HD>::NC * kTile * 8; i += threads) {
        const int row = (i >> 3) & (kTile - 1);
        if (row < lo || row >= hi)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + i * 16), "r"(0) : "memory");
    }
    fence_async_smem();
}

__device__ __forceinline__ void wait_bounded(uint32_t bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < kWaitTimeoutNs) {
    }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8], float f) {
    return make_uint4(pack_bf16(x[0] * f, x[1] * f), pack_bf16(x[2] * f, x[3] * f), pack_bf16(x[4] * f, x[5] * f),
                      pack_bf16(x[6] * f, x[7] * f));
}

// One arrival for the warp, after its TMEM reads and writes.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// A warp's 32 rows of an accumulator, each thread's times its `f`, as bf16 to rows dst, dst + stride, ... (`live` of them;
// columns below D, a multiple of 8), through 4 KB of shared memory of the warp's: in whole lines. A thread that stored
// its own row, 16 bytes at a time, took 4000 cycles for 64 columns and 8000 to 9000 for 128, a third of the time of 8 key
// tiles.
template <int COLS>
__device__ __forceinline__ void store_rows(__nv_bfloat16 *dst, int64_t stride, uint32_t taddr, int col0, int D, float f,
                                           int live, uint32_t stage) {
    constexpr int W = COLS < 64 ? COLS : 64, PIECES = W / 8, ROWS = 32 / PIECES;  // columns, 16-byte pieces, rows at once
    const int lane = threadIdx.x & 31;
    const auto at = [&](int row, int piece) {
        return stage + row * (W * 2) + ((piece ^ (W == 64 ? row & 7 : (row >> 1) & 3)) << 4);
    };
#pragma unroll 1
    for (int c = 0; c < COLS; c += W) {
#pragma unroll
        for (int g = 0; g < W; g += 32) {
            uint32_t r[32];
            tmem_load32(taddr + c + g, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(r[e + k]);
                const uint4 v = pack8(x, f);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at(lane, (g + e) / 8)), "r"(v.x), "r"(v.y),
                             "r"(v.z), "r"(v.w)
                             : "memory");
            }
        }
        __syncwarp();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            const int row = r0 + lane / PIECES, piece = lane % PIECES, col = col0 + c + 8 * piece;
            uint4 v;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(at(row, piece))
                         : "memory");
            if (row < live && col < D) *reinterpret_cast<uint4 *>(dst + row * stride + col) = v;
        }
        __syncwarp();
    }
}

__device__ __forceinline__ void zero_row(__nv_bfloat16 *dst, int D) {
    for (int e = 0; e < D; e += 8) *reinterpret_cast<uint4 *>(dst + e) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------------------ forward

// A stage of a ring and the parity of its barrier: counted up, since a remainder costs the issuing thread time in which
// the tensor core idles.
struct Turn {
    int at = 0;
    uint32_t parity = 0;
    template <int N>
    __device__ __forceinline__ void next() {
        if (++at == N) at = 0, parity ^= 1;
    }
};

// A float of another CTA's shared memory.
__device__ __forceinline__ float load_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

// The key tiles [j0, j0 + n) that the queries row0 .. row0 + 127 meet.
__device__ __forceinline__ int key_tiles(const Shape &s, int row0, int lo, int hi) {
    if (row0 >= s.Lq) return 0;
    const int last = min(row0 + kTile, s.Lq) - 1;
    const int end = s.causal ? min(hi, last + s.off + 1) : hi;
    return end <= lo ? 0 : (end + kTile - 1) / kTile - lo / kTile;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    attention_forward_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                             const __grid_constant__ CUtensorMap mapV, Shape s, Rows out, float *__restrict__ lse, int split) {
    using Z = Sizes<HD>;
    constexpr int STAGES = Z::FWD_STAGES, RING = STAGES / 2, NB = Z::FWD_S;
    extern __shared__ __align__(1024) uint8_t smem[];  // swizzled tiles start at multiples of 1024 bytes
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (2 + STAGES) * Z::TILE);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 2 * NB + 3);
    float *const parts = reinterpret_cast<float *>(smem + 2 * Z::TILE);
    float *const row_max = reinterpret_cast<float *>(smem + Z::FWD_SMEM - 4 * Z::ROW), *const row_sum = row_max + 2 * kTile;
    static_assert(2 * HD * kTile * 4 <= STAGES * Z::TILE, "the parts of O fit into the stages");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t k_full0 = smem_u32(bars), v_full0 = k_full0 + 8 * RING, k_empty0 = v_full0 + 8 * RING,
                   v_empty0 = k_empty0 + 8 * RING, q_full = v_empty0 + 8 * RING;
    // s_full: the issuing thread's barriers of the buffers and, last, of the query tile that ends first (Steps)
    const uint32_t s_full0 = q_full + 8, p_ready0 = s_full0 + 8 * (NB + 1), drain = p_ready0 + 8 * NB;
    const uint32_t sq = smem_u32(smem), sk = sq + 2 * Z::TILE, sv = sk + RING * Z::TILE;

    const int pairs = s.lq_pad / kTile / 2 + (s.lq_pad / kTile & 1);
    // `split` CTAs (a cluster) share a pair of query tiles where there would be too few: each takes a part of the keys
    const int unit = split == 1 ? (int)blockIdx.x : (int)blockIdx.x / split, rank = split == 1 ? 0 : (int)blockIdx.x % split;
    int bh, h, in_group;
    const int qp = pairs - 1 - s.by_heads.of(unit, bh);  // the longest rows of a causal mask first
    const int b = s.by_q.of(bh, h), hk = s.by_group.of(h, in_group);
    int lo, hi;
    key_range(s, b, lo, hi);
    const int all0 = key_tiles(s, (2 * qp) * kTile, lo, hi), all1 = key_tiles(s, (2 * qp + 1) * kTile, lo, hi);
    const int n_all = max(all0, all1), first = split == 1 ? 0 : n_all * rank / split;
    const int n = split == 1 ? n_all : n_all * (rank + 1) / split - first;
    const int n0 = min(n, max(0, all0 - first)), n1 = min(n, max(0, all1 - first)), j0 = lo / kTile + first;
    const Steps<NB> steps{n0, n1};

    // The loads, by the first thread: Q, then K and V through the rings in the order K0 K1 V0 K2 V1 ..., as the products
    // want them. What finds free stages is issued before the other warps have met.
    int k_issued = 0, v_issued = 0;
    const auto load_next = [&](bool wait) {
        const bool is_k = k_issued < n && k_issued <= v_issued + 1;
        int &issued = is_k ? k_issued : v_issued;
        const int st = issued % RING;
        const uint32_t full = (is_k ? k_full0 : v_full0) + 8 * st;
        if (wait && !await((is_k ? k_empty0 : v_empty0) + 8 * st, ((issued / RING) & 1) ^ 1, s.status)) return false;
        mbar_expect_tx(full, Z::TILE);
        load_tile<HD>((is_k ? sk : sv) + st * Z::TILE, is_k ? &mapK : &mapV, (j0 + issued) * kTile, hk, b, full);
        ++issued;
        return true;
    };
    constexpr int EARLY = 2 * RING - 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * STAGES + 1; ++i) mbar_init(k_full0 + 8 * i, 1);
        for (int i = 0; i < NB + 1; ++i) mbar_init(s_full0 + 8 * i, 1);
        for (int i = 0; i < NB; ++i) mbar_init(p_ready0 + 8 * i, 4);
        mbar_init(drain, 1);
        fence_mbar_init();
        if (n > 0) {
            mbar_expect_tx(q_full, 2 * Z::TILE);
            load_tile<HD>(sq, &mapQ, 2 * qp * kTile, h, b, q_full);
            load_tile<HD>(sq + Z::TILE, &mapQ, (2 * qp + 1) * kTile, h, b, q_full);
            for (int i = 0; i < min(2 * n, EARLY); ++i) load_next(false);
        }
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_holder), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0 && n > 0) {  // ---- TMA producer
            bool ok = true;
            for (int i = EARLY; ok && i < 2 * n; ++i) ok = load_next(true);
            // the copies land before the CTA exits, also where another thread's error keeps anyone else from waiting for them
            wait_bounded(q_full, 0);
            for (int i = max(0, k_issued - RING); i < k_issued; ++i) wait_bounded(k_full0 + 8 * (i % RING), (i / RING) & 1);
            for (int i = max(0, v_issued - RING); i < v_issued; ++i) wait_bounded(v_full0 + 8 * (i % RING), (i / RING) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0 && n > 0) {  // ---- MMA issuer. P lies over S: P·V of a step goes before the buffer's next S
            const uint64_t q_desc = rows_desc(sq), k_desc = rows_desc(sk), v_desc = cols_desc<HD>(sv);
            const int count = steps.count(), ends_first = steps.ends_first();
            Turn k, v, buf;
            bool ok = await(q_full, 0, s.status);
            const auto issue_s = [&](int u, int to) {
                if (steps.begins(u)) ok = await(k_full0 + 8 * k.at, k.parity, s.status);
                if (!ok) return;
                mma_rows_rows<HD>(tmem + to * kTile, q_desc + steps.query_tile(u) * (Z::TILE >> 4),
                                  k_desc + k.at * (Z::TILE >> 4));
                if (steps.ends(u)) {
                    mma_commit(k_empty0 + 8 * k.at);
                    k.next<RING>();
                }
            };
            // few commits: one takes this thread 85 cycles
            for (int u = 0; ok && u < min(NB, count); ++u) {
                issue_s(u, u);
                if (ok) mma_commit(s_full0 + 8 * u);
            }
            uint32_t first_of = 3;  // the query tiles (bits) whose O holds nothing yet
            int u = 0;
            const auto run_to = [&](int end) {
                for (; ok && u < end; ++u, buf.next<NB>()) {
                    const int t = steps.query_tile(u);
                    ok = (!steps.begins(u) || await(v_full0 + 8 * v.at, v.parity, s.status)) &&
                         await(p_ready0 + 8 * buf.at, buf.parity, s.status);
                    if (!ok) break;
                    tc_fence_after();
                    mma_tmem_rows<HD>(tmem + NB * kTile + t * HD, tmem + buf.at * kTile, 32, v_desc + v.at * (Z::TILE >> 4),
                                      !(first_of >> t & 1));
                    first_of &= ~(1u << t);
                    if (steps.ends(u)) {
                        mma_commit(v_empty0 + 8 * v.at);
                        v.next<RING>();
                    }
                    if (u + NB < count) issue_s(u + NB, buf.at);
                    if (ok) mma_commit(s_full0 + 8 * buf.at);
                }
            };
            run_to(ends_first + 1);
            // (a test in each step for this one commit took 3 % more: 2 x 8192, 15/5 heads of 64: 386 us instead of 370)
            if (ok && ends_first >= 0) mma_commit(s_full0 + 8 * NB);
            run_to(count);
            mma_commit(drain);  // every MMA this thread issued completes before TMEM is released
            wait_bounded(drain, 0);
        }
        __syncwarp();
    } else {  // ---- softmax: warps 2-5 tile 0, warps 6-9 tile 1, a thread per query
        const int t = (warp - 2) >> 2, quad = warp & 3, nt = t ? n1 : n0;
        const int row0 = (2 * qp + t) * kTile, i = row0 + 32 * quad + lane;
        const bool live = i < s.Lq;
        // the keys of the text, of the thread's row and of the rows that see all, from the first key tile's first key on
        const int start = j0 * kTile, from = lo - start, to_all = hi - start;
        const int to_row = s.causal ? min(to_all, i + s.off + 1 - start) : to_all;
        const int whole = s.causal ? min(to_all, row0 + s.off + 1 - start) : to_all;  // key tiles between need no mask
        const uint32_t lanes = (uint32_t)(32 * quad) << 16;
        const uint32_t to = tmem + lanes + NB * kTile + t * HD;
        float m = -INFINITY, sum = 0.f;  // m: the maximum that the exponentials are taken against
        bool ok = true;
        const auto wait_for = [&](Wait w) {
            return __all_sync(0xffffffffu, await(s_full0 + 8 * w.bar, w.phase & 1, s.status)) != 0;
        };
        for (int j = 0; j < nt; ++j) {
            const int u = steps.index(j, t), buf = u % NB;
            const uint32_t ts = tmem + lanes + buf * kTile;
            ok = wait_for(steps.scores(u));
            if (!ok) break;
            tc_fence_after();
            uint32_t r[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_load32(ts + 32 * c, r[c]);
            tmem_ld_wait();
            if (from > j * kTile || whole < (j + 1) * kTile) {
                const int clo = from - j * kTile, chi = to_row - j * kTile;
#pragma unroll
                for (int c = 0; c < kTile; ++c)
                    if (c < clo || c >= chi) r[c >> 5][c & 31] = 0xff800000u;
                if (from > j * kTile || to_all < (j + 1) * kTile) {  // (both tiles' warps do: the same zeros)
                    ok = __all_sync(0xffffffffu, await(v_full0 + 8 * (j % RING), (j / RING) & 1, s.status));
                    if (!ok) break;
                    zero_rows<HD>(sv + (j % RING) * Z::TILE, from - j * kTile, to_all - j * kTile,
                                  threadIdx.x - 64 - 128 * t, 128);
                }
            }
            float top[8];  // eight chains: one of 128 comparisons would take 500 cycles of latency
#pragma unroll
            for (int c = 0; c < 8; ++c) top[c] = __uint_as_float(r[0][c]);
#pragma unroll
            for (int c = 8; c < kTile - 8; c += 16)
#pragma unroll
                for (int e = c; e < c + 8; ++e)
                    top[e & 7] = max3(top[e & 7], __uint_as_float(r[e >> 5][e & 31]),
                                      __uint_as_float(r[(e + 8) >> 5][(e + 8) & 31]));
#pragma unroll
            for (int c = 0; c < 8; c += 2)
                top[c / 2] = max3(fmaxf(top[c], top[c + 1]), __uint_as_float(r[3][24 + c]), __uint_as_float(r[3][25 + c]));
            const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]);
            // O and the sum are rescaled only when the maximum has grown by more than 8 binary orders: until then P
            // stays below 2^8, exact enough in fp32 and bf16 alike
            const bool grow = mx > m && (m == -INFINITY || (mx - m) * s.sl > 8.f);
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2((m - mx) * s.sl) : 1.f;
                if (grow) m = mx;
                sum *= f;
                if (j > 0) {
                    ok = wait_for(steps.read(steps.index(j - 1, t)));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_load32(to + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_store32(to + c, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m * s.sl;
            float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t pk[32];
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float2 x = fma2(pair_of(&r[2 * g + (c >> 5)][c & 31]), make_float2(s.sl, s.sl),
                                          make_float2(-base, -base));
                    const float2 e = make_float2(ex2(x.x), ex2(x.y));
                    part[(c >> 1) & 1] = add2(part[(c >> 1) & 1], e);
                    pk[c >> 1] = pack_bf16(e.x, e.y);
                }
                tmem_store32(ts + 32 * g, pk);
            }
            sum += (part[0].x + part[1].x) + (part[0].y + part[1].y);
            tmem_st_wait();
            warp_arrive(p_ready0 + 8 * buf);
        }
        if (ok && nt > 0) {
            ok = wait_for(steps.last_read(steps.index(nt - 1, t)));
            tc_fence_after();
        }
        if (split > 1 && n > 0) ok = ok && __all_sync(0xffffffffu, await(drain, 0, s.status));  // the other tile's too
        if (ok && split > 1 && n_all > 0) {  // to the cluster: columns of 128 rows over the stages, which are done with
            row_max[t * kTile + 32 * quad + lane] = m;
            row_sum[t * kTile + 32 * quad + lane] = sum;
            float *const mine = parts + t * HD * kTile + 32 * quad + lane;
#pragma unroll 1
            for (int c = 0; nt > 0 && c < HD; c += 32) {
                uint32_t r[32];
                tmem_load32(to + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 32; ++x) mine[(c + x) * kTile] = __uint_as_float(r[x]);
            }
        } else if (ok && rank == 0) {
            __nv_bfloat16 *const dst = out.p + b * out.batch + h * out.head + (int64_t)(i - lane) * out.row;
            if (nt > 0) {
                store_rows<HD>(dst, out.row, to, 0, s.D, sum > 0.f || sum != sum ? 1.f / sum : 0.f, s.Lq - (i - lane),
                               sq + t * Z::TILE + quad * 4096);  // staged over the tile's Q: its products are done
            } else if (live) zero_row(dst + lane * out.row, s.D);
            if (live)
                lse[((int64_t)b * s.Hq + h) * s.Lq + i] =
                    sum == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m * s.sl) + log2f(sum)) * kLn2;
        }
    }
    if (split > 1 && n_all > 0) {  // the parts joined by their maxima, in the order of the keys, a share of the columns each
        cluster_sync_all();
        if (warp >= 2) {
            const int pieces = 2 * HD / 8, p0 = pieces * rank / split, p1 = pieces * (rank + 1) / split;
            for (int e = p0 * kTile + (int)threadIdx.x - 64; e < p1 * kTile; e += 256) {
                const int row = e % kTile, col = e / kTile * 8 % HD, t = e / kTile * 8 / HD;
                const int i = (2 * qp + t) * kTile + row;
                if (i >= s.Lq || col >= s.D) continue;
                const uint32_t at_max = smem_u32(row_max + t * kTile + row), at_sum = smem_u32(row_sum + t * kTile + row);
                const uint32_t at = smem_u32(parts + (t * HD + col) * kTile + row);
                float m = -INFINITY, sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int q = 0; q < split; ++q) m = fmaxf(m, load_cluster(map_to_rank(at_max, q)));
                for (int q = 0; q < split; ++q) {
                    const float mq = load_cluster(map_to_rank(at_max, q)), sq = load_cluster(map_to_rank(at_sum, q));
                    if (sq == 0.f) continue;  // no key of this part (its columns may not even be written)
                    const float w = mq == m ? 1.f : ex2((mq - m) * s.sl);
                    sum = fmaf(w, sq, sum);
                    const uint32_t from = map_to_rank(at, q);
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[x] = fmaf(w, load_cluster(from + x * kTile * 4), acc[x]);
                }
                *reinterpret_cast<uint4 *>(out.p + b * out.batch + h * out.head + (int64_t)i * out.row + col) =
                    pack8(acc, sum == 0.f ? 0.f : 1.f / sum);
                if (col == 0)
                    lse[((int64_t)b * s.Hq + h) * s.Lq + i] =
                        sum == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m * s.sl) + log2f(sum)) * kLn2;
            }
        }
        cluster_sync_all();  // a CTA's shared memory stays until all have read it
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// ----------------------------------------------------------------------------------------------------------- backward

// Sum of the products of two 16-byte pieces of bf16.
__device__ __forceinline__ float dot8(uint4 x, uint4 y, float d) {
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        d = fmaf(__uint_as_float(xs[e] << 16), __uint_as_float(ys[e] << 16), d);
        d = fmaf(__uint_as_float(xs[e] & 0xffff0000u), __uint_as_float(ys[e] & 0xffff0000u), d);
    }
    return d;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dq_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                        const __grid_constant__ CUtensorMap mapV, const __grid_constant__ CUtensorMap mapG, Shape s,
                        const float *__restrict__ lse, float *__restrict__ lse2, float *__restrict__ Dr, Rows o, Rows dq, int split) {
    using Z = Sizes<HD>;
    constexpr int KS = Z::LATE_STAGES, VS = Z::EARLY_STAGES;
    // TMEM columns. Q and dO lie there as A operands: from shared memory they would take, with the key tile's rows, all
    // of its bandwidth. dS (bf16) lies over dP, as in the dkv kernel.
    constexpr uint32_t kDQ = 0, kS = 128, kP = 256, kQ = 384, kG = 448;
    extern __shared__ __align__(1024) uint8_t smem[];  // swizzled tiles start at multiples of 1024 bytes
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (2 + KS + VS) * Z::TILE);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 2 * (KS + VS) + 9);
    float *const parts = reinterpret_cast<float *>(smem + 2 * Z::TILE);
    static_assert(HD * kTile * 4 <= (KS + VS) * Z::TILE, "the part of dQ fits into the stages");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t k_full0 = smem_u32(bars), v_full0 = k_full0 + 8 * KS, k_empty0 = v_full0 + 8 * VS,
                   v_empty0 = k_empty0 + 8 * KS, q_full = v_empty0 + 8 * VS;
    const uint32_t q_ready = q_full + 8, s_full = q_full + 16, s_free = q_full + 24, p_full = q_full + 32;
    const uint32_t ds_ready = q_full + 40, done = q_full + 48;
    float *row_D = reinterpret_cast<float *>(smem + Z::DQ_SMEM - Z::ROW);
    const uint32_t sq = smem_u32(smem), sg = sq + Z::TILE, sk = sg + Z::TILE, sv = sk + KS * Z::TILE;

    // as in the forward
    const int unit = split == 1 ? (int)blockIdx.x : (int)blockIdx.x / split, rank = split == 1 ? 0 : (int)blockIdx.x % split;
    int bh, h, in_group;
    const int row0 = (s.lq_pad / kTile - 1 - s.by_heads.of(unit, bh)) * kTile;
    const int b = s.by_q.of(bh, h), hk = s.by_group.of(h, in_group);
    int lo, hi;
    key_range(s, b, lo, hi);
    const int n_all = key_tiles(s, row0, lo, hi), first = split == 1 ? 0 : n_all * rank / split;
    const int n = split == 1 ? n_all : n_all * (rank + 1) / split - first;
    const int j0 = lo / kTile + first;

    // Every elementwise thread's lse, and O for D = Σ dO·O: 16 rows a warp, a row's 16-byte pieces in neighbouring lanes (a
    // thread that read its own row took 4000 cycles). All at once and before anything waits; rows past the end are the last.
    constexpr int PIECES = HD / 8, ROWS = 32 / PIECES;
    const int d_row = 16 * (warp - 2) + lane / PIECES, piece = lane % PIECES;
    uint4 orow[16 / ROWS];
    float o_lse[16 / ROWS], own_lse = 0.f;
    if (warp >= 2) {
        own_lse = lse[(int64_t)bh * s.Lq + min(row0 + 32 * (warp & 3) + lane, s.Lq - 1)];
#pragma unroll
        for (int x = 0; x < 16 / ROWS; ++x) {
            const int at = min(row0 + d_row + ROWS * x, s.Lq - 1);
            o_lse[x] = lse[(int64_t)bh * s.Lq + at];
            orow[x] = *reinterpret_cast<const uint4 *>(o.p + b * o.batch + h * o.head + (int64_t)at * o.row +
                                                       (8 * piece < s.D ? 8 * piece : 0));
        }
    }
    // The loads, by the first thread: Q and dO, then K and V through the rings; V's stage is released by an earlier product
    // than K's of the same key tile. What finds free stages is issued before the other warps have met.
    int k_issued = 0, v_issued = 0;
    const auto load = [&](int j, bool wait) {
        const int ks = j % KS, vs = j % VS, row = (j0 + j) * kTile;
        if (wait && !await(k_empty0 + 8 * ks, ((j / KS) & 1) ^ 1, s.status)) return false;
        mbar_expect_tx(k_full0 + 8 * ks, Z::TILE);
        load_tile<HD>(sk + ks * Z::TILE, &mapK, row, hk, b, k_full0 + 8 * ks);
        ++k_issued;
        if (wait && !await(v_empty0 + 8 * vs, ((j / VS) & 1) ^ 1, s.status)) return false;
        mbar_expect_tx(v_full0 + 8 * vs, Z::TILE);
        load_tile<HD>(sv + vs * Z::TILE, &mapV, row, hk, b, v_full0 + 8 * vs);
        ++v_issued;
        return true;
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * (KS + VS) + 1; ++i) mbar_init(k_full0 + 8 * i, 1);
        mbar_init(q_ready, 8);
        mbar_init(s_full, 1);
        mbar_init(s_free, 8);
        mbar_init(p_full, 1);
        mbar_init(ds_ready, 8);
        mbar_init(done, 1);
        fence_mbar_init();
        if (n > 0) {
            mbar_expect_tx(q_full, 2 * Z::TILE);
            load_tile<HD>(sq, &mapQ, row0, h, b, q_full);
            load_tile<HD>(sg, &mapG, row0, h, b, q_full);
            for (int j = 0; j < min(n, VS); ++j) load(j, false);
        }
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_holder), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0 && n > 0) {
            bool ok = true;
            for (int j = VS; ok && j < n; ++j) ok = load(j, true);
            wait_bounded(q_full, 0);  // the copies land before the CTA exits
            for (int i = max(0, k_issued - KS); i < k_issued; ++i) wait_bounded(k_full0 + 8 * (i % KS), (i / KS) & 1);
            for (int i = max(0, v_issued - VS); i < v_issued; ++i) wait_bounded(v_full0 + 8 * (i % VS), (i / VS) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0 && n > 0) {
            const uint64_t k_desc = rows_desc(sk), v_desc = rows_desc(sv), kc_desc = cols_desc<HD>(sk);
            bool ok = await(q_ready, 0, s.status);
            // in issue order: S(0) dP(0) | S(j + 1) | dQ(j) dP(j + 1) | ...: while the warps form P(j), S(j + 1) runs; while
            // they go on to P(j + 1), dQ(j) and, over the dS(j) that it read, dP(j + 1) run
            for (int j = -1; ok && j < n; ++j) {
                const int kn = (j + 1) % KS, vn = (j + 1) % VS;
                if (j + 1 < n) {
                    ok = await(k_full0 + 8 * kn, ((j + 1) / KS) & 1, s.status) &&
                         (j < 0 || await(s_free, j & 1, s.status));
                    if (!ok) break;
                    tc_fence_after();
                    mma_tmem_rows_t<HD>(tmem + kS, tmem + kQ, k_desc + kn * (Z::TILE >> 4));
                    mma_commit(s_full);
                    ok = await(v_full0 + 8 * vn, ((j + 1) / VS) & 1, s.status);
                    if (!ok) break;
                }
                if (j >= 0) {
                    ok = await(ds_ready, j & 1, s.status);
                    if (!ok) break;
                    tc_fence_after();
                    mma_tmem_rows<HD>(tmem + kDQ, tmem + kP, 64, kc_desc + (j % KS) * (Z::TILE >> 4), j > 0);
                    mma_commit(k_empty0 + 8 * (j % KS));
                }
                if (j + 1 < n) {
                    mma_tmem_rows_t<HD>(tmem + kP, tmem + kG, v_desc + vn * (Z::TILE >> 4));
                    mma_commit(p_full);
                    mma_commit(v_empty0 + 8 * vn);
                }
            }
            mma_commit(done);
            wait_bounded(done, 0);
        }
        __syncwarp();
    } else {  // two threads per query: columns 64·half ..
        const int half = (warp - 2) >> 2, quad = warp & 3;
        const int i = row0 + 32 * quad + lane;
        const bool live = i < s.Lq;
        const int row_hi = s.causal ? min(hi, i + s.off + 1) : hi;
        const uint32_t lanes = (uint32_t)(32 * quad) << 16;
        bool ok = n > 0 && __all_sync(0xffffffffu, await(q_full, 0, s.status));
        if (ok) {
            if (HD == 64) {
                chunk_to_tmem(half ? sg : sq, 32 * quad + lane, tmem + lanes + (half ? kG : kQ));
            } else {
                chunk_to_tmem(sq + half * Z::CHUNK, 32 * quad + lane, tmem + lanes + kQ + 32 * half);
                chunk_to_tmem(sg + half * Z::CHUNK, 32 * quad + lane, tmem + lanes + kG + 32 * half);
            }
            tmem_st_wait();
            warp_arrive(q_ready);
        }
        float d[16 / ROWS];
#pragma unroll
        for (int x = 0; x < 16 / ROWS; ++x) {
            const int row = d_row + ROWS * x;
            uint4 g = make_uint4(0, 0, 0, 0);
            if (ok)
                g = *reinterpret_cast<const uint4 *>(smem + Z::TILE + (piece >> 3) * Z::CHUNK + row * 128 +
                                                     (((piece & 7) ^ (row & 7)) << 4));
            // dO is zero beyond its columns and rows; O and dO of a row without a key may hold anything
            d[x] = o_lse[x] != -INFINITY && 8 * piece < s.D ? dot8(orow[x], g, 0.f) : 0.f;
        }
#pragma unroll
        for (int m = 1; m < PIECES; m *= 2)
#pragma unroll
            for (int x = 0; x < 16 / ROWS; ++x) d[x] += __shfl_xor_sync(0xffffffffu, d[x], m);
#pragma unroll
        for (int x = 0; x < 16 / ROWS; ++x)
            if (piece == 0) row_D[d_row + ROWS * x] = d[x];
        asm volatile("bar.sync 1, 256;" ::: "memory");
        // D, and lse in units of log 2 (+inf where there is no row or it is empty: P = 0); kept by padded rows for dkv
        const float Di = row_D[32 * quad + lane], l2 = live && own_lse != -INFINITY ? own_lse * kLog2e : INFINITY;
        if (half == 0 && rank == split - 1) {  // (the last part is never without keys where there are any)
            lse2[(int64_t)bh * s.lq_pad + i] = -l2;  // negated, as the dkv kernel adds them
            Dr[(int64_t)bh * s.lq_pad + i] = -Di;
        }
        for (int j = 0; ok && j < n; ++j) {
            ok = __all_sync(0xffffffffu, await(s_full, j & 1, s.status));
            if (!ok) break;
            tc_fence_after();
            uint32_t r[2][32], d[2][32];
            tmem_load32(tmem + lanes + kS + 64 * half, r[0]);
            tmem_load32(tmem + lanes + kS + 64 * half + 32, r[1]);
            tmem_ld_wait();
            warp_arrive(s_free);
            const int key0 = (j0 + j) * kTile;
            const bool edge = key0 < lo || key0 + kTile > hi || (s.causal && key0 + kTile - 1 > row0 + s.off);
            const int clo = lo - key0 - 64 * half, chi = row_hi - key0 - 64 * half;
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
                uint32_t *const at = &r[c >> 5][c & 31];
                const float2 x = fma2(pair_of(at), make_float2(s.sl, s.sl), make_float2(-l2, -l2));
                at[0] = __float_as_uint(ex2(x.x)), at[1] = __float_as_uint(ex2(x.y));
            }
            ok = __all_sync(0xffffffffu, await(p_full, j & 1, s.status));
            if (!ok) break;
            tc_fence_after();
            tmem_load32(tmem + lanes + kP + 64 * half, d[0]);
            tmem_load32(tmem + lanes + kP + 64 * half + 32, d[1]);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
                uint32_t *const at = &r[c >> 5][c & 31];
                const float2 x = mul2(pair_of(at), add2(pair_of(&d[c >> 5][c & 31]), make_float2(-Di, -Di)));
                at[0] = __float_as_uint(x.x), at[1] = __float_as_uint(x.y);
            }
            if (edge) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (c < clo || c >= chi) r[c >> 5][c & 31] = 0u;
            }
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 64; c += 2)
                pk[c >> 1] = pack_bf16(__uint_as_float(r[c >> 5][c & 31]), __uint_as_float(r[c >> 5][(c & 31) + 1]));
            if (key0 < lo || key0 + kTile > hi)  // S(j), the other reader of K(j), is done
                zero_rows<HD>(sk + (j % KS) * Z::TILE, lo - key0, hi - key0, threadIdx.x - 64, 256);
            tmem_store32(tmem + lanes + kP + 64 * half, pk);
            tmem_st_wait();
            warp_arrive(ds_ready);
        }
        if (ok) {
            ok = __all_sync(0xffffffffu, await(done, 0, s.status));
            tc_fence_after();
        }
        if (split > 1 && n_all > 0) {  // to the cluster: columns of 128 rows over the stages, which are done with
            float *const mine = parts + half * (HD / 2) * kTile + 32 * quad + lane;
#pragma unroll 1
            for (int c = 0; c < HD / 2; c += 32) {
                uint32_t r[32];
                tmem_load32(tmem + lanes + kDQ + half * (HD / 2) + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 32; ++x) mine[(c + x) * kTile] = n > 0 ? __uint_as_float(r[x]) : 0.f;
            }
        } else if ((ok || n == 0) && rank == 0) {
            __nv_bfloat16 *const dst = dq.p + b * dq.batch + h * dq.head + (int64_t)(i - lane) * dq.row;
            if (n > 0)  // (staged over Q and dO, which every warp has read)
                store_rows<HD / 2>(dst, dq.row, tmem + lanes + kDQ + half * (HD / 2), half * (HD / 2), s.D, s.scale,
                                   s.Lq - (i - lane), sq + (warp - 2) * 4096);
            else if (live && half == 0) zero_row(dst + lane * dq.row, s.D);
        }
    }
    if (split > 1 && n_all > 0) {  // the parts added in the order of the keys, a share of the columns each
        cluster_sync_all();
        if (warp >= 2) {
            const int pieces = HD / 8, p0 = pieces * rank / split, p1 = pieces * (rank + 1) / split;
            for (int e = p0 * kTile + (int)threadIdx.x - 64; e < p1 * kTile; e += 256) {
                const int row = e % kTile, col = e / kTile * 8;
                if (row0 + row >= s.Lq || col >= s.D) continue;
                float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int q = 0; q < split; ++q) {
                    const uint32_t from = map_to_rank(smem_u32(parts + col * kTile + row), q);
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[x] += load_cluster(from + x * kTile * 4);
                }
                *reinterpret_cast<uint4 *>(dq.p + b * dq.batch + h * dq.head + (int64_t)(row0 + row) * dq.row + col) =
                    pack8(acc, s.scale);
            }
        }
        cluster_sync_all();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dkv_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                         const __grid_constant__ CUtensorMap mapV, const __grid_constant__ CUtensorMap mapG, Shape s,
                         const float *__restrict__ lse2, const float *__restrict__ Dr, Rows dk, Rows dv, int split) {
    using Z = Sizes<HD>;
    constexpr int QS = Z::LATE_STAGES, GS = Z::EARLY_STAGES;  // Q (with lse), dO (with D)
    // TMEM columns. Pᵀ and dSᵀ (bf16) lie over Sᵀ and dPᵀ: the threads of columns 0..63 write columns 0..31 of them,
    // those of columns 64..127 write 64..95, so that no thread overwrites what another has yet to read
    constexpr uint32_t kS = 0, kP = 128, kDV = 256, kDK = 384;
    extern __shared__ __align__(1024) uint8_t smem[];  // swizzled tiles start at multiples of 1024 bytes
    float *row_lse = reinterpret_cast<float *>(smem + (2 + QS + GS) * Z::TILE), *row_d = row_lse + QS * kTile;
    uint64_t *bars = reinterpret_cast<uint64_t *>(row_d + GS * kTile);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 2 * (QS + GS) + 7);
    float *const parts = reinterpret_cast<float *>(smem + 2 * Z::TILE);
    static_assert(2 * HD * kTile * 4 <= (QS + GS) * Z::TILE, "the parts of dK and dV fit into the stages");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t q_full0 = smem_u32(bars), g_full0 = q_full0 + 8 * QS, q_empty0 = g_full0 + 8 * GS,
                   g_empty0 = q_empty0 + 8 * QS, kv_full = g_empty0 + 8 * GS;
    const uint32_t s_full = kv_full + 8, p_full = kv_full + 16, p_ready = kv_full + 24, ds_ready = kv_full + 32;
    const uint32_t done = kv_full + 40;
    const uint32_t sk = smem_u32(smem), sv = sk + Z::TILE, sq = sv + Z::TILE, sg = sq + QS * Z::TILE;

    // `split` CTAs (a cluster) share a key tile where there would be too few: each takes a part of the group's query heads
    const int unit = split == 1 ? (int)blockIdx.x : (int)blockIdx.x / split, rank = split == 1 ? 0 : (int)blockIdx.x % split;
    int bh, hk;
    const int key0 = s.by_kv_heads.of(unit, bh) * kTile;  // the first keys are seen by the most queries: they come first
    const int b = s.by_kv.of(bh, hk), share = split == 1 ? s.group : s.group / split, h0 = hk * s.group + rank * share;
    int lo, hi;
    key_range(s, b, lo, hi);
    const int q_lo = s.causal ? max(0, lo - s.off) : 0;  // the queries before see no key
    const int first = s.causal ? max(q_lo, key0 - s.off) : 0;
    const int t0 = first / kTile, tiles = s.lq_pad / kTile;
    const int nq = key0 >= hi || key0 + kTile <= lo || first >= s.Lq ? 0 : tiles - t0;
    const int n = nq * share;

    // The loads, by the first thread: K and V, then Q and dO (with the rows' lse and D) through the rings; dO's stage is
    // released by an earlier product than Q's of the same query tile. What finds free stages is issued before the other
    // warps have met.
    int q_issued = 0, g_issued = 0, h = h0, row = t0 * kTile;  // (a division by nq for each tile would take longer)
    const auto load = [&](int j, bool wait) {
        const int qs = j % QS, gs = j % GS;
        const int64_t at = ((int64_t)b * s.Hq + h) * s.lq_pad + row;
        if (wait && !await(q_empty0 + 8 * qs, ((j / QS) & 1) ^ 1, s.status)) return false;
        mbar_expect_tx(q_full0 + 8 * qs, Z::TILE + Z::ROW);
        load_tile<HD>(sq + qs * Z::TILE, &mapQ, row, h, b, q_full0 + 8 * qs);
        bulk_load(smem_u32(row_lse + qs * kTile), lse2 + at, Z::ROW, q_full0 + 8 * qs);
        ++q_issued;
        if (wait && !await(g_empty0 + 8 * gs, ((j / GS) & 1) ^ 1, s.status)) return false;
        mbar_expect_tx(g_full0 + 8 * gs, Z::TILE + Z::ROW);
        load_tile<HD>(sg + gs * Z::TILE, &mapG, row, h, b, g_full0 + 8 * gs);
        bulk_load(smem_u32(row_d + gs * kTile), Dr + at, Z::ROW, g_full0 + 8 * gs);
        ++g_issued;
        row += kTile;
        if (row == s.lq_pad) row = t0 * kTile, ++h;
        return true;
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * (QS + GS) + 1; ++i) mbar_init(q_full0 + 8 * i, 1);
        mbar_init(s_full, 1);
        mbar_init(p_full, 1);
        mbar_init(p_ready, 8);
        mbar_init(ds_ready, 8);
        mbar_init(done, 1);
        fence_mbar_init();
        if (n > 0) {
            mbar_expect_tx(kv_full, 2 * Z::TILE);
            load_tile<HD>(sk, &mapK, key0, hk, b, kv_full);
            load_tile<HD>(sv, &mapV, key0, hk, b, kv_full);
            for (int j = 0; j < min(n, GS); ++j) load(j, false);
        }
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_holder), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0 && n > 0) {
            bool ok = true;
            for (int j = GS; ok && j < n; ++j) ok = load(j, true);
            wait_bounded(kv_full, 0);  // the copies land before the CTA exits
            for (int i = max(0, q_issued - QS); i < q_issued; ++i) wait_bounded(q_full0 + 8 * (i % QS), (i / QS) & 1);
            for (int i = max(0, g_issued - GS); i < g_issued; ++i) wait_bounded(g_full0 + 8 * (i % GS), (i / GS) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0 && n > 0) {
            const uint64_t k_desc = rows_desc(sk), v_desc = rows_desc(sv), q_desc = rows_desc(sq), g_desc = rows_desc(sg),
                           qc_desc = cols_desc<HD>(sq), gc_desc = cols_desc<HD>(sg);
            bool ok = await(kv_full, 0, s.status);
            // in issue order: S(0) dP(0) | dV(j) S(j + 1) | dK(j) dP(j + 1) | ...: the warps form P(j) while dK(j − 1)
            // and dP(j) run, and dS(j) while dV(j) and S(j + 1) run
            for (int j = -1; ok && j < n; ++j) {
                const int qs = j % QS, gs = j % GS, qn = (j + 1) % QS, gn = (j + 1) % GS;
                if (j + 1 < n) ok = await(q_full0 + 8 * qn, ((j + 1) / QS) & 1, s.status);
                if (j >= 0) {
                    ok = ok && await(p_ready, j & 1, s.status);
                    if (!ok) break;
                    tc_fence_after();
                    mma_tmem_rows<HD>(tmem + kDV, tmem + kS, 64, gc_desc + gs * (Z::TILE >> 4), j > 0);
                }
                if (j + 1 < n) {
                    if (!ok) break;
                    mma_rows_rows<HD>(tmem + kS, k_desc, q_desc + qn * (Z::TILE >> 4));
                    mma_commit(s_full);
                    ok = await(g_full0 + 8 * gn, ((j + 1) / GS) & 1, s.status);
                }
                if (j >= 0) {
                    ok = ok && await(ds_ready, j & 1, s.status);
                    if (!ok) break;
                    tc_fence_after();
                    mma_commit(g_empty0 + 8 * gs);  // D(j) was read before ds_ready, dO(j) by dV(j)
                    mma_tmem_rows<HD>(tmem + kDK, tmem + kP, 64, qc_desc + qs * (Z::TILE >> 4), j > 0);
                    mma_commit(q_empty0 + 8 * qs);
                }
                if (j + 1 < n) {
                    if (!ok) break;
                    mma_rows_rows<HD>(tmem + kP, v_desc, g_desc + gn * (Z::TILE >> 4));
                    mma_commit(p_full);
                }
            }
            mma_commit(done);
            wait_bounded(done, 0);
        }
        __syncwarp();
    } else {  // two threads per key: queries 64·half .. of each tile
        const int half = (warp - 2) >> 2, quad = warp & 3;
        const int key = key0 + 32 * quad + lane;
        const bool in = key >= lo && key < hi;
        const uint32_t lanes = (uint32_t)(32 * quad) << 16;
        const bool edge_keys = key0 < lo || key0 + kTile > hi;
        bool ok = true;
        for (int j = 0, row0 = t0 * kTile; j < n; ++j, row0 = row0 + kTile == s.lq_pad ? t0 * kTile : row0 + kTile) {
            const int qs = j % QS, gs = j % GS;
            const float4 *l4 = reinterpret_cast<const float4 *>(row_lse + qs * kTile + 64 * half);
            const float4 *d4 = reinterpret_cast<const float4 *>(row_d + gs * kTile + 64 * half);
            const bool edge = edge_keys || (s.causal && key0 + kTile - 1 > row0 + s.off);
            const int clo = !in ? 64 : s.causal ? key - s.off - row0 - 64 * half : 0;  // columns before are masked
            // the tile's statistics came with Q and dO: their barriers make them visible to this thread
            ok = __all_sync(0xffffffffu, await(s_full, j & 1, s.status) &&
                                             await(q_full0 + 8 * qs, (j / QS) & 1, s.status));
            if (!ok) break;
            tc_fence_after();
            uint32_t r[2][32], pk[32];
            tmem_load32(tmem + lanes + kS + 64 * half, r[0]);
            tmem_load32(tmem + lanes + kS + 64 * half + 32, r[1]);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 64; c += 4) {
                const float4 l = l4[c >> 2];  // negated
                const float2 ls[2] = {make_float2(l.x, l.y), make_float2(l.z, l.w)};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t *const at = &r[c >> 5][(c & 31) + 2 * e];
                    const float2 x = fma2(pair_of(at), make_float2(s.sl, s.sl), ls[e]);
                    // a quarter of the exponentials in fp32 instructions: the 16 a cycle of the special-function unit hold the
                    // step up (dkv of 2 x 4096, 32/8 heads of 128: 432 -> 418 us; of 2 x 8192, 15/5 of 64: 650 -> 614; a
                    // third: 424 and 607; the dq kernel, with more to do beside, became 4 to 14 % slower)
                    const float2 y = (c / 2 + e) % 4 == 3 ? ex2_pair(x) : make_float2(ex2(x.x), ex2(x.y));
                    at[0] = __float_as_uint(y.x), at[1] = __float_as_uint(y.y);
                }
            }
            if (edge) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (c < clo) r[c >> 5][c & 31] = 0u;
            }
#pragma unroll
            for (int c = 0; c < 64; c += 2)
                pk[c >> 1] = pack_bf16(__uint_as_float(r[c >> 5][c & 31]), __uint_as_float(r[c >> 5][(c & 31) + 1]));
            if (row0 < q_lo) {  // dV sums over dO's rows, dK over Q's: those of queries without a key
                ok = __all_sync(0xffffffffu, await(g_full0 + 8 * gs, (j / GS) & 1, s.status));
                if (!ok) break;
                zero_rows<HD>(sg + gs * Z::TILE, q_lo - row0, kTile, threadIdx.x - 64, 256);
                zero_rows<HD>(sq + qs * Z::TILE, q_lo - row0, kTile, threadIdx.x - 64, 256);
            }
            tmem_store32(tmem + lanes + kS + 64 * half, pk);
            tmem_st_wait();
            warp_arrive(p_ready);

            ok = __all_sync(0xffffffffu, await(p_full, j & 1, s.status) &&
                                             await(g_full0 + 8 * gs, (j / GS) & 1, s.status));
            if (!ok) break;
            tc_fence_after();
            uint32_t d[2][32];
            tmem_load32(tmem + lanes + kP + 64 * half, d[0]);
            tmem_load32(tmem + lanes + kP + 64 * half + 32, d[1]);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 64; c += 4) {
                const float4 l = d4[c >> 2];  // negated
                const float2 ds[2] = {make_float2(l.x, l.y), make_float2(l.z, l.w)};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t *const at = &d[c >> 5][(c & 31) + 2 * e];
                    const float2 x = mul2(pair_of(&r[c >> 5][(c & 31) + 2 * e]), add2(pair_of(at), ds[e]));
                    at[0] = __float_as_uint(x.x), at[1] = __float_as_uint(x.y);
                }
            }
            if (edge) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (c < clo) d[c >> 5][c & 31] = 0u;
            }
#pragma unroll
            for (int c = 0; c < 64; c += 2)
                pk[c >> 1] = pack_bf16(__uint_as_float(d[c >> 5][c & 31]), __uint_as_float(d[c >> 5][(c & 31) + 1]));
            tmem_store32(tmem + lanes + kP + 64 * half, pk);
            tmem_st_wait();
            warp_arrive(ds_ready);
        }
        const bool live = key < s.Lk;
        if (ok && n > 0) {
            ok = __all_sync(0xffffffffu, await(done, 0, s.status));
            tc_fence_after();
        }
        if (ok) {  // columns half·HD/2 .. of the thread's key
            const int c0 = half * (HD / 2);
            __nv_bfloat16 *const pk_ = dk.p + b * dk.batch + hk * dk.head + (int64_t)(key - lane) * dk.row;
            __nv_bfloat16 *const pv_ = dv.p + b * dv.batch + hk * dv.head + (int64_t)(key - lane) * dv.row;
            if (split > 1 && n > 0) {  // to the cluster: columns of 128 rows over the stages, which are done with
                float *const mine = parts + c0 * kTile + 32 * quad + lane;
#pragma unroll 1
                for (int m = 0; m < 2; ++m)
#pragma unroll 1
                    for (int c = 0; c < HD / 2; c += 32) {
                        uint32_t r[32];
                        tmem_load32(tmem + lanes + (m ? kDV : kDK) + c0 + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 32; ++x) mine[(m * HD + c + x) * kTile] = __uint_as_float(r[x]);
                    }
            } else if (n > 0) {
                const int rows = s.Lk - (key - lane);
                const uint32_t stage = sk + (warp - 2) * 4096;  // over K and V, which the products are done with
                store_rows<HD / 2>(pk_, dk.row, tmem + lanes + kDK + c0, c0, s.D, s.scale, rows, stage);
                store_rows<HD / 2>(pv_, dv.row, tmem + lanes + kDV + c0, c0, s.D, 1.f, rows, stage);
            } else if (live && rank == 0) {
                zero_row(half ? pv_ + lane * dv.row : pk_ + lane * dk.row, s.D);
            }
        }
    }
    if (split > 1 && n > 0) {  // each CTA adds its share of the columns over the cluster, in the order of the heads
        cluster_sync_all();
        if (warp >= 2) {
            const int pieces = 2 * HD / 8, p0 = pieces * rank / split, p1 = pieces * (rank + 1) / split;
            for (int i = p0 * kTile + (int)threadIdx.x - 64; i < p1 * kTile; i += 256) {
                const int row = i % kTile, col = i / kTile * 8 % HD, m = i / kTile * 8 / HD;
                if (key0 + row >= s.Lk || col >= s.D) continue;
                float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int q = 0; q < split; ++q) {
                    const uint32_t from = map_to_rank(smem_u32(parts + (m * HD + col) * kTile + row), q);
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[x] += load_cluster(from + x * kTile * 4);
                }
                const Rows &to = m ? dv : dk;
                *reinterpret_cast<uint4 *>(to.p + b * to.batch + hk * to.head + (int64_t)(key0 + row) * to.row + col) =
                    pack8(acc, m ? 1.f : s.scale);
            }
        }
        cluster_sync_all();  // a CTA's shared memory stays until all have read it
    }
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

// A (B, H, L, D) bf16 tensor in boxes of 64 x 128 rows, 128-byte swizzle, zero outside.
int tile_map(CUtensorMap *m, const lamq_heads &t, int B, int H, int64_t L, int D) {
    EncodeTiled enc = encode_fn();
    if (enc == nullptr) {
        set_error("lamq_attention: cuTensorMapEncodeTiled is unavailable");
        return LAMQ_ERR_CUDA;
    }
    const auto stride = [](int64_t n, int64_t s, int64_t other) { return (cuuint64_t)(n > 1 ? s : other) * 2; };
    const int64_t dense = (D + 7) / 8 * 8;  // the stride of an axis of one entry is not used: any valid value
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B};
    const cuuint64_t strides[3] = {stride(L, t.row, dense), stride(H, t.head, dense), stride(B, t.batch, dense)};
    const cuuint32_t box[4] = {64, kTile, 1, 1}, step[4] = {1, 1, 1, 1};
    const auto make = [&] {
        return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t.data, dims, strides, box, step,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = make();
    if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
        // a driver call needs the device's context bound to the thread, and one that has made no runtime call yet
        // (autograd's) has none: bind it
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = make();
    }
    if (r != CUDA_SUCCESS) {
        set_error("lamq_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
        return LAMQ_ERR_CUDA;
    }
    return LAMQ_OK;
}

int check_heads(const char *fn, const char *name, const lamq_heads &t, int64_t B, int64_t H, int64_t L) {
    LAMQ_REQUIRE(t.data != nullptr, "%s: null pointer (%s)", fn, name);
    const auto fits = [](int64_t n, int64_t s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
    LAMQ_REQUIRE(reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && fits(B, t.batch) && fits(H, t.head) && fits(L, t.row),
                 "%s: %s must be 16-byte aligned with positive strides that are multiples of 8", fn, name);
    return LAMQ_OK;
}

int shape_of(const char *fn, const lamq_attention_args &a, int *status, Shape &s, bool &empty) {
    LAMQ_REQUIRE(a.batch >= 0 && a.heads >= 0 && a.kv_heads >= 0 && a.q_len >= 0 && a.kv_len >= 0, "%s: bad shape", fn);
    LAMQ_REQUIRE(a.head_dim >= 8 && a.head_dim <= 128 && a.head_dim % 8 == 0,
                 "%s: head_dim must be a multiple of 8 in 8..128 (got %d)", fn, a.head_dim);
    LAMQ_REQUIRE(a.heads == 0 || (a.kv_heads > 0 && a.heads % a.kv_heads == 0),
                 "%s: %d query heads are not a multiple of %d key heads", fn, a.heads, a.kv_heads);
    LAMQ_REQUIRE(a.scale > 0.f && a.scale < INFINITY, "%s: the scale must be positive and finite", fn);
    LAMQ_REQUIRE(a.q_len <= (1 << 30) && a.kv_len <= (1 << 30) && a.batch * (int64_t)a.heads <= (1 << 20),
                 "%s: lengths up to 2^30 and up to 2^20 heads in all", fn);
    empty = a.batch == 0 || a.heads == 0;
    if (empty) return LAMQ_OK;
    LAMQ_REQUIRE(status != nullptr, "%s: null pointer (status)", fn);
    s.B = (int)a.batch;
    s.Hq = a.heads;
    s.Hkv = a.kv_heads;
    s.group = a.heads / a.kv_heads;
    s.D = a.head_dim;
    s.Lq = (int)a.q_len;
    s.Lk = (int)a.kv_len;
    s.off = s.Lk - s.Lq;
    s.lq_pad = (s.Lq + kTile - 1) / kTile * kTile;
    s.causal = a.causal;
    s.by_heads = Div((uint32_t)(s.B * s.Hq));
    s.by_kv_heads = Div((uint32_t)(s.B * s.Hkv));
    s.by_q = Div((uint32_t)s.Hq);
    s.by_kv = Div((uint32_t)s.Hkv);
    s.by_group = Div((uint32_t)s.group);
    s.scale = a.scale;
    s.sl = a.scale * kLog2e;
    s.ks = a.key_start;
    s.ke = a.key_end;
    s.status = status;
    return LAMQ_OK;
}

Rows rows_of(const lamq_heads &t) { return {reinterpret_cast<__nv_bfloat16 *>(t.data), t.batch, t.head, t.row}; }

int launch_failed(const char *what, cudaError_t e) {
    set_error("%s: %s", what, cudaGetErrorString(e));
    return LAMQ_ERR_CUDA;
}

// A launch of `units` clusters of `split` CTAs.
template <typename K, typename... A>
cudaError_t launch_split(K *kernel, int64_t units, int split, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(units * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// CTAs per pair of query tiles (forward) or query tile (dq): 1, or where the device would hold more the largest power of
// two up to 8 that it holds at once, in parts of four key tiles or more. 32/8 heads of 128, one query over 4096 keys:
// forward 57 us whole, 26 in parts; dq 44 and 18. (A second wave of parts costs more than it gains: 32/8 heads, 512
// queries and keys, dq 13 us whole, 23 in 256 CTAs.)
int split_keys(int64_t units, int Lk) {
    int split = 1;
    while (split < 8 && units * split * 2 <= kFill && (Lk + kTile - 1) / kTile >= 8 * split) split *= 2;
    return split;
}

// CTAs per key tile (dkv): 1, or where the tiles leave SMs idle the part of the group's query heads, up to 8, with which
// they fill it; beyond one wave only if a CTA keeps eight query tiles or more. 2048 queries and keys, 15/5 heads of 64 (80
// tiles): 86 us whole, 43 by heads; 1000 of 8/1 heads of 96 (8 tiles): 119 and 25; one query over 2048 keys: 10 and 20.
int split_heads(int64_t units, int group, int q_tiles) {
    int split = 1;
    for (int c = 2; c <= 8 && units * split < kFill; ++c)
        if (group % c == 0 && (units * c <= kFill || group / c * q_tiles >= 8)) split = c;
    return split;
}

template <int HD>
int run_forward(const lamq_attention_args &a, const Shape &s, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    if (int e = tile_map(&mq, a.q, s.B, s.Hq, s.Lq, s.D)) return e;
    if (s.Lk > 0) {
        if (int e = tile_map(&mk, a.k, s.B, s.Hkv, s.Lk, s.D)) return e;
        if (int e = tile_map(&mv, a.v, s.B, s.Hkv, s.Lk, s.D)) return e;
    } else {
        mk = mv = mq;  // not read: no query meets a key tile
    }
    const int64_t pairs = (s.lq_pad / kTile + 1) / 2, blocks = pairs * s.Hq * s.B;
    LAMQ_REQUIRE(blocks <= INT_MAX, "lamq_attention_forward: too many query tiles");
    auto *k = attention_forward_kernel<HD>;
    if (cudaError_t e = smem_limit_once((const void *)k, (int)Sizes<HD>::FWD_SMEM))
        return launch_failed("lamq_attention_forward", e);
    const int split = split_keys(blocks, s.Lk);
    if (cudaError_t e = launch_split(k, blocks, split, Sizes<HD>::FWD_SMEM, st, mq, mk, mv, s, rows_of(a.o), a.lse, split))
        return launch_failed("lamq_attention_forward", e);
    LAMQ_CHECK_LAUNCH("lamq_attention_forward");
    return LAMQ_OK;
}

template <int HD>
int run_backward(const lamq_attention_args &a, const Shape &s, float *lse2, float *D, cudaStream_t st) {
    CUtensorMap mq, mk, mv, mg;
    const bool queries = s.Lq > 0, keys = s.Lk > 0;
    if (queries) {
        if (int e = tile_map(&mq, a.q, s.B, s.Hq, s.Lq, s.D)) return e;
        if (int e = tile_map(&mg, a.d_o, s.B, s.Hq, s.Lq, s.D)) return e;
    }
    if (keys) {
        if (int e = tile_map(&mk, a.k, s.B, s.Hkv, s.Lk, s.D)) return e;
        if (int e = tile_map(&mv, a.v, s.B, s.Hkv, s.Lk, s.D)) return e;
    }
    if (!keys) mk = mv = mq;   // not read: no query meets a key tile
    if (!queries) mq = mg = mk;
    if (queries) {
        const int64_t tiles = (int64_t)(s.lq_pad / kTile) * s.Hq * s.B;
        LAMQ_REQUIRE(tiles <= INT_MAX, "lamq_attention_backward: too many query tiles");
        auto *k = attention_dq_kernel<HD>;
        if (cudaError_t e = smem_limit_once((const void *)k, (int)Sizes<HD>::DQ_SMEM))
            return launch_failed("lamq_attention_backward", e);
        const int split = split_keys(tiles, s.Lk);
        if (cudaError_t e = launch_split(k, tiles, split, Sizes<HD>::DQ_SMEM, st, mq, mk, mv, mg, s,
                                         (const float *)a.lse, lse2, D, rows_of(a.o), rows_of(a.dq), split))
            return launch_failed("lamq_attention_backward", e);
        LAMQ_CHECK_LAUNCH("lamq_attention_backward dq");
    }
    if (keys) {
        const int64_t tiles = (int64_t)((s.Lk + kTile - 1) / kTile) * s.Hkv * s.B;
        LAMQ_REQUIRE(tiles <= INT_MAX, "lamq_attention_backward: too many key tiles");
        auto *k = attention_dkv_kernel<HD>;
        if (cudaError_t e = smem_limit_once((const void *)k, (int)Sizes<HD>::DKV_SMEM))
            return launch_failed("lamq_attention_backward", e);
        const int split = split_heads(tiles, s.group, s.lq_pad / kTile);
        if (cudaError_t e = launch_split(k, tiles, split, Sizes<HD>::DKV_SMEM, st, mq, mk, mv, mg, s,
                                         (const float *)lse2, (const float *)D, rows_of(a.dk), rows_of(a.dv), split))
            return launch_failed("lamq_attention_backward", e);
        LAMQ_CHECK_LAUNCH("lamq_attention_backward dkv");
    }
    return LAMQ_OK;
}

}  // namespace
}  // namespace lamq

using namespace lamq;

static_assert(sizeof(lamq_heads) == 32 && sizeof(lamq_attention_args) == 328, "lamq_attention_args' layout in the C ABI");

extern "C" int lamq_attention_forward(const lamq_attention_args *args, int *status, lamq_stream_t stream) {
    const char *fn = "lamq_attention_forward";
    LAMQ_REQUIRE(args != nullptr, "%s: null pointer", fn);
    const lamq_attention_args &a = *args;
    Shape s{};
    bool empty = false;
    if (int e = shape_of(fn, a, status, s, empty)) return e;
    if (empty || s.Lq == 0) return LAMQ_OK;
    if (int e = check_heads(fn, "q", a.q, s.B, s.Hq, s.Lq)) return e;
    if (int e = check_heads(fn, "o", a.o, s.B, s.Hq, s.Lq)) return e;
    if (s.Lk > 0) {
        if (int e = check_heads(fn, "k", a.k, s.B, s.Hkv, s.Lk)) return e;
        if (int e = check_heads(fn, "v", a.v, s.B, s.Hkv, s.Lk)) return e;
    }
    LAMQ_REQUIRE(a.lse != nullptr, "%s: null pointer (lse)", fn);
    return s.D <= 64 ? run_forward<64>(a, s, (cudaStream_t)stream) : run_forward<128>(a, s, (cudaStream_t)stream);
}

extern "C" size_t lamq_attention_backward_workspace_size(int64_t batch, int heads, int64_t q_len) {
    if (batch <= 0 || heads <= 0 || q_len <= 0) return 0;
    return (size_t)batch * (size_t)heads * (size_t)((q_len + kTile - 1) / kTile * kTile) * 2 * sizeof(float);
}

extern "C" int lamq_attention_backward(const lamq_attention_args *args, void *workspace, size_t workspace_bytes,
                                       int *status, lamq_stream_t stream) {
    const char *fn = "lamq_attention_backward";
    LAMQ_REQUIRE(args != nullptr, "%s: null pointer", fn);
    const lamq_attention_args &a = *args;
    Shape s{};
    bool empty = false;
    if (int e = shape_of(fn, a, status, s, empty)) return e;
    if (empty || (s.Lq == 0 && s.Lk == 0)) return LAMQ_OK;
    if (s.Lq > 0) {
        if (int e = check_heads(fn, "q", a.q, s.B, s.Hq, s.Lq)) return e;
        if (int e = check_heads(fn, "o", a.o, s.B, s.Hq, s.Lq)) return e;
        if (int e = check_heads(fn, "do", a.d_o, s.B, s.Hq, s.Lq)) return e;
        if (int e = check_heads(fn, "dq", a.dq, s.B, s.Hq, s.Lq)) return e;
        LAMQ_REQUIRE(a.lse != nullptr, "%s: null pointer (lse)", fn);
    }
    if (s.Lk > 0) {
        if (int e = check_heads(fn, "k", a.k, s.B, s.Hkv, s.Lk)) return e;
        if (int e = check_heads(fn, "v", a.v, s.B, s.Hkv, s.Lk)) return e;
        if (int e = check_heads(fn, "dk", a.dk, s.B, s.Hkv, s.Lk)) return e;
        if (int e = check_heads(fn, "dv", a.dv, s.B, s.Hkv, s.Lk)) return e;
    }
    const size_t need = lamq_attention_backward_workspace_size(s.B, s.Hq, s.Lq);
    LAMQ_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
                 "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", fn, need, workspace_bytes);
    float *lse2 = reinterpret_cast<float *>(workspace);
    float *D = lse2 + need / (2 * sizeof(float));
    return s.D <= 64 ? run_backward<64>(a, s, lse2, D, (cudaStream_t)stream)
                     : run_backward<128>(a, s, lse2, D, (cudaStream_t)stream);
}
