// The embedding of a training step: rows of the table looked up and scaled, and the table's gradient.
//
//   lookup     Y_t = scale · E[id_t]
//   gradient   dE_v = scale · Σ_{t: id_t = v} dY_t        (rows no token names are zero)
//
// Both are bound by memory: the lookup reads each token's row and writes it, the gradient reads dY once and writes the
// whole of dE once (rows nobody named included), so for a large table most of its bytes are zeros.
//
// The gradient's sums have a fixed order and no float is added by an atomic: repeated calls agree bit for bit.
//
// Up to kDirectTokens tokens (one launch, no workspace): each block owns a range of the table's rows, reads all ids,
// keeps those of its range in the order of the tokens and links the tokens of a row; then it writes its rows, sums or
// zeros. Every id is read by every block, which a few thousand ids from L2 can afford.
//
// More tokens (three launches): some blocks of a cooperative kernel sort the tokens by id (a stable radix sort, digits of
// up to 9 bits: counts per block, then each block places its tokens) while the others write the zeros; then the sorted
// tokens, cut into chunks, are summed in fp32. A row whose tokens lie in one chunk is written at once; a row that crosses chunks (a
// frequent token: its run may be a tenth of all tokens) leaves a partial per chunk, and these are added chunk by chunk
// by a last kernel.
#include <algorithm>
#include <climits>
#include <cstdint>

#include <cuda_bf16.h>

#include "../../include/lamq_b200_train.h"
#include "lamq_common.cuh"

namespace lamq {
namespace {

// The status word keeps the greatest code: a bad id (LAMQ_ERR_INVALID) does not hide a wait that gave up (LAMQ_ERR_TIMEOUT).
static_assert(LAMQ_ERR_TIMEOUT > LAMQ_ERR_INVALID, "atomicMax keeps the graver error");

// ---- element access: V values of T at p as fp32, V·sizeof(T) = 16 bytes where rows are 16-byte aligned, else V = 1

template <typename T, int V>
struct Pack;

template <>
struct Pack<float, 4> {
    float4 v;
    __device__ static Pack load(const float *p) { return {__ldg(reinterpret_cast<const float4 *>(p))}; }
    __device__ static Pack load_plain(const float *p) { return {*reinterpret_cast<const float4 *>(p)}; }
    __device__ void get(float (&f)[4]) const { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
    __device__ void set(const float (&f)[4]) { v = make_float4(f[0], f[1], f[2], f[3]); }
    __device__ void store(float *p) const { *reinterpret_cast<float4 *>(p) = v; }
    __device__ void store_stream(float *p) const { __stcs(reinterpret_cast<float4 *>(p), v); }
};

template <>
struct Pack<float, 1> {
    float v;
    __device__ static Pack load(const float *p) { return {__ldg(p)}; }
    __device__ static Pack load_plain(const float *p) { return {*p}; }
    __device__ void get(float (&f)[1]) const { f[0] = v; }
    __device__ void set(const float (&f)[1]) { v = f[0]; }
    __device__ void store(float *p) const { *p = v; }
    __device__ void store_stream(float *p) const { __stcs(p, v); }
};

template <>
struct Pack<__nv_bfloat16, 8> {
    uint4 v;
    __device__ static Pack load(const __nv_bfloat16 *p) { return {__ldg(reinterpret_cast<const uint4 *>(p))}; }
    __device__ static Pack load_plain(const __nv_bfloat16 *p) { return {*reinterpret_cast<const uint4 *>(p)}; }
    __device__ void get(float (&f)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ void set(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ void store(__nv_bfloat16 *p) const { *reinterpret_cast<uint4 *>(p) = v; }
    __device__ void store_stream(__nv_bfloat16 *p) const { __stcs(reinterpret_cast<uint4 *>(p), v); }
};

template <>
struct Pack<__nv_bfloat16, 1> {
    __nv_bfloat16 v;
    __device__ static Pack load(const __nv_bfloat16 *p) { return {*p}; }
    __device__ static Pack load_plain(const __nv_bfloat16 *p) { return {*p}; }
    __device__ void get(float (&f)[1]) const { f[0] = __bfloat162float(v); }
    __device__ void set(const float (&f)[1]) { v = __float2bfloat16_rn(f[0]); }
    __device__ void store(__nv_bfloat16 *p) const { *p = v; }
    __device__ void store_stream(__nv_bfloat16 *p) const { *p = v; }
};

__device__ __forceinline__ int64_t id_at(const void *ids, int ids64, int64_t t) {
    return ids64 ? __ldg(reinterpret_cast<const long long *>(ids) + t)
                 : (int64_t)__ldg(reinterpret_cast<const int *>(ids) + t);
}

// ---- lookup: a warp copies kLookupVecs packs per lane of one token's row

constexpr int kThreads = 256;
constexpr int kLookupVecs = 4;

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(const T *__restrict__ table, int64_t ldt, int64_t rows, int packs, int parts,
                  const void *__restrict__ ids, int ids64, int64_t n, float scale, int64_t padding,
                  T *__restrict__ out, int64_t ldo, int *status) {
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int64_t t = parts == 1 ? item : item / parts;
    if (t >= n) return;
    const int first = (int)(parts == 1 ? 0 : item - t * parts) * (32 * kLookupVecs) + lane;
    const int64_t id = id_at(ids, ids64, t);
    const bool valid = id >= 0 && id < rows, live = valid && id != padding;
    if (!valid && first == 0) atomicMax(status, LAMQ_ERR_INVALID);
    const T *src = table + (live ? id : 0) * ldt;
    T *dst = out + t * ldo;
    Pack<T, V> x[kLookupVecs];
#pragma unroll
    for (int i = 0; i < kLookupVecs; ++i)
        if (live && first + 32 * i < packs) x[i] = Pack<T, V>::load(src + (int64_t)(first + 32 * i) * V);
#pragma unroll
    for (int i = 0; i < kLookupVecs; ++i) {
        if (first + 32 * i >= packs) break;
        float f[V];
        if (live) x[i].get(f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = live ? f[e] * scale : 0.f;
        x[i].set(f);
        x[i].store_stream(dst + (int64_t)(first + 32 * i) * V);
    }
}

// ---- gradient, few tokens

// Tokens up to which the gradient is one launch: what its lists in shared memory hold. Measured at 2048 of them, us (so,
// sorted): 49152 x 960 fp32 46.5, 55.8, bf16 33.5, 43.8; 8000 x 1024 fp32 17, 36; 131072 x 64 13, 41. Where the zeros are most
// of the work the sorted path's writers do better: 131072 x 2560 bf16 160, 136, and 147, 129 at 64 tokens.
constexpr int kDirectTokens = 2048;
constexpr int kDirectRows = 2048;   // rows a block can own
constexpr int kDirectCols = 32;     // packs of columns a block can own
constexpr int kDirectBlocks = 4;    // blocks per SM
constexpr int kFrequent = 32;       // tokens of a row from which on the block shares it
constexpr int kAhead = 8;           // rows of dY in flight per thread

struct GradParams {
    const void *ids;
    int ids64;
    int64_t n, rows, padding, ldy, lde;
    int packs;
    float scale;
    int accumulate;
    int *status;
};

template <typename T, int V>
__device__ __forceinline__ void write_row(T *dst, float (&acc)[V], float scale, int accumulate) {
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= scale;
    Pack<T, V> p;
    if (accumulate) {
        float old[V];
        Pack<T, V>::load_plain(dst).get(old);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += old[e];
    }
    p.set(acc);
    p.store(dst);
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> zero_pack() {
    float z[V];
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = 0.f;
    Pack<T, V> p;
    p.set(z);
    return p;
}

// The sum of `count` tokens' rows in order, one pack of columns.
template <typename T, int V>
__device__ __forceinline__ void sum_tokens(const T *__restrict__ dy, int64_t ldy, const uint16_t *order, int count,
                                           float (&acc)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    for (int k = 0; k < count; k += kAhead) {
        Pack<T, V> x[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (k + a < count) x[a] = Pack<T, V>::load(dy + (int64_t)order[k + a] * ldy);
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (k + a < count) {
                float f[V];
                x[a].get(f);
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += f[e];
            }
    }
}

// Block (b, c): rows [b·own, (b + 1)·own), packs of columns [c·tpr, (c + 1)·tpr); tpr lanes (a power of two up to 32)
// share a row. Warp 0 orders the range's tokens by row while the others write the zeros of the rows without one; then a
// slot of tpr lanes sums each row, and all slots together a frequent token's row: each a part of its tokens, the parts
// added in order.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 4)
    gradient_direct_kernel(const T *__restrict__ dy, T *__restrict__ dE, GradParams p, int own, int tpr) {
    constexpr int kWarps = kThreads / 32, kRounds = kDirectTokens / kThreads;
    __shared__ uint16_t count[kDirectRows], start[kDirectRows];  // of each row of the range: tokens, place in order
    __shared__ uint8_t touched[kDirectRows];
    __shared__ uint16_t pos[kDirectTokens], row[kDirectTokens], rank[kDirectTokens];  // the range's tokens as they come
    __shared__ uint16_t order[kDirectTokens], rows[kDirectTokens];  // by row; the rows that have tokens
    __shared__ float part[kThreads * V];
    __shared__ int warp_count[kWarps], nrow;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r0 = (int64_t)blockIdx.x * own;
    const int nrows = (int)std::min<int64_t>(own, p.rows - r0);
    for (int i = tid; i < nrows; i += kThreads) {
        count[i] = 0;
        touched[i] = 0;
    }
    // each warp takes a contiguous piece of the tokens
    const int t0 = warp * (kRounds * 32) + lane;
    int64_t my[kRounds];
#pragma unroll
    for (int q = 0; q < kRounds; ++q) my[q] = t0 + 32 * q < p.n ? id_at(p.ids, p.ids64, t0 + 32 * q) : 0;
    uint32_t mask[kRounds];
    int mine = 0;
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
        const bool in = t0 + 32 * q < p.n;
        if (blockIdx.x == 0 && in && (my[q] < 0 || my[q] >= p.rows)) atomicMax(p.status, LAMQ_ERR_INVALID);
        mask[q] = __ballot_sync(0xffffffffu, in && my[q] >= r0 && my[q] < r0 + nrows && my[q] != p.padding);
        mine += __popc(mask[q]);
    }
    if (lane == 0) warp_count[warp] = mine;
    __syncthreads();
    int at = 0, m = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += warp_count[w];
        m += warp_count[w];
    }
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
        if (mask[q] >> lane & 1u) {
            const int to = at + __popc(mask[q] & ((1u << lane) - 1u));
            pos[to] = (uint16_t)(t0 + 32 * q);
            row[to] = (uint16_t)(my[q] - r0);
            touched[my[q] - r0] = 1;
        }
        at += __popc(mask[q]);
    }
    __syncthreads();
    const int per_warp = 32 / tpr, sub = lane % tpr, slot = warp * per_warp + lane / tpr, slots = kWarps * per_warp;
    const int col = blockIdx.y * tpr + sub;
    const bool in_cols = col < p.packs;
    T *const base = dE + r0 * p.lde + (int64_t)col * V;
    dy += (int64_t)col * V;
    if (warp > 0) {
        if (!p.accumulate && in_cols) {
            const Pack<T, V> z = zero_pack<T, V>();
            for (int r = slot - per_warp; r < nrows; r += slots - per_warp)
                if (!touched[r]) z.store(base + (int64_t)r * p.lde);
        }
    } else {
        int have = 0;
        for (int b = 0; b < m; b += 32) {  // each token's rank among its row's
            const int i = b + lane;
            const bool in = i < m;
            const uint32_t key = in ? row[i] : 0x10000u + lane;
            const uint32_t peers = __match_any_sync(0xffffffffu, key);
            const int before = in ? count[key] : 0, earlier = __popc(peers & ((1u << lane) - 1u));
            const uint32_t f = __ballot_sync(0xffffffffu, in && before + earlier == 0);
            __syncwarp();
            if (in) {
                rank[i] = (uint16_t)(before + earlier);
                if (before + earlier == 0) rows[have + __popc(f & ((1u << lane) - 1u))] = (uint16_t)key;
                if (earlier == 0) count[key] = (uint16_t)(before + __popc(peers));
            }
            have += __popc(f);
            __syncwarp();
        }
        int first = 0;
        for (int b = 0; b < have; b += 32) {
            const int c = b + lane < have ? count[rows[b + lane]] : 0;
            int incl = c;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (b + lane < have) start[rows[b + lane]] = (uint16_t)(first + incl - c);
            first += __shfl_sync(0xffffffffu, incl, 31);
        }
        __syncwarp();
        for (int i = lane; i < m; i += 32) order[start[row[i]] + rank[i]] = pos[i];
        if (lane == 0) nrow = have;
    }
    __syncthreads();
    const int have = nrow;
    float acc[V];
    if (m > kFrequent)
        for (int k = 0; k < have; ++k) {
            const int r = rows[k], c = count[r];
            if (c <= kFrequent) continue;
            const int from = c * slot / slots, to = c * (slot + 1) / slots;
            if (in_cols) {
                sum_tokens<T, V>(dy, p.ldy, order + start[r] + from, to - from, acc);
#pragma unroll
                for (int e = 0; e < V; ++e) part[(slot * tpr + sub) * V + e] = acc[e];
            }
            __syncthreads();
            if (in_cols && slot == 0) {
                for (int w = 1; w < slots; ++w)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] += part[(w * tpr + sub) * V + e];
                write_row<T, V>(base + (int64_t)r * p.lde, acc, p.scale, p.accumulate);
            }
            __syncthreads();
        }
    if (!in_cols) return;
    for (int k = slot; k < have; k += slots) {
        const int r = rows[k], c = count[r];
        if (c > kFrequent) continue;
        sum_tokens<T, V>(dy, p.ldy, order + start[r], c, acc);
        write_row<T, V>(base + (int64_t)r * p.lde, acc, p.scale, p.accumulate);
    }
}

// ---- gradient, many tokens: sort (and write the zeros), sum, join

constexpr int kMaxDigitBits = 9, kMaxBins = 1 << kMaxDigitBits;
constexpr int kRounds = 4, kTile = kThreads * kRounds;  // tokens that a block ranks at a time
constexpr int kWarps = kThreads / 32;
constexpr int kMaxSorters = 64;                         // blocks that sort
constexpr unsigned long long kBarrierTimeoutNs = 2000000000ull;

struct SortedParams {
    GradParams g;
    int sorters, passes, bits;
    int64_t per_sorter;       // tokens of each sorting block, a multiple of kTile
    uint32_t *keys[2], *pos[2], *counts;
    int chunk;
    int64_t chunks;
    float *head, *tail;       // a partial per chunk: of the row that began before it, of the row that goes on after it
    unsigned *barrier;        // arrivals of the sorting blocks, zero before the launch
    unsigned *gave_up;        // not zero once a sorting block has given up, zero before the launch: no keys to go by
};

// The blocks that count on `counter` have arrived `target` times in all and see each other's writes. Bounded.
__device__ __forceinline__ bool wait_all(unsigned *counter, unsigned target, int *status, int *shared_ok) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(counter, 1u);
        int ok = 1;
        unsigned long long t0, t;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
        for (unsigned it = 1;; ++it) {
            unsigned v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
            if (v >= target) break;
            if ((it & 255u) == 0u) {
                asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
                if (t - t0 > kBarrierTimeoutNs) {
                    atomicMax(status, LAMQ_ERR_TIMEOUT);
                    ok = 0;
                    break;
                }
            }
        }
        __threadfence();
        *shared_ok = ok;
    }
    __syncthreads();
    return *shared_ok != 0;
}

__device__ __forceinline__ uint32_t key_at(const SortedParams &s, int pass, int64_t t) {
    if (pass > 0) return s.keys[(pass - 1) & 1][t];
    const int64_t id = id_at(s.g.ids, s.g.ids64, t);  // a padding or invalid id sorts last, as `rows`
    return (id < 0 || id >= s.g.rows || id == s.g.padding) ? (uint32_t)s.g.rows : (uint32_t)id;
}

// One sorting block's part: its tokens' digits counted, then (all blocks' counts known) its tokens placed in order.
__device__ bool sort_tokens(const SortedParams &s, uint32_t (*seen)[kMaxBins], uint32_t *place, uint32_t *scan,
                            int *shared_ok) {
    const int me = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << s.bits;
    const int64_t lo = me * s.per_sorter, hi = std::min<int64_t>(s.g.n, lo + s.per_sorter);
    unsigned target = 0;
    for (int pass = 0; pass < s.passes; ++pass) {
        const int shift = pass * s.bits;
        for (int b = threadIdx.x; b < bins; b += kThreads) place[b] = 0;
        __syncthreads();
        for (int64_t t = lo + threadIdx.x; t < hi; t += kThreads) {
            const uint32_t key = key_at(s, pass, t);
            if (pass == 0 && key == (uint32_t)s.g.rows) {
                const int64_t id = id_at(s.g.ids, s.g.ids64, t);
                if (id < 0 || id >= s.g.rows) atomicMax(s.g.status, LAMQ_ERR_INVALID);
            }
            atomicAdd(&place[(key >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        for (int b = threadIdx.x; b < bins; b += kThreads) s.counts[b * kMaxSorters + me] = place[b];
        if (!wait_all(s.barrier, target += s.sorters, s.g.status, shared_ok)) return false;
        // this block's first place for each digit: all smaller digits, and the same digit in the blocks before
        uint32_t mine[kMaxBins / kThreads], sum[kMaxBins / kThreads], run = 0;
#pragma unroll
        for (int q = 0; q < kMaxBins / kThreads; ++q) {
            const int b = threadIdx.x * (kMaxBins / kThreads) + q;
            mine[q] = sum[q] = 0;
            if (b < bins) {
#pragma unroll 8
                for (int w = 0; w < kMaxSorters; w += 4) {
                    const uint4 c = __ldcg(reinterpret_cast<const uint4 *>(s.counts + b * kMaxSorters + w));
                    const uint32_t cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (w + e < me) mine[q] += cs[e];
                        if (w + e < s.sorters) sum[q] += cs[e];
                    }
                }
            }
            run += sum[q];
        }
        uint32_t incl = run;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        uint32_t at = incl - run;
        for (int w = 0; w < warp; ++w) at += scan[w];
#pragma unroll
        for (int q = 0; q < kMaxBins / kThreads; ++q) {
            const int b = threadIdx.x * (kMaxBins / kThreads) + q;
            if (b < bins) place[b] = at + mine[q];
            at += sum[q];
        }
        uint32_t *const ko = s.keys[pass & 1], *const po = s.pos[pass & 1];
        for (int64_t t0 = lo; t0 < hi; t0 += kTile) {  // each warp ranks a contiguous piece, so equal digits keep order
            __syncthreads();
            for (int b = lane; b < bins; b += 32) seen[warp][b] = 0;
            __syncwarp();
            uint32_t key[kRounds], rank[kRounds];
            const int64_t w0 = t0 + warp * (32 * kRounds) + lane;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) key[r] = w0 + r * 32 < hi ? key_at(s, pass, w0 + r * 32) : 0u;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const bool in = w0 + r * 32 < hi;
                const uint32_t digit = in ? (key[r] >> shift) & (bins - 1) : (uint32_t)bins;  // the tail matches itself
                const uint32_t peers = __match_any_sync(0xffffffffu, digit);
                const uint32_t before = in ? seen[warp][digit] : 0u;
                rank[r] = before + __popc(peers & ((1u << lane) - 1u));
                __syncwarp();
                if (in && (__ffs(peers) - 1) == lane) seen[warp][digit] = before + __popc(peers);
                __syncwarp();
            }
            __syncthreads();
            for (int b = threadIdx.x; b < bins; b += kThreads) {  // each warp's first place for each digit
                uint32_t next = place[b];
                for (int w = 0; w < kWarps; ++w) {
                    const uint32_t c = seen[w][b];
                    seen[w][b] = next;
                    next += c;
                }
                place[b] = next;
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int64_t t = w0 + r * 32;
                if (t >= hi) break;
                const uint32_t to = seen[warp][(key[r] >> shift) & (bins - 1)] + rank[r];
                ko[to] = key[r];
                po[to] = pass > 0 ? s.pos[(pass - 1) & 1][t] : (uint32_t)t;
            }
        }
        if (pass + 1 < s.passes && !wait_all(s.barrier, target += s.sorters, s.g.status, shared_ok)) return false;
    }
    return true;
}

template <int V>
__device__ __forceinline__ void write_partial(float *dst, const float (&acc)[V]) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4)
            *reinterpret_cast<float4 *>(dst + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) dst[e] = acc[e];
    }
}

template <int V>
__device__ __forceinline__ void read_partial(const float *src, float (&f)[V]) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(src + e));
            f[e] = v.x, f[e + 1] = v.y, f[e + 2] = v.z, f[e + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = __ldcg(src + e);
    }
}

// The first blocks sort the tokens by id while the others write the zeros.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 4)
    gradient_sort_kernel(T *__restrict__ dE, SortedParams s) {
    __shared__ uint32_t seen[kWarps][kMaxBins], place[kMaxBins], scan[kWarps];
    __shared__ int shared_ok;
    if ((int)blockIdx.x < s.sorters) {
        if (!sort_tokens(s, seen, place, scan, &shared_ok) && threadIdx.x == 0) *s.gave_up = 1u;
        return;
    }
    const int64_t total = s.g.rows * s.g.packs, step = (int64_t)(gridDim.x - s.sorters) * kThreads;
    const Pack<T, V> z = zero_pack<T, V>();
    for (int64_t i = (int64_t)(blockIdx.x - s.sorters) * kThreads + threadIdx.x; i < total; i += step)
        z.store(dE + (i / s.g.packs) * s.g.lde + (i % s.g.packs) * V);
}

constexpr int kSumThreads = 128;

// Block (chunk, column part): the chunk's tokens in sorted order, a thread per pack of columns. (As a phase of the
// cooperative kernel, with its registers and two blocks per SM, this took 200 us instead of 79 for 65536 x 2560 bf16.)
template <typename T, int V>
__global__ void __launch_bounds__(kSumThreads)
    gradient_sum_kernel(const T *__restrict__ dy, T *__restrict__ dE, SortedParams s, const uint32_t *__restrict__ keys,
                        const uint32_t *__restrict__ pos) {
    constexpr int kBatch = 8;
    const int64_t c = blockIdx.x, lo = c * s.chunk, hi = std::min<int64_t>(s.g.n, lo + s.chunk);
    const int col = blockIdx.y * blockDim.x + threadIdx.x;
    if (col >= s.g.packs) return;
    const uint32_t dead = (uint32_t)s.g.rows;
    const uint32_t prev = lo > 0 ? keys[lo - 1] : dead, next = hi < s.g.n ? keys[hi] : dead;
    if (*s.gave_up) return;  // without a whole sort, keys and pos may hold anything
    float acc[V];
    bool open = false;   // acc holds tokens of row `cur`
    bool first = true;   // no row has been closed in this chunk yet
    uint32_t cur = dead;
    const auto close = [&](bool goes_on) {
        if (!open) return;
        const int64_t at = (c * s.g.packs + col) * V;
        if (first && cur == prev) write_partial<V>(s.head + at, acc);
        else if (goes_on) write_partial<V>(s.tail + at, acc);
        else write_row<T, V>(dE + (int64_t)cur * s.g.lde + (int64_t)col * V, acc, s.g.scale, s.g.accumulate);
        open = false;
        first = false;
    };
    for (int64_t base = lo; base < hi; base += kBatch) {
        Pack<T, V> x[kBatch];
        uint32_t key[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            key[i] = base + i < hi ? keys[base + i] : dead;
            if (key[i] < dead) x[i] = Pack<T, V>::load(dy + (int64_t)pos[base + i] * s.g.ldy + (int64_t)col * V);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (base + i >= hi) break;
            if (key[i] >= dead) {  // padding sorts last: nothing follows
                close(false);
                return;
            }
            float f[V];
            x[i].get(f);
            if (open && key[i] == cur) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += f[e];
            } else {
                close(false);
                cur = key[i];
                open = true;
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = f[e];
            }
        }
    }
    close(cur == next);
}

// A warp per chunk and 32 packs of columns: where a row goes on past the chunk in which it began, its partials in chunk
// order.
template <typename T, int V>
__global__ void __launch_bounds__(kSumThreads)
    gradient_join_kernel(T *__restrict__ dE, SortedParams s, const uint32_t *__restrict__ keys, int slices) {
    constexpr int kBatch = 16;
    const int64_t item = (int64_t)blockIdx.x * (kSumThreads / 32) + (threadIdx.x >> 5), c = item / slices;
    const int col = (int)(item - c * slices) * 32 + (threadIdx.x & 31);
    const int64_t lo = c * s.chunk, hi = lo + s.chunk;
    if (hi >= s.g.n) return;
    const uint32_t key = keys[hi - 1], next = keys[hi], begin = keys[lo], prev = lo > 0 ? keys[lo - 1] : (uint32_t)s.g.rows;
    if (*s.gave_up || key >= (uint32_t)s.g.rows || next != key) return;  // no sort; nothing goes on
    if (begin == key && prev == key) return;               // it began before
    int64_t end = c + 1;  // the row's last chunk: the first whose next token is another's, 32 at a time
    for (;; end += 32) {
        const int64_t after = (end + (threadIdx.x & 31) + 1) * s.chunk;
        const uint32_t stop = __ballot_sync(0xffffffffu, after >= s.g.n || keys[after] != key);
        if (stop) {
            end += __ffs(stop) - 1;
            break;
        }
    }
    if (col >= s.g.packs) return;
    const int64_t step = (int64_t)s.g.packs * V, at = (int64_t)col * V;
    float acc[V];
    read_partial<V>(s.tail + c * step + at, acc);
    for (int64_t k = c + 1; k <= end; k += kBatch) {
        float f[kBatch][V];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (k + i <= end) read_partial<V>(s.head + (k + i) * step + at, f[i]);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (k + i <= end) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += f[i][e];
            }
    }
    write_row<T, V>(dE + (int64_t)key * s.g.lde + at, acc, s.g.scale, s.g.accumulate);
}

// Tokens per chunk: enough chunks to fill the device for few tokens, long ones (fewer partials) for many.
int chunk_tokens(int64_t n) { return (int)std::min<int64_t>(64, std::max<int64_t>(8, n / 1024)); }

struct Layout {
    int64_t chunks;
    size_t keys, counts, partial, total;  // bytes of one buffer of each kind, and of all
};

Layout layout_of(int64_t n, int d) {
    Layout L;
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    L.chunks = (n + chunk_tokens(n) - 1) / chunk_tokens(n);
    L.keys = up((size_t)n * 4);
    L.counts = up((size_t)kMaxSorters * kMaxBins * 4);
    L.partial = up((size_t)L.chunks * (size_t)d * 4);
    L.total = 256 + 4 * L.keys + L.counts + 2 * L.partial;
    return L;
}

bool packs_ok(const void *p, int64_t ld, int d, int V, size_t size) {
    return d % V == 0 && ld % V == 0 && reinterpret_cast<uintptr_t>(p) % (V * size) == 0;
}

template <typename T, int V>
int run_lookup(const void *table, int64_t ldt, int64_t rows, int d, const void *ids, int ids64, int64_t n, float scale,
               int64_t padding, void *out, int64_t ldo, int *status, cudaStream_t s) {
    const int packs = d / V, parts = (packs + 32 * kLookupVecs - 1) / (32 * kLookupVecs);
    const int64_t blocks = (n * parts + kThreads / 32 - 1) / (kThreads / 32);
    LAMQ_REQUIRE(blocks <= INT_MAX, "lamq_embedding_lookup: too many tokens");
    lookup_kernel<T, V><<<(unsigned)blocks, kThreads, 0, s>>>(reinterpret_cast<const T *>(table), ldt, rows, packs,
                                                              parts, ids, ids64, n, scale, padding,
                                                              reinterpret_cast<T *>(out), ldo, status);
    LAMQ_CHECK_LAUNCH("lamq_embedding_lookup");
    return LAMQ_OK;
}

int cuda_failed(cudaError_t e) {
    set_error("lamq_embedding_gradient: %s", cudaGetErrorString(e));
    return LAMQ_ERR_CUDA;
}

template <typename T, int V>
int run_gradient(const void *dyv, void *dEv, GradParams g, int d, void *workspace, cudaStream_t s) {
    const T *dy = reinterpret_cast<const T *>(dyv);
    T *dE = reinterpret_cast<T *>(dEv);
    g.packs = d / V;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_failed(e);
    if (g.n <= kDirectTokens) {
        int tpr = 1;
        while (tpr < kDirectCols && tpr < g.packs) tpr *= 2;
        const int slices = (g.packs + tpr - 1) / tpr;
        const int64_t want = std::max<int64_t>(1, (int64_t)sms * kDirectBlocks / slices);
        const int own = (int)std::min<int64_t>(kDirectRows, (g.rows + want - 1) / want);
        const dim3 grid((unsigned)((g.rows + own - 1) / own), (unsigned)slices);
        LAMQ_REQUIRE(slices <= 65535, "lamq_embedding_gradient: rows too long");
        gradient_direct_kernel<T, V><<<grid, kThreads, 0, s>>>(dy, dE, g, own, tpr);
        LAMQ_CHECK_LAUNCH("lamq_embedding_gradient");
        return LAMQ_OK;
    }
    const Layout L = layout_of(g.n, d);
    char *ws = reinterpret_cast<char *>(workspace);
    SortedParams p{};
    p.g = g;
    p.barrier = reinterpret_cast<unsigned *>(ws);
    p.gave_up = p.barrier + 1;
    for (int i = 0; i < 2; ++i) {
        p.keys[i] = reinterpret_cast<uint32_t *>(ws + 256 + (2 * i) * L.keys);
        p.pos[i] = reinterpret_cast<uint32_t *>(ws + 256 + (2 * i + 1) * L.keys);
    }
    p.counts = reinterpret_cast<uint32_t *>(ws + 256 + 4 * L.keys);
    p.head = reinterpret_cast<float *>(ws + 256 + 4 * L.keys + L.counts);
    p.tail = reinterpret_cast<float *>(ws + 256 + 4 * L.keys + L.counts + L.partial);
    p.chunk = chunk_tokens(g.n);
    p.chunks = L.chunks;
    int key_bits = 1;
    while ((g.rows >> key_bits) != 0) ++key_bits;  // keys are 0 .. rows
    p.passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    const int64_t tiles = (g.n + kTile - 1) / kTile;
    p.per_sorter = (tiles + kMaxSorters - 1) / kMaxSorters * kTile;
    p.sorters = (int)((g.n + p.per_sorter - 1) / p.per_sorter);
    const auto kernel = gradient_sort_kernel<T, V>;
    int per_sm = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, 0);
    if (e == cudaSuccess) e = cudaMemsetAsync(p.barrier, 0, 2 * sizeof(unsigned), s);
    if (e != cudaSuccess) return cuda_failed(e);
    const int grid = g.accumulate ? p.sorters : p.sorters + sms * std::max(1, std::min(per_sm, 4) - 1);
    LAMQ_REQUIRE(grid <= sms * per_sm, "lamq_embedding_gradient: the device has too few multiprocessors");
    void *args[] = {&dE, &p};
    e = cudaLaunchCooperativeKernel((const void *)kernel, dim3(grid), dim3(kThreads), args, 0, s);
    if (e != cudaSuccess) return cuda_failed(e);
    LAMQ_CHECK_LAUNCH("lamq_embedding_gradient sort");
    const uint32_t *keys = p.keys[(p.passes - 1) & 1], *pos = p.pos[(p.passes - 1) & 1];
    const int threads = std::min(kSumThreads, (p.g.packs + 31) / 32 * 32), slices = (p.g.packs + 31) / 32;
    const dim3 sums((unsigned)p.chunks, (unsigned)((p.g.packs + threads - 1) / threads));
    LAMQ_REQUIRE(sums.y <= 65535, "lamq_embedding_gradient: rows too long");
    gradient_sum_kernel<T, V><<<sums, threads, 0, s>>>(dy, dE, p, keys, pos);
    LAMQ_CHECK_LAUNCH("lamq_embedding_gradient sums");
    const int64_t joins = (p.chunks * slices + kSumThreads / 32 - 1) / (kSumThreads / 32);
    LAMQ_REQUIRE(joins <= INT_MAX, "lamq_embedding_gradient: too many tokens");
    gradient_join_kernel<T, V><<<(unsigned)joins, kSumThreads, 0, s>>>(dE, p, keys, slices);
    LAMQ_CHECK_LAUNCH("lamq_embedding_gradient join");
    return LAMQ_OK;
}

}  // namespace
}  // namespace lamq

using namespace lamq;

extern "C" int lamq_embedding_lookup(const void *table, int dtype, int64_t ldt, int64_t rows, int d, const void *ids,
                                     int ids64, int64_t n, float scale, int64_t padding, void *out, int64_t ldo,
                                     int *status, lamq_stream_t stream) {
    LAMQ_REQUIRE(n >= 0 && rows >= 0 && d >= 0 && ldt >= d && ldo >= d, "lamq_embedding_lookup: bad shape");
    LAMQ_REQUIRE(dtype == LAMQ_F32 || dtype == LAMQ_BF16,
                 "lamq_embedding_lookup: dtype must be LAMQ_F32 or LAMQ_BF16");
    if (n == 0 || d == 0) return LAMQ_OK;
    LAMQ_REQUIRE(ids && out && status && (table || rows == 0), "lamq_embedding_lookup: null pointer");
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == LAMQ_F32)
        return packs_ok(table, ldt, d, 4, 4) && packs_ok(out, ldo, d, 4, 4)
                   ? run_lookup<float, 4>(table, ldt, rows, d, ids, ids64, n, scale, padding, out, ldo, status, s)
                   : run_lookup<float, 1>(table, ldt, rows, d, ids, ids64, n, scale, padding, out, ldo, status, s);
    using B = __nv_bfloat16;
    return packs_ok(table, ldt, d, 8, 2) && packs_ok(out, ldo, d, 8, 2)
               ? run_lookup<B, 8>(table, ldt, rows, d, ids, ids64, n, scale, padding, out, ldo, status, s)
               : run_lookup<B, 1>(table, ldt, rows, d, ids, ids64, n, scale, padding, out, ldo, status, s);
}

extern "C" size_t lamq_embedding_gradient_workspace_size(int64_t n, int d) {
    if (n <= kDirectTokens || d <= 0 || n > INT_MAX) return 0;
    return layout_of(n, d).total;
}

extern "C" int lamq_embedding_gradient(const void *dy, int dtype, int64_t ldy, const void *ids, int ids64, int64_t n,
                                       int64_t rows, int d, float scale, int64_t padding, int accumulate, void *dE,
                                       int64_t lde, void *workspace, size_t workspace_bytes, int *status,
                                       lamq_stream_t stream) {
    LAMQ_REQUIRE(n >= 0 && rows >= 0 && d >= 0 && ldy >= d && lde >= d, "lamq_embedding_gradient: bad shape");
    LAMQ_REQUIRE(dtype == LAMQ_F32 || dtype == LAMQ_BF16,
                 "lamq_embedding_gradient: dtype must be LAMQ_F32 or LAMQ_BF16");
    LAMQ_REQUIRE(n <= INT_MAX && rows < INT_MAX, "lamq_embedding_gradient: more than 2^31 tokens or rows");
    if (rows == 0 || d == 0) return LAMQ_OK;
    LAMQ_REQUIRE(dE && status && (n == 0 || (dy && ids)), "lamq_embedding_gradient: null pointer");
    const size_t need = lamq_embedding_gradient_workspace_size(n, d);
    LAMQ_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
                 "lamq_embedding_gradient: workspace of %zu bytes (16-byte aligned) needed, %zu given", need,
                 workspace_bytes);
    cudaStream_t s = (cudaStream_t)stream;
    GradParams g{ids, ids64, n, rows, padding, ldy, lde, 0, scale, accumulate, status};
    using B = __nv_bfloat16;
    if (dtype == LAMQ_F32)
        return packs_ok(dy, ldy, d, 4, 4) && packs_ok(dE, lde, d, 4, 4) ? run_gradient<float, 4>(dy, dE, g, d, workspace, s)
                                                                        : run_gradient<float, 1>(dy, dE, g, d, workspace, s);
    return packs_ok(dy, ldy, d, 8, 2) && packs_ok(dE, lde, d, 8, 2) ? run_gradient<B, 8>(dy, dE, g, d, workspace, s)
                                                                    : run_gradient<B, 1>(dy, dE, g, d, workspace, s);
}
