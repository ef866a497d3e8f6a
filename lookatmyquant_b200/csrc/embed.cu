// The embedding of a training step: rows of the table looked up and scaled, and the table's gradient.
//
//   lookup     Y_t = scale · E[id_t]
//   gradient   dE_v = scale · Σ_{t: id_t = v} dY_t        (rows no token names are zero)
//
// Both are bound by memory: the lookup reads each token's row and writes it, the gradient reads dY once and writes the
// whole of dE once (rows nobody named included), so for a large table most of its bytes are zeros.
//
// The gradient's sums have a fixed order, the tokens' own: the ids are sorted by a stable radix sort (digits of up to
// 9 bits: a histogram per tile of tokens, one scan over digits and tiles, a scatter that ranks equal digits by
// position), and the sorted tokens are cut into chunks that are summed in fp32 by separate blocks. A row whose tokens
// lie in one chunk is written at once; a row that crosses chunks (a frequent token: its run may be a tenth of all
// tokens) leaves a partial per chunk, which a last kernel adds chunk by chunk. No float is added by an atomic: repeated
// calls agree bit for bit.
#include <algorithm>
#include <climits>
#include <cstdint>

#include <cuda_bf16.h>

#include "../../include/lamq_b200_train.h"
#include "lamq_common.cuh"

namespace lamq {
namespace {

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
    if (!valid && first == 0) atomicCAS(status, 0, LAMQ_ERR_INVALID);
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

// ---- the stable radix sort of (id, position)

constexpr int kMaxDigitBits = 9, kMaxBins = 1 << kMaxDigitBits;
constexpr int kTileRounds = 8, kTile = kThreads * kTileRounds;  // tokens a block ranks at a time
constexpr int kWarps = kThreads / 32;
constexpr int kScanThreads = 1024;

struct SortSource {
    const void *ids;        // the first pass: the caller's ids (a padding or invalid id sorts last, as `rows`)
    int ids64;
    int64_t rows, padding;
    const uint32_t *keys;   // later passes
    const uint32_t *pos;
    int *status;
};

__device__ __forceinline__ uint32_t key_at(const SortSource &s, int64_t t) {
    if (s.keys) return s.keys[t];
    const int64_t id = id_at(s.ids, s.ids64, t);
    return (id < 0 || id >= s.rows || id == s.padding) ? (uint32_t)s.rows : (uint32_t)id;
}

__global__ void __launch_bounds__(kThreads)
    sort_count_kernel(SortSource s, int64_t n, int shift, int bits, int tiles, uint32_t *__restrict__ counts) {
    __shared__ uint32_t hist[kMaxBins];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += kThreads) hist[b] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * kTile;
    for (int r = 0; r < kTileRounds; ++r) {
        const int64_t t = t0 + r * kThreads + threadIdx.x;
        if (t >= n) break;
        const uint32_t key = key_at(s, t);
        if (s.keys == nullptr && key == (uint32_t)s.rows) {
            const int64_t id = id_at(s.ids, s.ids64, t);
            if (id < 0 || id >= s.rows) atomicCAS(s.status, 0, LAMQ_ERR_INVALID);
        }
        atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) counts[(int64_t)b * tiles + blockIdx.x] = hist[b];
}

// Exclusive scan of `len` counts in place, one block: each thread's run of entries, then a scan of the runs' sums.
__global__ void __launch_bounds__(kScanThreads) sort_scan_kernel(uint32_t *__restrict__ counts, int64_t len) {
    __shared__ uint32_t warp_sum[kScanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t each = (len + kScanThreads - 1) / kScanThreads;
    const int64_t lo = std::min<int64_t>(len, threadIdx.x * each), hi = std::min<int64_t>(len, lo + each);
    uint32_t sum = 0;
    for (int64_t i = lo; i < hi; ++i) sum += counts[i];
    uint32_t incl = sum;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = warp_sum[lane], wi = w;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, wi, o);
            if (lane >= o) wi += v;
        }
        warp_sum[lane] = wi - w;
    }
    __syncthreads();
    uint32_t run = warp_sum[warp] + incl - sum;
    for (int64_t i = lo; i < hi; ++i) {
        const uint32_t c = counts[i];
        counts[i] = run;
        run += c;
    }
}

// Each warp ranks a contiguous piece of the tile in order, so equal digits keep their order.
__global__ void __launch_bounds__(kThreads)
    sort_scatter_kernel(SortSource s, int64_t n, int shift, int bits, int tiles, const uint32_t *__restrict__ offsets,
                        uint32_t *__restrict__ keys_out, uint32_t *__restrict__ pos_out) {
    __shared__ uint32_t seen[kWarps][kMaxBins];
    const int bins = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = lane; b < bins; b += 32) seen[warp][b] = 0;
    __syncwarp();
    const int64_t t0 = (int64_t)blockIdx.x * kTile + warp * (32 * kTileRounds);
    uint32_t key[kTileRounds], rank[kTileRounds];
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int64_t t = t0 + r * 32 + lane;
        const bool in = t < n;
        key[r] = in ? key_at(s, t) : 0u;
        const uint32_t digit = in ? (key[r] >> shift) & (bins - 1) : (uint32_t)bins;  // the tail matches nobody
        const uint32_t peers = __match_any_sync(0xffffffffu, digit);
        const uint32_t before = in ? seen[warp][digit] : 0u;
        rank[r] = before + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (in && (__ffs(peers) - 1) == lane) seen[warp][digit] = before + __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) {  // each warp's first place in each digit
        uint32_t at = offsets[(int64_t)b * tiles + blockIdx.x];
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = seen[w][b];
            seen[w][b] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int64_t t = t0 + r * 32 + lane;
        if (t >= n) break;
        const uint32_t at = seen[warp][(key[r] >> shift) & (bins - 1)] + rank[r];
        keys_out[at] = key[r];
        pos_out[at] = s.pos ? s.pos[t] : (uint32_t)t;
    }
}

// ---- the sums

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    zero_rows_kernel(T *__restrict__ out, int64_t ld, int64_t rows, int packs) {
    const int64_t total = rows * packs;
    float z[V];
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = 0.f;
    Pack<T, V> p;
    p.set(z);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads)
        p.store(out + (i / packs) * ld + (i % packs) * V);
}

struct SumParams {
    const uint32_t *keys, *pos;
    int64_t n, ldy, lde;
    int rows;        // keys from here on are padding or invalid
    int packs, chunk;
    float scale;
    int accumulate;
    float *head, *tail;  // a partial per chunk: of the row that began before it, of the row that goes on after it
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

constexpr int kAhead = 8;  // rows of dY in flight per thread

// Block (chunk, column part): the chunk's tokens in sorted order, a thread per pack of columns.
template <typename T, int V>
__global__ void __launch_bounds__(128)
    sum_chunks_kernel(const T *__restrict__ dy, T *__restrict__ dE, SumParams p) {
    const int64_t c = blockIdx.x, lo = c * p.chunk, hi = std::min<int64_t>(p.n, lo + p.chunk);
    const int col = blockIdx.y * blockDim.x + threadIdx.x;
    if (col >= p.packs) return;
    const uint32_t dead = (uint32_t)p.rows;
    const uint32_t prev = lo > 0 ? p.keys[lo - 1] : dead, next = hi < p.n ? p.keys[hi] : dead;
    float acc[V];
    bool open = false;        // acc holds tokens of row `cur`
    bool first = true;        // no row has been closed in this chunk yet
    uint32_t cur = dead;
    const auto close = [&](bool goes_on) {
        if (!open) return;
        const int64_t at = (c * p.packs + col) * V;
        if (first && cur == prev) write_partial<V>(p.head + at, acc);
        else if (goes_on) write_partial<V>(p.tail + at, acc);
        else write_row<T, V>(dE + (int64_t)cur * p.lde + (int64_t)col * V, acc, p.scale, p.accumulate);
        open = false;
        first = false;
    };
    for (int64_t base = lo; base < hi; base += kAhead) {
        Pack<T, V> x[kAhead];
        uint32_t key[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            key[i] = base + i < hi ? p.keys[base + i] : dead;
            if (key[i] < dead) x[i] = Pack<T, V>::load(dy + (int64_t)p.pos[base + i] * p.ldy + (int64_t)col * V);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
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

// Block (chunk, column part): where a row goes on past the chunk in which it began, its partials in chunk order.
template <typename T, int V>
__global__ void __launch_bounds__(128) join_chunks_kernel(T *__restrict__ dE, SumParams p) {
    const int64_t c = blockIdx.x, lo = c * p.chunk, hi = lo + p.chunk;
    if (hi >= p.n) return;
    const uint32_t key = p.keys[hi - 1];
    if (key >= (uint32_t)p.rows || p.keys[hi] != key) return;          // nothing goes on
    if (p.keys[lo] == key && lo > 0 && p.keys[lo - 1] == key) return;  // it began in an earlier chunk
    const int col = blockIdx.y * blockDim.x + threadIdx.x;
    if (col >= p.packs) return;
    float acc[V];
    const int64_t step = (int64_t)p.packs * V, at = (int64_t)col * V;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = p.tail[c * step + at + e];
    for (int64_t k = c + 1;; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += p.head[k * step + at + e];
        const int64_t end = (k + 1) * p.chunk;
        if (end >= p.n || p.keys[end] != key) break;
    }
    write_row<T, V>(dE + (int64_t)key * p.lde + at, acc, p.scale, p.accumulate);
}

// Tokens per chunk: enough chunks to fill the device for few tokens, long ones (fewer partials) for many.
int chunk_tokens(int64_t n) { return (int)std::min<int64_t>(64, std::max<int64_t>(8, n / 1024)); }

struct Layout {
    int64_t tiles, chunks;
    size_t keys, counts, partial, total;  // bytes of one buffer of each kind, and of all
};

Layout layout_of(int64_t n, int d) {
    Layout L;
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    L.tiles = (n + kTile - 1) / kTile;
    L.chunks = (n + chunk_tokens(n) - 1) / chunk_tokens(n);
    L.keys = up((size_t)n * 4);
    L.counts = up((size_t)L.tiles * kMaxBins * 4);
    L.partial = up((size_t)L.chunks * (size_t)d * 4);
    L.total = 4 * L.keys + L.counts + 2 * L.partial;
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

template <typename T, int V>
int run_sums(const void *dy, void *dE, SumParams p, int d, int64_t rows, int64_t chunks, cudaStream_t s) {
    p.packs = d / V;
    T *out = reinterpret_cast<T *>(dE);
    if (!p.accumulate) {
        const int64_t blocks = std::min<int64_t>((rows * p.packs + kThreads - 1) / kThreads, 148 * 8);
        zero_rows_kernel<T, V><<<(unsigned)blocks, kThreads, 0, s>>>(out, p.lde, rows, p.packs);
        LAMQ_CHECK_LAUNCH("lamq_embedding_gradient zero");
    }
    if (p.n == 0) return LAMQ_OK;
    const int threads = std::min(128, (p.packs + 31) / 32 * 32);
    const dim3 grid((unsigned)chunks, (unsigned)((p.packs + threads - 1) / threads));
    sum_chunks_kernel<T, V><<<grid, threads, 0, s>>>(reinterpret_cast<const T *>(dy), out, p);
    LAMQ_CHECK_LAUNCH("lamq_embedding_gradient sums");
    join_chunks_kernel<T, V><<<grid, threads, 0, s>>>(out, p);
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
    if (n <= 0 || d <= 0 || n > INT_MAX) return 0;
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
    SumParams p{};
    p.n = n;
    p.ldy = ldy;
    p.lde = lde;
    p.rows = (int)rows;
    p.scale = scale;
    p.accumulate = accumulate;
    int64_t chunks = 0;
    if (n > 0) {
        const Layout L = layout_of(n, d);
        char *ws = reinterpret_cast<char *>(workspace);
        uint32_t *keys[2], *pos[2];
        for (int i = 0; i < 2; ++i) {
            keys[i] = reinterpret_cast<uint32_t *>(ws + (2 * i) * L.keys);
            pos[i] = reinterpret_cast<uint32_t *>(ws + (2 * i + 1) * L.keys);
        }
        uint32_t *counts = reinterpret_cast<uint32_t *>(ws + 4 * L.keys);
        p.head = reinterpret_cast<float *>(ws + 4 * L.keys + L.counts);
        p.tail = reinterpret_cast<float *>(ws + 4 * L.keys + L.counts + L.partial);
        p.chunk = chunk_tokens(n);
        chunks = L.chunks;
        int key_bits = 1;
        while ((rows >> key_bits) != 0) ++key_bits;  // keys are 0 .. rows
        const int passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits, bits = (key_bits + passes - 1) / passes;
        SortSource src{ids, ids64, rows, padding, nullptr, nullptr, status};
        for (int pass = 0; pass < passes; ++pass) {
            const int shift = pass * bits;
            sort_count_kernel<<<(unsigned)L.tiles, kThreads, 0, s>>>(src, n, shift, bits, (int)L.tiles, counts);
            LAMQ_CHECK_LAUNCH("lamq_embedding_gradient count");
            sort_scan_kernel<<<1, kScanThreads, 0, s>>>(counts, L.tiles << bits);
            LAMQ_CHECK_LAUNCH("lamq_embedding_gradient scan");
            uint32_t *ko = keys[pass & 1], *po = pos[pass & 1];
            sort_scatter_kernel<<<(unsigned)L.tiles, kThreads, 0, s>>>(src, n, shift, bits, (int)L.tiles, counts, ko,
                                                                       po);
            LAMQ_CHECK_LAUNCH("lamq_embedding_gradient scatter");
            src.keys = ko;
            src.pos = po;
        }
        p.keys = src.keys;
        p.pos = src.pos;
    }
    using B = __nv_bfloat16;
    if (dtype == LAMQ_F32)
        return packs_ok(dy, ldy, d, 4, 4) && packs_ok(dE, lde, d, 4, 4) ? run_sums<float, 4>(dy, dE, p, d, rows, chunks, s)
                                                                        : run_sums<float, 1>(dy, dE, p, d, rows, chunks, s);
    return packs_ok(dy, ldy, d, 8, 2) && packs_ok(dE, lde, d, 8, 2) ? run_sums<B, 8>(dy, dE, p, d, rows, chunks, s)
                                                                    : run_sums<B, 1>(dy, dE, p, d, rows, chunks, s);
}
