// The global norm of many gradients, and their clipping:
//
//   norm = sqrt(Σ over the tensors Σ x²),   out = x · min(1, max_norm / (norm + eps))
//
// Bound by memory: the norm reads everything once, a step that clips reads it again and writes it. The tensors of the list
// lie end to end in one sequence of tiles that the blocks share evenly, so a few large and many small ones cost one launch;
// the list itself travels in the kernel's parameters (no copy to the device, and a CUDA graph keeps it).
//
// The sum: eight squares in fp32 at a time, added in fp64; where their fp32 sum overflows or is so small that squares may
// have been lost, those eight are squared in fp64. Every block leaves one partial sum, and whoever needs the norm adds the
// partials in the same order: equal calls give equal bits.
//
// Measured (us; bytes at 6551 GB/s in brackets): the norm of 372 M fp32 in 36 tensors 214 (227: reads alone are faster than the
// copy that the rate is of), of 67 M bf16 in 19 tensors 23 and 3 for the partials (20); 372 M fp32 clipped into other tensors 707
// (455; 682 with the second read).
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <new>
#include <vector>

#include <cuda_bf16.h>

#include "../../include/lamq_b200_step.h"
#include "dependent.cuh"

namespace lamq {
namespace {

constexpr int kThreads = 256;
constexpr int kTileBytes = 32768;  // of a tile's input: eight 16-byte loads a thread
constexpr int kLoads = kTileBytes / 16 / kThreads;
constexpr int kSMs = 148;
constexpr int kMaxBlocks = 4 * kSMs;

// The tensors of one launch. `start`: the first tile of each (and of what follows the last).
template <int kCount>
struct List {
    const void *data[kCount];
    void *out[kCount];
    int64_t n[kCount];
    uint32_t start[kCount + 1];
    uint8_t types[kCount];  // bit 0: bf16, bit 1: out is bf16, bit 2: both begin on 16 bytes
    int count;
};
constexpr int kMaxCount = 1000;  // 29 KB of the 32 KB that a kernel's parameters may take
constexpr int64_t kMaxElements = (int64_t)1 << 43;  // of a list: its tiles have 32-bit numbers

enum { kInBf16 = 1, kOutBf16 = 2, kAligned = 4 };

// ---- the sum of squares

// Where fp32 may not do. A call of its own: the path is rare, and eight times the code of the other.
__device__ __noinline__ double squares_f64(float4 a, float4 b) {
    double s = (double)a.x * a.x;
    s = fma((double)a.y, (double)a.y, s);
    s = fma((double)a.z, (double)a.z, s);
    s = fma((double)a.w, (double)a.w, s);
    s = fma((double)b.x, (double)b.x, s);
    s = fma((double)b.y, (double)b.y, s);
    s = fma((double)b.z, (double)b.z, s);
    return fma((double)b.w, (double)b.w, s);
}

// The sum of eight squares. Between the bounds no square was lost that could matter: one that is subnormal or zero in fp32
// is 2^-46 of the sum or less.
__device__ __forceinline__ double squares(const float (&x)[8]) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) a = fmaf(x[i], x[i], a), b = fmaf(x[i + 4], x[i + 4], b);
    a += b;
    if (a >= 0x1p-80f && a <= 0x1p126f) return (double)a;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));
    if (most == 0.f && a == 0.f) return 0.0;  // the zeros of a table's gradient (a: NaN where an element is)
    return squares_f64(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
}

__device__ __forceinline__ void unpack(const uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ float element(const void *data, bool bf16, int64_t i) {
    uint16_t half;
    float x;
    if (bf16) {  // volatile: neither load is run for the other type
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(half) : "l"(reinterpret_cast<const uint16_t *>(data) + i));
        return __uint_as_float((uint32_t)half << 16);
    }
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(x) : "l"(reinterpret_cast<const float *>(data) + i));
    return x;
}

// Elements [from, to) of a tensor, at most a tile.
__device__ double tile_squares(const void *data, bool bf16, bool aligned, int64_t from, int64_t to) {
    double s = 0.0;
    const int per = bf16 ? 8 : 4;
    int64_t rest = from;
    if (aligned) {
        const int64_t packs = (to - from) / per;
        const uint4 *const src = reinterpret_cast<const uint4 *>(data) + from / per;
        uint4 v[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int64_t at = threadIdx.x + i * kThreads;
            v[i] = at < packs ? __ldcg(src + at) : make_uint4(0, 0, 0, 0);
        }
        if (bf16) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                float f[8];
                unpack(v[i], f);
                s += squares(f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; i += 2) {
                const float f[8] = {__uint_as_float(v[i].x), __uint_as_float(v[i].y), __uint_as_float(v[i].z),
                                    __uint_as_float(v[i].w), __uint_as_float(v[i + 1].x), __uint_as_float(v[i + 1].y),
                                    __uint_as_float(v[i + 1].z), __uint_as_float(v[i + 1].w)};
                s += squares(f);
            }
        }
        rest += packs * per;
    }
    for (int64_t i = rest + threadIdx.x; i < to; i += kThreads) {
        const double x = element(data, bf16, i);
        s = fma(x, x, s);
    }
    return s;
}

// Sums over the block in a fixed order; the result in every thread.
__device__ double block_sum(double s) {
    __shared__ double part[kThreads / 32];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    s = part[0];
    for (int w = 1; w < kThreads / 32; ++w) s += part[w];
    return s;
}

// The tensor that holds a tile.
template <int kCount>
__device__ __forceinline__ int tensor_of(const List<kCount> &list, uint32_t tile) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (list.start[mid] <= tile) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ uint32_t first_tile(uint32_t tiles, uint32_t block) {
    return (uint32_t)((uint64_t)tiles * block / gridDim.x);
}

template <int kCount>
__global__ void __launch_bounds__(kThreads) gradient_squares_kernel(const __grid_constant__ List<kCount> list, double *part) {
    const uint32_t tiles = list.start[list.count];
    uint32_t tile = first_tile(tiles, blockIdx.x);
    const uint32_t end = first_tile(tiles, blockIdx.x + 1);
    double s = 0.0;
    if (tile < end)
        for (int k = tensor_of(list, tile); tile < end; ++k) {
            const bool bf16 = list.types[k] & kInBf16;
            const int64_t size = kTileBytes / (bf16 ? 2 : 4);
            const uint32_t stop = min(end, list.start[k + 1]);
            for (; tile < stop; ++tile) {
                const int64_t from = (int64_t)(tile - list.start[k]) * size;
                s += tile_squares(list.data[k], bf16, list.types[k] & kAligned, from, min(list.n[k], from + size));
            }
        }
    // Not before: blocks of the clipping kernel that found room beside these would crowd on the SMs that had some (372 M fp32
    // clipped: 1039 us instead of 700).
    let_follow();
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from all partial sums, in every thread.
__device__ double norm_of(const double *part, int parts) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += __ldcg(part + i);
    return sqrt(block_sum(s));
}

__global__ void __launch_bounds__(kThreads) gradient_norm_kernel(const double *part, int parts, float *norm) {
    await_previous();
    const double x = norm_of(part, parts);
    if (threadIdx.x == 0) *norm = (float)x;
}

// ---- clipping

// x · factor in fp32, or in fp64 where the factor is outside fp32's normal range.
struct Scale {
    double exact;
    float f;
    bool wide;
    __device__ float operator()(float x) const { return wide ? (float)(x * exact) : x * f; }
};

__device__ __forceinline__ void store8(void *out, bool bf16, int64_t pack, const float (&f)[8]) {
    if (bf16) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        reinterpret_cast<uint4 *>(out)[pack] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        reinterpret_cast<float4 *>(out)[2 * pack] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4 *>(out)[2 * pack + 1] = make_float4(f[4], f[5], f[6], f[7]);
    }
}

__device__ void tile_scale(const void *data, void *out, int types, int64_t from, int64_t to, const Scale &scale) {
    const bool in16 = types & kInBf16, out16 = types & kOutBf16;
    int64_t rest = from;
    if (types & kAligned) {
        const int64_t packs = (to - from) / 8, first = from / 8;
        for (int64_t i = threadIdx.x; i < packs; i += kThreads) {
            float f[8];
            if (in16) {
                unpack(reinterpret_cast<const uint4 *>(data)[first + i], f);
            } else {
                const float4 a = reinterpret_cast<const float4 *>(data)[2 * (first + i)];
                const float4 b = reinterpret_cast<const float4 *>(data)[2 * (first + i) + 1];
                f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = scale(f[e]);
            store8(out, out16, first + i, f);
        }
        rest += packs * 8;
    }
    for (int64_t i = rest + threadIdx.x; i < to; i += kThreads) {
        const float x = scale(element(data, in16, i));
        if (out16)
            reinterpret_cast<__nv_bfloat16 *>(out)[i] = __float2bfloat16_rn(x);
        else
            reinterpret_cast<float *>(out)[i] = x;
    }
}

// Tiles are taken from the last to the first: what the sum of squares read last may still be in L2.
template <int kCount>
__global__ void __launch_bounds__(kThreads)
    gradient_clip_kernel(const __grid_constant__ List<kCount> list, const double *part, int parts, double max_norm, double eps,
                         float *norm) {
    await_previous();
    const double x = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm) *norm = (float)x;
    const double factor = max_norm / (x + eps);
    const bool clips = !(factor >= 1.0);  // a NaN clips
    Scale scale;
    scale.exact = clips ? factor : 1.0;
    scale.f = (float)scale.exact;
    scale.wide = scale.f < 0x1p-126f;  // zero included
    const uint32_t tiles = list.start[list.count];
    const uint32_t begin = first_tile(tiles, blockIdx.x);
    uint32_t tile = first_tile(tiles, blockIdx.x + 1);
    if (tile <= begin) return;
    for (int k = tensor_of(list, tile - 1); tile > begin; --k) {
        const bool bf16 = list.types[k] & kInBf16;
        const int64_t size = kTileBytes / (bf16 ? 2 : 4);
        const uint32_t stop = max(begin, list.start[k]);
        if (!clips && list.out[k] == list.data[k]) {
            tile = stop;
            continue;
        }
        while (tile > stop) {
            --tile;
            const int64_t from = (int64_t)(tile - list.start[k]) * size;
            tile_scale(list.data[k], list.out[k], list.types[k], from, min(list.n[k], from + size), scale);
        }
    }
}

// ---- the host's side

static_assert(sizeof(lamq_gradient) == 32 && offsetof(lamq_gradient, n) == 16 && offsetof(lamq_gradient, out_dtype) == 28,
              "the bindings pack 32 bytes an entry");

int64_t tiles_of(const lamq_gradient &g) {
    const int64_t size = kTileBytes / (g.dtype == LAMQ_BF16 ? 2 : 4);
    return (g.n + size - 1) / size;
}

int blocks_for(int64_t tiles) { return (int)std::min<int64_t>(std::max<int64_t>(tiles, 1), kMaxBlocks); }

// Whether a written range of memory meets another range of the list.
struct Range {
    uintptr_t begin, end;
    bool written;
};

bool overlap(std::vector<Range> &ranges) {
    std::sort(ranges.begin(), ranges.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;  // where the ranges so far end
    for (const Range &r : ranges) {
        if (r.begin < (r.written ? any : written)) return true;
        any = std::max(any, r.end);
        if (r.written) written = std::max(written, r.end);
    }
    return false;
}

int check_list(const lamq_gradient *list, int64_t count, bool clip) {
    LAMQ_REQUIRE(count >= 0 && count <= INT_MAX, "bad shape: %lld tensors", (long long)count);
    LAMQ_REQUIRE(list || count == 0, "null pointer (list)");
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) {
        const lamq_gradient &g = list[i];
        LAMQ_REQUIRE(g.n >= 0 && g.n <= kMaxElements, "bad shape: a tensor of %lld elements", (long long)g.n);
        LAMQ_REQUIRE((total += g.n) <= kMaxElements, "more than 2^43 elements");
        LAMQ_REQUIRE((g.dtype == LAMQ_F32 || g.dtype == LAMQ_BF16) &&
                         (!clip || g.out_dtype == LAMQ_F32 || g.out_dtype == LAMQ_BF16),
                     "dtype: LAMQ_F32 or LAMQ_BF16");
        LAMQ_REQUIRE(g.n == 0 || (g.data && (!clip || g.out)), "null pointer (tensor %lld)", (long long)i);
        LAMQ_REQUIRE(g.n == 0 || (aligned_to(g.data, g.dtype == LAMQ_BF16 ? 2 : 4) &&
                                  (!clip || aligned_to(g.out, g.out_dtype == LAMQ_BF16 ? 2 : 4))),
                     "tensor %lld: not aligned to its elements", (long long)i);
        LAMQ_REQUIRE(!clip || g.n == 0 || g.out != g.data || g.out_dtype == g.dtype, "dtype: in place it stays");
    }
    if (!clip) return LAMQ_OK;
    try {
        std::vector<Range> ranges;
        ranges.reserve(2 * (size_t)count);
        for (int64_t i = 0; i < count; ++i) {
            const lamq_gradient &g = list[i];
            if (g.n == 0) continue;
            const uintptr_t in = reinterpret_cast<uintptr_t>(g.data), out = reinterpret_cast<uintptr_t>(g.out);
            if (in != out) ranges.push_back({in, in + (uintptr_t)g.n * (g.dtype == LAMQ_BF16 ? 2 : 4), false});
            ranges.push_back({out, out + (uintptr_t)g.n * (g.out_dtype == LAMQ_BF16 ? 2 : 4), true});
        }
        LAMQ_REQUIRE(!overlap(ranges), "tensors of the list overlap where they are written");
    } catch (const std::bad_alloc &) {
        LAMQ_REQUIRE(false, "no host memory for a list of %lld tensors", (long long)count);
    }
    return LAMQ_OK;
}

// f(first, count, tiles) for each launch that a list takes.
template <typename F>
int each_launch(const lamq_gradient *list, int64_t count, F f) {
    for (int64_t i = 0; i < count; i += kMaxCount) {
        const int64_t n = std::min<int64_t>(kMaxCount, count - i);
        int64_t tiles = 0;
        for (int64_t k = i; k < i + n; ++k) tiles += tiles_of(list[k]);
        if (const int st = f(i, n, tiles)) return st;
    }
    return LAMQ_OK;
}

template <int kCount>
void fill(List<kCount> &l, const lamq_gradient *list, int64_t count, bool clip) {
    uint32_t tile = 0;
    l.count = 0;
    for (int64_t i = 0; i < count; ++i) {
        const lamq_gradient &g = list[i];
        if (g.n == 0) continue;
        const int k = l.count++;
        l.data[k] = g.data, l.out[k] = clip ? g.out : nullptr, l.n[k] = g.n, l.start[k] = tile;
        const uintptr_t where = reinterpret_cast<uintptr_t>(g.data) | (clip ? reinterpret_cast<uintptr_t>(g.out) : 0);
        l.types[k] = (g.dtype == LAMQ_BF16 ? kInBf16 : 0) | (clip && g.out_dtype == LAMQ_BF16 ? kOutBf16 : 0) |
                     ((where & 15) == 0 ? kAligned : 0);
        tile += (uint32_t)tiles_of(g);
    }
    l.start[l.count] = tile;
}

template <int kCount>
int launch_squares(const lamq_gradient *list, int64_t count, int64_t tiles, double *part, cudaStream_t stream) {
    List<kCount> l;
    fill(l, list, count, false);
    gradient_squares_kernel<kCount><<<blocks_for(tiles), kThreads, 0, stream>>>(l, part);
    LAMQ_CHECK_LAUNCH("lamq_gradient (sum of squares)");
    return LAMQ_OK;
}

template <int kCount>
int launch_clip(const lamq_gradient *list, int64_t count, int64_t tiles, const double *part, int parts, double max_norm,
                double eps, float *norm, cudaStream_t stream) {
    List<kCount> l;
    fill(l, list, count, true);
    launch_following(gradient_clip_kernel<kCount>, blocks_for(tiles), kThreads, stream, l, part, parts, max_norm, eps, norm);
    LAMQ_CHECK_LAUNCH("lamq_gradient_clip");
    return LAMQ_OK;
}

// Partial sums of all launches, one behind the other.
int all_squares(const lamq_gradient *list, int64_t count, double *part, int &parts, cudaStream_t stream) {
    parts = 0;
    return each_launch(list, count, [&](int64_t i, int64_t n, int64_t tiles) {
        double *const to = part + parts;
        parts += blocks_for(tiles);
        return n <= 32 ? launch_squares<32>(list + i, n, tiles, to, stream)
               : n <= 256 ? launch_squares<256>(list + i, n, tiles, to, stream)
                          : launch_squares<kMaxCount>(list + i, n, tiles, to, stream);
    });
}

int check_call(const lamq_gradient *list, int64_t count, bool clip, const float *norm, const void *workspace, size_t bytes) {
    if (const int st = check_list(list, count, clip)) return st;
    LAMQ_REQUIRE(norm, "null pointer (norm)");
    LAMQ_REQUIRE(aligned_to(norm, sizeof(float)), "norm: not aligned to its elements");
    const size_t need = lamq_gradient_workspace_size(count);
    LAMQ_REQUIRE(bytes >= need, "a workspace of %zu bytes is needed", need);
    LAMQ_REQUIRE(need == 0 || workspace, "null pointer (workspace)");
    LAMQ_REQUIRE(aligned_to(workspace, sizeof(double)), "the workspace must be 8-byte aligned");
    return LAMQ_OK;
}

}  // namespace
}  // namespace lamq

using namespace lamq;

extern "C" size_t lamq_gradient_workspace_size(int64_t count) {
    return count < 0 ? 0 : (size_t)((count + kMaxCount - 1) / kMaxCount) * kMaxBlocks * sizeof(double);
}

extern "C" int lamq_gradient_norm(const lamq_gradient *list, int64_t count, float *norm, void *workspace,
                                  size_t workspace_bytes, lamq_stream_t stream) {
    if (const int st = check_call(list, count, false, norm, workspace, workspace_bytes)) return st;
    double *const part = reinterpret_cast<double *>(workspace);
    int parts = 0;
    if (const int st = all_squares(list, count, part, parts, (cudaStream_t)stream)) return st;
    launch_following(gradient_norm_kernel, 1, kThreads, (cudaStream_t)stream, part, parts, norm);
    LAMQ_CHECK_LAUNCH("lamq_gradient_norm");
    return LAMQ_OK;
}

extern "C" int lamq_gradient_clip(const lamq_gradient *list, int64_t count, double max_norm, double eps, float *norm,
                                  void *workspace, size_t workspace_bytes, lamq_stream_t stream) {
    LAMQ_REQUIRE(max_norm >= 0.0, "max_norm must not be negative");
    LAMQ_REQUIRE(std::isfinite(eps) && eps >= 0.0, "eps must not be negative");
    if (const int st = check_call(list, count, true, norm, workspace, workspace_bytes)) return st;
    double *const part = reinterpret_cast<double *>(workspace);
    int parts = 0;
    if (const int st = all_squares(list, count, part, parts, (cudaStream_t)stream)) return st;
    if (count == 0) {
        gradient_norm_kernel<<<1, kThreads, 0, (cudaStream_t)stream>>>(part, 0, norm);
        LAMQ_CHECK_LAUNCH("lamq_gradient_clip");
        return LAMQ_OK;
    }
    return each_launch(list, count, [&](int64_t i, int64_t n, int64_t tiles) {
        float *const to = i == 0 ? norm : nullptr;  // one launch writes the norm
        const lamq_gradient *const of = list + i;
        const cudaStream_t st = (cudaStream_t)stream;
        return n <= 32    ? launch_clip<32>(of, n, tiles, part, parts, max_norm, eps, to, st)
               : n <= 256 ? launch_clip<256>(of, n, tiles, part, parts, max_norm, eps, to, st)
                          : launch_clip<kMaxCount>(of, n, tiles, part, parts, max_norm, eps, to, st);
    });
}
