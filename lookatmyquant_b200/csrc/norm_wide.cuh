// Rows of more elements than the teams' registers hold, where they may begin anywhere, the full join's backward of more than
// 8192, and what finds no room for its stages (norm_layout): a block for each row, its threads taking every 1024th element. What a later pass needs of a row stays in shared memory as
// fp32; each thread reads there what it wrote itself. Sums over rows are added up in the block's partial row, each column by the
// thread that owns it. Bound by the latency of the passes over a row (three in the join's forward, three in its backward).
#pragma once

#include "norm.cuh"

namespace lamq {
namespace {

constexpr int kWideThreads = 1024;

__device__ __forceinline__ float value_at(const void *p, int dtype, int64_t i) {
    float f[1];
    load_typed<1>(p, dtype, i, f);
    return f[0];
}

// What this thread has written itself (not through the read-only path; volatile for the reason that all loads are).
__device__ __forceinline__ float own_at(const float *p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}

// The sums over the block, in every thread, in a fixed order. scratch: K x 32 floats.
template <int K>
__device__ __forceinline__ void wide_sum(float (&v)[K], float *scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    __syncthreads();  // the last sums have been read
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) scratch[k * 32 + warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = scratch[k * 32 + lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
}

// f(j) for this thread's elements of a row, four of them on their way at a time.
template <typename F>
__device__ __forceinline__ void wide_each(int d, F f) {
#pragma unroll 4
    for (int j = threadIdx.x; j < d; j += kWideThreads) f(j);
}

// The factor of a row whose sum of squares is ss, x(j) its elements; where the sum overflowed, that of x(j) · shrunk.
template <typename F>
__device__ __forceinline__ float wide_factor(float ss, int d, F x, float inv_d, float eps, float &shrunk, float *scratch) {
    shrunk = 1.f;
    if (isinf(ss)) {
        shrunk = kShrink;
        eps = 0.f;
        float s[1] = {0.f};
        wide_each(d, [&](int j) {
            const float y = x(j) * kShrink;
            s[0] = fmaf(y, y, s[0]);
        });
        wide_sum(s, scratch);
        ss = s[0];
    }
    return reciprocal_root(fmaf(ss, inv_d, eps));
}

}  // namespace
}  // namespace lamq
