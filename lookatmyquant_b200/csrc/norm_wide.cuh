// Rows of more elements than the teams' registers hold, where they may begin anywhere: a block for each row, its threads
// taking every 512th element and reading them again (from L1 and L2) wherever they are needed. Sums over rows are added up in
// the block's partial row itself, each column by the thread that owns it.
#pragma once

#include "norm.cuh"

namespace lamq {
namespace {

constexpr int kWideThreads = kNormThreads;

__device__ __forceinline__ float value_at(const void *p, int dtype, int64_t i) {
    float f[1];
    load_typed<1>(p, dtype, i, f);
    return f[0];
}

// The sum of f(j) over the row, in every thread.
template <typename F>
__device__ __forceinline__ float wide_sum(Team &team, int d, F f) {
    float s[1] = {0.f};
    for (int j = threadIdx.x; j < d; j += kWideThreads) s[0] += f(j);
    team.sum(s);
    return s[0];
}

// As unit_factor, of the row x(j); here x stays, and the factor is that of x(j) · shrunk.
template <typename F>
__device__ __forceinline__ float wide_factor(Team &team, int d, F x, float inv_d, float eps, float &shrunk) {
    shrunk = 1.f;
    float ss = wide_sum(team, d, [&](int j) { return x(j) * x(j); });
    if (isinf(ss)) {
        shrunk = kShrink;
        eps = 0.f;
        ss = wide_sum(team, d, [&](int j) { return x(j) * kShrink * (x(j) * kShrink); });
    }
    return reciprocal_root(fmaf(ss, inv_d, eps));
}

}  // namespace
}  // namespace lamq
