// A kernel that follows another one of the same call: launched while that still runs, it gets on its way (its launch, its
// block's start) and then waits for the other's end and memory.
#pragma once

#include "lamq_common.cuh"

namespace lamq {
namespace {

// In the first kernel: the second one may be launched once every block has come here.
__device__ __forceinline__ void let_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// In the second: what the first one wrote can be read from here on.
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_following(void (*kernel)(P...), unsigned grid, unsigned block, cudaStream_t stream, A &&...args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid), config.blockDim = dim3(block), config.stream = stream;
    cudaLaunchAttribute follows;
    follows.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    follows.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &follows, config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

}  // namespace
}  // namespace lamq
