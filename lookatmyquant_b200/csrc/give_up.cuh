// Bounded waits whose failure is the launch's own: a status word that still holds the error of an earlier call, or gets one
// from a call on another stream, ends nothing here.
#pragma once

#include "lamq_common.cuh"
#include "sm100.cuh"

// The limit of a wait, and after how many polls it is looked at. (A poll suspends the thread for a while by itself.)
#ifndef LAMQ_GIVE_UP_NS
#define LAMQ_GIVE_UP_NS sm100::kWaitTimeoutNs
#endif
#ifndef LAMQ_GIVE_UP_POLLS
#define LAMQ_GIVE_UP_POLLS 256u
#endif

namespace lamq {
namespace {

__device__ unsigned long long g_gave_up;  // the last launch of this file's kernels in which a wait gave up (0: none)

__device__ __forceinline__ unsigned long long this_launch() {
    unsigned long long id;
    asm volatile("mov.u64 %0, %%gridid;" : "=l"(id));  // volatile: read where it is wanted, not kept in registers (3 % of
                                                       // the attention forward's time, through spills)
    return id + 1;
}

// Another wait of this launch has given up.
__device__ __forceinline__ bool launch_gave_up() {
    return *reinterpret_cast<volatile unsigned long long *>(&g_gave_up) == this_launch();
}

__device__ __forceinline__ void give_up(int *status) {
    atomicExch(&g_gave_up, this_launch());
    atomicMax(status, LAMQ_ERR_TIMEOUT);
}

// Waits for the mbarrier's phase with the given parity. False, and LAMQ_ERR_TIMEOUT in *status, if it does not complete
// within the limit, or as soon as another wait of this launch has given up.
__device__ __forceinline__ bool await(uint32_t bar, uint32_t parity, int *status) {
    using namespace sm100;
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if (it % LAMQ_GIVE_UP_POLLS == 0u && (launch_gave_up() || globaltimer() - t0 > LAMQ_GIVE_UP_NS)) {
            give_up(status);
            return false;
        }
    }
}

}  // namespace
}  // namespace lamq
