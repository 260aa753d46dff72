// What the roles of a product on tcgen05 know of one another's waits.  Every wait is bounded; one that gives up tells all of them, and the
// launch's error flag, and each runs to its end.
#pragma once

#include "tma.cuh"

#include <cooperative_groups.h>

namespace linear8 {

struct Waits {
    int* gave_up;  // in shared memory
    int ctas;      // of the cluster, all of which are told; 0: this one alone
    int* error_flag;
    __device__ __forceinline__ bool flag() const { return *(volatile int*)gave_up != 0; }
    __device__ __forceinline__ void fail() const {
        *(volatile int*)gave_up = 1;
        for (int r = 0; r < ctas; ++r) *(volatile int*)cooperative_groups::this_cluster().map_shared_rank(gave_up, r) = 1;
        if (error_flag) atomicExch(error_flag, 1);
    }
    // For whole warps, with one answer for all lanes, whichever of them saw the flag or whose wait ran out: what follows (an election, a load of
    // tensor memory, the next vote) is for whole warps too.
    __device__ __forceinline__ bool failed() const { return __any_sync(0xffffffffu, flag()); }
    __device__ __forceinline__ bool there(unsigned long long* bar, unsigned parity) const {
        if (__all_sync(0xffffffffu, tma::mbar_wait(bar, parity))) return true;
        fail();
        return false;
    }
    // ... which does not wait once it has been told.  (The issuers need not be: what they wait for no longer comes once another role has left.)
    __device__ __forceinline__ bool there_untold(unsigned long long* bar, unsigned parity) const {
        if (__all_sync(0xffffffffu, !flag() && tma::mbar_wait(bar, parity))) return true;
        fail();
        return false;
    }
};

}  // namespace linear8
