// fp4_tc.cuh — what the tensor-core kernels on 4-bit operands share.
#pragma once
#include "common.cuh"

namespace tsd {

constexpr int kAtomK = 256;                // elements of K in a 128-byte row of codes

// A bounded wait by a whole warp, with one answer for all of it. Voting on every try keeps the warp
// together: no lane runs ahead and nothing has to be joined afterwards.
__device__ __forceinline__ bool warp_wait(uint64_t * bar, uint32_t parity, volatile int * abort, int * err, int code) {
#pragma unroll 1
    for (int it = 0; it < 32; ++it)
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, err, code));
}

}  // namespace tsd
