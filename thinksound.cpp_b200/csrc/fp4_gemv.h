// fp4_gemv.h — arguments of the 4-bit GEMV kernels and its tensor-core form (internal to libtsd_b200).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace tsd {

struct Fp4GemvArgs {
    const uint8_t * W, * Ws;
    const float * W_amax, * x, * bias;
    void * y;
    long long ldx, ldy;
    int M, K, N, silu, bf16, x_vec, units;
};

// fp4_gemv_tc.cu: how many of N vectors of K elements fit at a time (0: not one), and the call.
int fp4_gemv_tc_group(int fmt, int N, int K);
cudaError_t fp4_gemv_tc(int fmt, const Fp4GemvArgs & a, int group, int dev, int sms, cudaStream_t st);

}  // namespace tsd
