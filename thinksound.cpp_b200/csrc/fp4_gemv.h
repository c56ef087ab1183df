// fp4_gemv.h — arguments of the 4-bit GEMV kernels and its tensor-core form (internal to libtsd_b200).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "fp4.cuh"

namespace tsd {

struct Fp4GemvArgs {
    const uint8_t * W, * Ws;
    const float * W_amax, * x, * bias;
    void * y;
    long long ldx, ldy;
    int M, K, N, silu, bf16, x_vec, units;
};

// A row of W (its codes, its first scale) times a vector in f64, by a whole warp: every lane gets the sum. Not inlined, so that
// the kernels' registers go to their loops.
template <int FMT> __device__ __noinline__ double warp_dot(const uint8_t * codes, const uint8_t * scales, const float * x, int K, int lane) {
    double s = 0.0;
    for (int k = 8 * lane; k < K; k += 256) {
        const int blk = k / fp4_block(FMT);
        const double f = fp4_scale_value<FMT>(scales[(long long)(blk >> 2) * kScaleTile + (blk & 3)]);
        float c[8];
        fp4_values8(__ldg(reinterpret_cast<const uint32_t *>(codes + k / 2)), c);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fma(c[i] * f, (double)__ldg(x + k + i), s);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}
// put(row m times vector n again in f64, times dec) in the lanes of `lost` (the whole warp calls): sums that are not finite.
// The kernels apply scales and factors after they have summed, so that f32's range can end on the way to a result that
// lies in it.
template <int FMT, typename F>
__device__ __forceinline__ void sum_again(const Fp4GemvArgs & a, unsigned lost, int m, int n, double dec, int lane, F && put) {
    for (; lost; lost &= lost - 1) {
        const int src = __ffs(lost) - 1, row = __shfl_sync(0xffffffffu, m, src), vec = __shfl_sync(0xffffffffu, n, src);
        const double s = warp_dot<FMT>(a.W + (long long)row * (a.K / 2), a.Ws + fp4_scale_at(row, 0, fp4_ktiles(a.K, FMT)),
                                       a.x + vec * a.ldx, a.K, lane);
        if (lane == src) put((float)(s * dec));
    }
}

// fp4_gemv_tc.cu: how many of N vectors of K elements fit at a time (0: not one), and the call.
int fp4_gemv_tc_group(int fmt, int N, int K);
cudaError_t fp4_gemv_tc(int fmt, const Fp4GemvArgs & a, int group, int dev, int sms, cudaStream_t st);

}  // namespace tsd
