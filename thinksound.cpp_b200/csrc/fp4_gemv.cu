// fp4_gemv.cu — microscaled 4-bit weights times a few f32 vectors (sm_100a); format: include/tsd_ops.h.
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "op_check.h"

#include <cstdio>

namespace tsd {

namespace {

constexpr int kMaxN = 8;

struct Fp4GemvArgs {
    const uint8_t * W, * Ws;
    const float * W_amax, * x, * bias;
    void * y;
    long long ldx, ldy;
    int M, K, N, silu, bf16;
};

// One warp per weight row; a lane takes eight codes at a time.
template <int FMT>
__global__ void __launch_bounds__(256) fp4_gemv_kernel(const Fp4GemvArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int m = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (m >= a.M) return;
    const int kt = fp4_ktiles(a.K, FMT);
    const uint32_t * row = reinterpret_cast<const uint32_t *>(a.W + (long long)m * (a.K / 2));
    float acc[kMaxN] = {};
    for (int c = lane; c < a.K / 8; c += 32) {
        const int j = c * 8 / fp4_block(FMT);
        const float s = fp4_scale_value<FMT>(a.Ws[fp4_scale_at(m, j >> 2, kt) + (j & 3)]);
        float v[8];
        fp4_values8(row[c], v);
#pragma unroll
        for (int n = 0; n < kMaxN; ++n)
            if (n < a.N) {
                float t = 0.f;
                for (int e = 0; e < 8; ++e) t = fmaf(v[e], a.x[n * a.ldx + c * 8 + e], t);
                acc[n] = fmaf(t, s, acc[n]);
            }
    }
    const float dec = fp4_dec(a.W_amax);
#pragma unroll
    for (int n = 0; n < kMaxN; ++n) {
        if (n >= a.N) break;
        float t = acc[n];
        for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (lane == 0) {
            t *= dec;
            if (a.bias) t += a.bias[m];
            if (a.silu) t = silu_f(t);
            if (a.bf16) static_cast<__nv_bfloat16 *>(a.y)[n * a.ldy + m] = __float2bfloat16_rn(t);
            else static_cast<float *>(a.y)[n * a.ldy + m] = t;
        }
    }
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int tsd_op_fp4_gemv(const void * W, const void * W_scales, const float * W_amax, int fmt, int M, int K,
                               const float * x, int64_t ldx, int N, const float * bias, int act, void * y, int y_type,
                               int64_t ldy, void * stream) {
    if (tsd_fp4_scale_bytes(M, K, fmt) < 0 || M < 1 || N < 0 || N > kMaxN || ldx < K || ldy < M ||
        (act != TSD_ACT_NONE && act != TSD_ACT_SILU) || (fmt == TSD_FP4_MX && W_amax) ||
        (y_type != TSD_TYPE_F32 && y_type != TSD_TYPE_BF16))
        return TSD_ERR_ARG;
    if (N == 0) return TSD_OK;
    if (!W || !W_scales || !x || !y || !aligned(W, 16) || !aligned(W_scales, 16) || !aligned(x, 4) || !aligned(bias, 4) ||
        !aligned(W_amax, 4) || !aligned(y, float_size(y_type)))
        return TSD_ERR_ARG;
    OperandDevice dev({W, W_scales, W_amax, x, bias, y});
    if (dev.rc) return dev.rc;
    Fp4GemvArgs a;
    a.W = static_cast<const uint8_t *>(W); a.Ws = static_cast<const uint8_t *>(W_scales);
    a.W_amax = W_amax; a.x = x; a.bias = bias; a.y = y; a.ldx = ldx; a.ldy = ldy;
    a.M = M; a.K = K; a.N = N; a.silu = act == TSD_ACT_SILU; a.bf16 = y_type == TSD_TYPE_BF16;
    const dim3 grid((M + 7) / 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = fmt == TSD_FP4_MX ? launch_pdl(fp4_gemv_kernel<TSD_FP4_MX>, grid, dim3(256), 0, st, a)
                                            : launch_pdl(fp4_gemv_kernel<TSD_FP4_NV>, grid, dim3(256), 0, st, a);
    if (e != cudaSuccess) {
        fprintf(stderr, "tsd_op_fp4_gemv: %s\n", cudaGetErrorString(e));
        return TSD_ERR_CUDA;
    }
    return TSD_OK;
}
