// fp4_gemm.cu — product of two microscaled 4-bit tensors (sm_100a); format: include/tsd_ops.h.
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "op_check.h"

#include <cstdio>

namespace tsd {

namespace {

struct Fp4GemmArgs {
    const uint8_t * W, * Ws, * X, * Xs;
    const float * W_amax, * X_amax, * bias;
    void * out;
    long long ldo;
    int M, N, K, swiglu, silu, bf16;
};

constexpr int kT = 64, kKS = 32;   // tile of tokens x features, K step

// Plain form: operands dequantised into shared memory, f32 FMAs, 4 x 4 outputs per thread.
template <int FMT>
__global__ void __launch_bounds__(256) fp4_gemm_kernel(const Fp4GemmArgs a) {
    __shared__ float xs[kKS][kT + 1], ws[kKS][kT + 1];
    pdl_launch_dependents();
    pdl_wait();
    const int n0 = blockIdx.y * kT, m0 = blockIdx.x * kT;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int kt = fp4_ktiles(a.K, FMT);
    float acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += kKS) {
        // 64 rows x 4 words of 8 codes for each operand
        const int row = threadIdx.x / 4, w = threadIdx.x % 4;
        const int k = k0 + w * 8, j = k / fp4_block(FMT);
#pragma unroll
        for (int op = 0; op < 2; ++op) {
            const int r = (op ? m0 : n0) + row;
            float v[8] = {};
            if (r < (op ? a.M : a.N)) {
                const uint8_t * c = op ? a.W : a.X, * s = op ? a.Ws : a.Xs;
                fp4_values8(*reinterpret_cast<const uint32_t *>(c + (long long)r * (a.K / 2) + k / 2), v);
                const float sc = fp4_scale_value<FMT>(s[fp4_scale_at(r, j >> 2, kt) + (j & 3)]);
                for (int e = 0; e < 8; ++e) v[e] *= sc;
            }
            for (int e = 0; e < 8; ++e) (op ? ws : xs)[w * 8 + e][row] = v[e];
        }
        __syncthreads();
#pragma unroll 8
        for (int kk = 0; kk < kKS; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int jj = 0; jj < 4; ++jj) acc[i][jj] = fmaf(xs[kk][ty * 4 + i], ws[kk][tx * 4 + jj], acc[i][jj]);
        __syncthreads();
    }
    const float alpha = fp4_dec(a.W_amax) * fp4_dec(a.X_amax);
    const auto put = [&](long long at, float v) {
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
        else static_cast<float *>(a.out)[at] = v;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + ty * 4 + i;
        if (n >= a.N) break;
#pragma unroll
        for (int jj = 0; jj < 4; jj += 2) {
            const int m = m0 + tx * 4 + jj;
            float u = acc[i][jj] * alpha, v = acc[i][jj + 1] * alpha;
            if (a.swiglu) {
                if (m < a.M) put(n * a.ldo + m / 2, silu_f(u) * v);
                continue;
            }
            if (m < a.M) {
                if (a.bias) u += a.bias[m];
                put(n * a.ldo + m, a.silu ? silu_f(u) : u);
            }
            if (m + 1 < a.M) {
                if (a.bias) v += a.bias[m + 1];
                put(n * a.ldo + m + 1, a.silu ? silu_f(v) : v);
            }
        }
    }
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int tsd_op_fp4_gemm(const void * W, const void * W_scales, const float * W_amax, int M, const void * X,
                               const void * X_scales, const float * X_amax, int N, int K, int fmt, int mode, int act,
                               const float * bias, void * out, int out_type, int64_t ldo, int * err, void * stream) {
    if (tsd_fp4_scale_bytes(M, K, fmt) < 0 || tsd_fp4_scale_bytes(N, K, fmt) < 0 || M < 1 ||
        (mode != TSD_EPI_STORE && mode != TSD_EPI_SWIGLU) || (act != TSD_ACT_NONE && act != TSD_ACT_SILU) ||
        (mode == TSD_EPI_SWIGLU && (M % 2 || bias || act != TSD_ACT_NONE)) || (fmt == TSD_FP4_MX && (W_amax || X_amax)) ||
        (out_type != TSD_TYPE_F32 && out_type != TSD_TYPE_BF16) || ldo < (mode == TSD_EPI_SWIGLU ? M / 2 : M))
        return TSD_ERR_ARG;
    if (N == 0) return TSD_OK;
    if (!W || !W_scales || !X || !X_scales || !out || !aligned(W, 16) || !aligned(W_scales, 16) || !aligned(X, 16) ||
        !aligned(X_scales, 16) || !aligned(out, float_size(out_type)) || !aligned(bias, 4) || !aligned(W_amax, 4) ||
        !aligned(X_amax, 4) || !aligned(err, 4))
        return TSD_ERR_ARG;
    OperandDevice dev({W, W_scales, W_amax, X, X_scales, X_amax, bias, out, err});
    if (dev.rc) return dev.rc;
    Fp4GemmArgs a;
    a.W = static_cast<const uint8_t *>(W); a.Ws = static_cast<const uint8_t *>(W_scales);
    a.X = static_cast<const uint8_t *>(X); a.Xs = static_cast<const uint8_t *>(X_scales);
    a.W_amax = W_amax; a.X_amax = X_amax; a.bias = bias; a.out = out; a.ldo = ldo;
    a.M = M; a.N = N; a.K = K; a.swiglu = mode == TSD_EPI_SWIGLU; a.silu = act == TSD_ACT_SILU;
    a.bf16 = out_type == TSD_TYPE_BF16;
    const dim3 grid((M + kT - 1) / kT, (N + kT - 1) / kT);
    if (grid.y > 65535) return TSD_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = fmt == TSD_FP4_MX ? launch_pdl(fp4_gemm_kernel<TSD_FP4_MX>, grid, dim3(256), 0, st, a)
                                            : launch_pdl(fp4_gemm_kernel<TSD_FP4_NV>, grid, dim3(256), 0, st, a);
    if (e != cudaSuccess) {
        fprintf(stderr, "tsd_op_fp4_gemm: %s\n", cudaGetErrorString(e));
        return TSD_ERR_CUDA;
    }
    return TSD_OK;
}
