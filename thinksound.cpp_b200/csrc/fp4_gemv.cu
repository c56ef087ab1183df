// fp4_gemv.cu — microscaled 4-bit weights times a few f32 vectors (sm_100a); format: include/tsd_ops.h.
//
//   y[n][m] = act(dec * sum over blocks b of s[m][b] * sum_{k in b} c[m][k] x[n][k] + bias[m])
//
// Bound: the weight bytes for few vectors, instructions for many. A code costs half a conversion (e2m1x2 ->
// f16x2), one f16 -> f32 and N / 2 packed f32 FMAs (fma.rn.f32x2); the block's scale is applied to the
// block's sum. Everything after the (exact) conversion is f32.
//
// A warp takes R rows and 32 * KL elements of K at a time: a lane's KL elements (a block, or a part of
// one) of its N vectors stay in registers for all R rows, whose codes and scales are all requested
// before the first is used. The rows are those whose scale bytes share sectors: 2 p, 2 p + 1 of
// one or more of the four groups of 32 in a scale tile. At the end a transposing butterfly adds the
// R * N sums over the lanes, in a fixed order.
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "op_check.h"

#include <cstdio>

namespace tsd {

namespace {

struct Fp4GemvArgs {
    const uint8_t * W, * Ws;
    const float * W_amax, * x, * bias;
    void * y;
    long long ldx, ldy;
    int M, K, N, silu, bf16, x_vec, units;
};

constexpr int kGemvWarps = 4;

// Sum over the lanes of V values each (V a power of two up to 32): afterwards v[0] of lane l is the total of
// value l / (32 / V).
template <int V> __device__ __forceinline__ void lanes_sum(float (&v)[V], int lane) {
    int o = 16;
#pragma unroll
    for (int n = V / 2; n >= 1; n /= 2, o /= 2) {
        const bool up = lane & o;          // this lane keeps the upper half of the values
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
#pragma unroll
    for (; o >= 1; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
}

template <int FMT, int N, int KL, int R>
__global__ void __launch_bounds__(32 * kGemvWarps) fp4_gemv_kernel(const Fp4GemvArgs a) {
    constexpr int G = R / 2;               // groups of 32 rows a unit takes its row pair from
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int u = blockIdx.x * kGemvWarps + (threadIdx.x >> 5);
    if (u >= a.units) return;
    const int tile = u / (64 / G), p = u % 16, g0 = u % (64 / G) / 16 * G;
    const int kt = fp4_ktiles(a.K, FMT);
    const int row0 = tile * 128 + g0 * 32 + 2 * p;       // row i of the unit: row0 + i / 2 * 32 + i % 2
    const float dec = fp4_dec(a.W_amax);
    float acc[R * N] = {};
    for (int k = lane * KL; k - lane * KL < a.K; k += 32 * KL) {
        const bool live = k < a.K;
        uint32_t w[R][KL / 8];
        uint32_t sc[2][G];
        float x[N][KL];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = row0 + i / 2 * 32 + i % 2;
            const uint8_t * c = a.W + (long long)r * (a.K / 2) + k / 2;
#pragma unroll
            for (int j = 0; j < KL / 8; ++j) w[i][j] = 0;
            if (live && r < a.M) {
                if constexpr (KL == 16) {
                    const uint2 t = __ldg(reinterpret_cast<const uint2 *>(c));
                    w[i][0] = t.x;
                    w[i][1] = t.y;
                } else {
                    w[i][0] = __ldg(reinterpret_cast<const uint32_t *>(c));
                }
            }
        }
        const int blk = k / fp4_block(FMT);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int g = 0; g < G; ++g) sc[b][g] = 0;
            if (live) {                    // words of the unit's groups: consecutive bytes of the scale tile
                const uint8_t * s = a.Ws + fp4_scale_at(row0 + b, blk >> 2, kt);
                if constexpr (G == 4) {
                    const uint4 t = __ldg(reinterpret_cast<const uint4 *>(s));
                    sc[b][0] = t.x; sc[b][1] = t.y; sc[b][2] = t.z; sc[b][3] = t.w;
                } else if constexpr (G == 2) {
                    const uint2 t = __ldg(reinterpret_cast<const uint2 *>(s));
                    sc[b][0] = t.x; sc[b][1] = t.y;
                } else {
                    sc[b][0] = __ldg(reinterpret_cast<const uint32_t *>(s));
                }
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float * xr = a.x + n * a.ldx + k;
            if (live && n < a.N && a.x_vec) {
#pragma unroll
                for (int e = 0; e < KL; e += 4) {
                    const float4 t = __ldg(reinterpret_cast<const float4 *>(xr + e));
                    x[n][e] = t.x; x[n][e + 1] = t.y; x[n][e + 2] = t.z; x[n][e + 3] = t.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < KL; ++e) x[n][e] = live && n < a.N ? __ldg(xr + e) : 0.f;
            }
        }
        const int shift = 8 * (blk & 3);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float s = fp4_scale_value<FMT>((sc[i & 1][i / 2] >> shift) & 255u);
            float v[KL];
#pragma unroll
            for (int j = 0; j < KL / 8; ++j) fp4_values8(w[i][j], v + 8 * j);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float2 t = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < KL; e += 2) t = fma2(make_float2(v[e], v[e + 1]), make_float2(x[n][e], x[n][e + 1]), t);
                acc[i * N + n] = fmaf(t.x + t.y, s, acc[i * N + n]);
            }
        }
    }
    constexpr int V = R * N;
    lanes_sum<V>(acc, lane);
    const int i = lane / (32 / V) / N, n = lane / (32 / V) % N;
    const int m = row0 + i / 2 * 32 + i % 2;
    if (lane % (32 / V) == 0 && n < a.N && m < a.M) {
        float t = acc[0] * dec;
        if (a.bias) t += __ldg(a.bias + m);
        if (a.silu) t = silu_f(t);
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.y)[n * a.ldy + m] = __float2bfloat16_rn(t);
        else static_cast<float *>(a.y)[n * a.ldy + m] = t;
    }
}

template <int FMT, int N, int KL, int R> cudaError_t launch(Fp4GemvArgs & a, cudaStream_t st) {
    const long long units = (long long)((a.M + 127) / 128) * (128 / R);
    a.units = (int)units;
    return launch_pdl(fp4_gemv_kernel<FMT, N, KL, R>, dim3((unsigned)((units + kGemvWarps - 1) / kGemvWarps)),
                      dim3(32 * kGemvWarps), 0, st, a);
}

template <int FMT> cudaError_t launch_fmt(Fp4GemvArgs & a, int sms, cudaStream_t st) {
    // Rows per warp: many share the vectors' loads; few make enough warps of a small matrix.
    const bool many = a.M >= 128 * sms;
    if (a.N <= 1) return many ? launch<FMT, 1, 16, 8>(a, st) : launch<FMT, 1, 16, 2>(a, st);
    if (a.N <= 2) return many ? launch<FMT, 2, 16, 8>(a, st) : launch<FMT, 2, 16, 2>(a, st);
    if (a.N <= 4) return many ? launch<FMT, 4, 8, 8>(a, st) : launch<FMT, 4, 8, 2>(a, st);
    return many ? launch<FMT, 8, 8, 4>(a, st) : launch<FMT, 8, 8, 2>(a, st);
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int tsd_op_fp4_gemv(const void * W, const void * W_scales, const float * W_amax, int fmt, int M, int K,
                               const float * x, int64_t ldx, int N, const float * bias, int act, void * y, int y_type,
                               int64_t ldy, void * stream) {
    if (tsd_fp4_scale_bytes(M, K, fmt) < 0 || M < 1 || N < 0 || N > 8 || ldx < K || ldy < M ||
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
    a.x_vec = ldx % 4 == 0 && aligned(x, 16);
    int cur = 0, sms = 148;
    cudaGetDevice(&cur);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cur);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = fmt == TSD_FP4_MX ? launch_fmt<TSD_FP4_MX>(a, sms, st) : launch_fmt<TSD_FP4_NV>(a, sms, st);
    if (e != cudaSuccess) {
        fprintf(stderr, "tsd_op_fp4_gemv: %s\n", cudaGetErrorString(e));
        return TSD_ERR_CUDA;
    }
    return TSD_OK;
}
