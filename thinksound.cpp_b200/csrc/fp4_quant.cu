// fp4_quant.cu — tensors into and out of microscaled 4-bit floating point (sm_100a).
//
// Format and definitions: include/tsd_ops.h. Bound: memory; a few operations per element.
//
// The roundings are those of the exact quotients. z / s with s a power of two (MX) is exact in f32.
// With s an e4m3 value (NV) the f32 quotient can land on a border between two codes that the exact
// one misses, so the quotient is rounded to odd: q = z * (1 / s) is within one ulp, the remainder
// z - q s is exact in an FMA, and where it is not zero the last bit of q is set on the side of
// the exact quotient. Every border has a zero last bit, so the conversion then decides as for
// the exact quotient. The scale max|z| / 6 -> e4m3 is treated in the same way.
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "op_check.h"

#include <cstdio>

namespace tsd {

namespace {

// a / b for b > 0, rounded to odd (r = 1 / b to nearest). The first product can be two ulps off, so
// it is refined once; then the exact quotient lies within one ulp. Quotients that underflow
// stay as they are: far below the first border.
__device__ __forceinline__ float div_to_odd(float a, float b, float r) {
    const float q0 = a * r;
    const float q = fmaf(fmaf(-q0, b, a), r, q0);
    const float rem = fmaf(-q, b, a);
    int bits = __float_as_int(q);
    if (rem != 0.f && q != 0.f && !(bits & 1)) bits += ((rem < 0.f) == (q < 0.f)) ? 1 : -1;   // magnitude up / down
    return copysignf(__int_as_float(bits), a);   // the refinement loses the sign of a zero
}

__device__ __forceinline__ float load_any(const void * x, int type, long long i) {
    if (type == TSD_TYPE_F32) return static_cast<const float *>(x)[i];
    if (type == TSD_TYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(x)[i]);
    return __half2float(static_cast<const __half *>(x)[i]);
}

__global__ void absmax_kernel(const void * __restrict__ x, int type, long long rows, int K, long long ldx,
                              unsigned * __restrict__ amax) {
    pdl_launch_dependents();
    pdl_wait();
    // |x| as an unsigned integer orders like |x|, with NaN above everything
    unsigned m = 0;
    const long long n = rows * K;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x)
        m = max(m, __float_as_uint(load_any(x, type, i / K * ldx + i % K)) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0 && m) atomicMax(amax, m);
}

// One thread per block of elements, blocks of the padding included (their scales are zero).
template <int FMT>
__global__ void quantize_kernel(const void * __restrict__ x, int type, long long rows, int K, long long ldx,
                                const float * __restrict__ amax, uint8_t * __restrict__ codes,
                                uint8_t * __restrict__ scales) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int B = fp4_block(FMT);
    const int kt = fp4_ktiles(K, FMT), nb = K / B;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long r = i / (4 * kt);
    const int j = (int)(i % (4 * kt));
    if (r >= (rows + 127) / 128 * 128) return;
    uint8_t * sp = scales + fp4_scale_at(r, j >> 2, kt) + (j & 3);
    if (r >= rows || j >= nb) {
        *sp = 0;
        return;
    }
    const float enc = fp4_enc(amax);
    float z[B];
    unsigned m = 0;
    for (int e = 0; e < B; ++e) {
        z[e] = load_any(x, type, r * ldx + (long long)j * B + e) * enc;
        m = max(m, __float_as_uint(z[e]) & 0x7fffffffu);
    }
    const float top = __uint_as_float(m);
    if (m >= 0x7f800000u) {   // an infinity or a NaN: the whole block is NaN
        *sp = FMT == TSD_FP4_MX ? 255 : 0x7f;
    } else if constexpr (FMT == TSD_FP4_MX) {
        // exponent field of the maximum is floor(log2) + 127 (subnormals: far below 2^-125)
        const int b = max((int)(m >> 23) - 2, 0);
        *sp = (uint8_t)b;
        const float inv = __int_as_float((254 - b) << 23);
        for (int e = 0; e < B; ++e) z[e] *= inv;
    } else {
        uint16_t s8;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(s8) : "f"(0.f), "f"(div_to_odd(top, 6.0f, 1.0f / 6.0f)));
        *sp = (uint8_t)s8;
        const float s = fp4_scale_value<FMT>(s8);
        const float inv = s > 0.f ? 1.0f / s : 0.f;
        for (int e = 0; e < B; ++e) z[e] = s > 0.f ? div_to_odd(z[e], s, inv) : 0.f;
    }
    uint32_t * cp = reinterpret_cast<uint32_t *>(codes + r * (K / 2) + (long long)j * (B / 2));
#pragma unroll
    for (int e = 0; e < B / 8; ++e) cp[e] = fp4_codes8(z + 8 * e);
}

// One thread per eight elements.
template <int FMT>
__global__ void dequantize_kernel(const uint32_t * __restrict__ codes, const uint8_t * __restrict__ scales,
                                  const float * __restrict__ amax, long long rows, int K, void * __restrict__ y, int type,
                                  long long ldy) {
    pdl_launch_dependents();
    pdl_wait();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int per = K / 8;
    if (i >= rows * per) return;
    const long long r = i / per;
    const int k = (int)(i % per) * 8;
    const int j = k / fp4_block(FMT);
    const float s = fp4_scale_value<FMT>(scales[fp4_scale_at(r, j >> 2, fp4_ktiles(K, FMT)) + (j & 3)]);
    const float dec = fp4_dec(amax);
    float v[8];
    fp4_values8(codes[i], v);
    for (int e = 0; e < 8; ++e) {
        const float o = v[e] * s * dec;
        const long long at = r * ldy + k + e;
        if (type == TSD_TYPE_F32) static_cast<float *>(y)[at] = o;
        else if (type == TSD_TYPE_BF16) static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(o);
        else static_cast<__half *>(y)[at] = __float2half_rn(o);
    }
}

int done(const char * fn, cudaError_t e) {
    if (e == cudaSuccess) return TSD_OK;
    fprintf(stderr, "%s: %s\n", fn, cudaGetErrorString(e));
    return TSD_ERR_CUDA;
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int64_t tsd_fp4_scale_bytes(int64_t rows, int64_t K, int fmt) {
    if (rows < 0 || rows > INT32_MAX || K < 32 || K > INT32_MAX || K % 32 || (fmt != TSD_FP4_MX && fmt != TSD_FP4_NV)) return -1;
    return (rows + 127) / 128 * fp4_ktiles((int)K, fmt) * kScaleTile;
}

extern "C" int tsd_op_fp4_absmax(const void * x, int type, int rows, int K, int64_t ldx, float * amax, void * stream) {
    const int xs = float_size(type);
    if (rows < 0 || K < 1 || ldx < K || !xs || !amax || !aligned(amax, 4) || (rows && (!x || !aligned(x, xs)))) return TSD_ERR_ARG;
    OperandDevice dev({rows ? x : nullptr, amax});
    if (dev.rc) return dev.rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaMemsetAsync(amax, 0, sizeof(float), st);
    if (e == cudaSuccess && rows) {
        const long long n = (long long)rows * K;
        const unsigned grid = (unsigned)(n / 2048 + 1 < 1184 ? n / 2048 + 1 : 1184);
        e = launch_pdl(absmax_kernel, dim3(grid), dim3(256), 0, st, x, type, (long long)rows, K, (long long)ldx,
                       reinterpret_cast<unsigned *>(amax));
    }
    return done("tsd_op_fp4_absmax", e);
}

extern "C" int tsd_op_fp4_quantize(const void * x, int type, int rows, int K, int64_t ldx, int fmt, const float * amax,
                                   void * codes, void * scales, void * stream) {
    const int xs = float_size(type);
    if (tsd_fp4_scale_bytes(rows, K, fmt) < 0 || ldx < K || !xs || (fmt == TSD_FP4_MX && amax)) return TSD_ERR_ARG;
    if (rows == 0) return TSD_OK;
    if (!x || !codes || !scales || !aligned(x, xs) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(amax, 4))
        return TSD_ERR_ARG;
    OperandDevice dev({x, codes, scales, amax});
    if (dev.rc) return dev.rc;
    const long long n = ((long long)rows + 127) / 128 * 128 * fp4_ktiles(K, fmt) * 4;
    if ((n + 127) / 128 > INT32_MAX) return TSD_ERR_ARG;
    const dim3 grid((unsigned)((n + 127) / 128));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t * c = static_cast<uint8_t *>(codes), * s = static_cast<uint8_t *>(scales);
    const cudaError_t e =
        fmt == TSD_FP4_MX
            ? launch_pdl(quantize_kernel<TSD_FP4_MX>, grid, dim3(128), 0, st, x, type, (long long)rows, K, (long long)ldx, amax, c, s)
            : launch_pdl(quantize_kernel<TSD_FP4_NV>, grid, dim3(128), 0, st, x, type, (long long)rows, K, (long long)ldx, amax, c, s);
    return done("tsd_op_fp4_quantize", e);
}

extern "C" int tsd_op_fp4_dequantize(const void * codes, const void * scales, int fmt, const float * amax, int rows, int K,
                                     void * y, int type, int64_t ldy, void * stream) {
    const int ys = float_size(type);
    if (tsd_fp4_scale_bytes(rows, K, fmt) < 0 || ldy < K || !ys || (fmt == TSD_FP4_MX && amax)) return TSD_ERR_ARG;
    if (rows == 0) return TSD_OK;
    if (!y || !codes || !scales || !aligned(y, ys) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(amax, 4))
        return TSD_ERR_ARG;
    OperandDevice dev({codes, scales, amax, y});
    if (dev.rc) return dev.rc;
    const long long n = (long long)rows * (K / 8);
    if ((n + 255) / 256 > INT32_MAX) return TSD_ERR_ARG;
    const dim3 grid((unsigned)((n + 255) / 256));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint32_t * c = static_cast<const uint32_t *>(codes);
    const uint8_t * s = static_cast<const uint8_t *>(scales);
    const cudaError_t e =
        fmt == TSD_FP4_MX
            ? launch_pdl(dequantize_kernel<TSD_FP4_MX>, grid, dim3(256), 0, st, c, s, amax, (long long)rows, K, y, type, (long long)ldy)
            : launch_pdl(dequantize_kernel<TSD_FP4_NV>, grid, dim3(256), 0, st, c, s, amax, (long long)rows, K, y, type, (long long)ldy);
    return done("tsd_op_fp4_dequantize", e);
}
