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

#include <type_traits>

namespace tsd {

namespace {

// a / b for b > 0, rounded to odd (r = 1 / b to nearest). The first product can be two ulps off, so
// it is refined once; then the exact quotient lies within one ulp. Inexact: of the two neighbours
// around the exact quotient the odd one, (q or q - 1) | 1 in magnitude. The refinement loses the
// sign of a zero, hence the copysign.
__device__ __forceinline__ float div_to_odd(float a, float b, float r) {
    const float q0 = a * r;
    const float q = fmaf(fmaf(-q0, b, a), r, q0);
    const float rem = fmaf(-q, b, a);
    const int bits = __float_as_int(q), below = (bits ^ __float_as_int(rem)) >> 31;   // -1 where the quotient is smaller
    return copysignf(rem != 0.f ? __int_as_float((bits + below) | 1) : q, a);
}

// Every kernel here gives a thread 16 consecutive elements at a time (a "piece": one NV block, half an
// MX block) and a warp 32 pieces of one row; a thread has 128 bytes of loads (stores) in flight.
constexpr int kPiece = 16, kWarps = 8;
template <typename T> constexpr int kDeep = 8 / (int)sizeof(T);

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// 16 elements as stored. ALIGN: bytes that every piece is known to be aligned to (32, 16, or 0: of one element only).
template <typename T> struct alignas(32) Piece { T e[kPiece]; };
template <typename T, int ALIGN> __device__ __forceinline__ void load_piece(const T * p, Piece<T> & v) {
    constexpr int kBytes = kPiece * (int)sizeof(T);
    if constexpr (ALIGN == 32) {
#pragma unroll
        for (int i = 0; i < kBytes / 32; ++i) {
            uint32_t * u = reinterpret_cast<uint32_t *>(&v) + 8 * i;
            asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
                         : "l"(reinterpret_cast<const char *>(p) + 32 * i));
        }
    } else if constexpr (ALIGN == 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4 *>(&v)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v.e[i] = p[i];
    }
}
template <typename T, int ALIGN> __device__ __forceinline__ void store_piece(T * p, const Piece<T> & v) {
    constexpr int kBytes = kPiece * (int)sizeof(T);
    if constexpr (ALIGN == 32) {
#pragma unroll
        for (int i = 0; i < kBytes / 32; ++i) {
            const uint32_t * u = reinterpret_cast<const uint32_t *>(&v) + 8 * i;
            asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                         ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
                           "l"(reinterpret_cast<char *>(p) + 32 * i) : "memory");
        }
    } else if constexpr (ALIGN == 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(&v)[i];
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) p[i] = v.e[i];
    }
}

__global__ void zero_kernel(unsigned * p) {
    pdl_launch_dependents();
    pdl_wait();
    *p = 0;
}

// max |x|: |x| as an unsigned integer orders like |x|, with NaN above everything. K need not be a
// multiple of the piece: a row's last elements are taken one by one. One atomic per CTA.
template <typename T, int ALIGN>
__global__ void __launch_bounds__(32 * kWarps) absmax_kernel(const T * __restrict__ x, int rows, int K, long long ldx,
                                                             unsigned * __restrict__ amax) {
    __shared__ unsigned part[kWarps];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pieces = K / kPiece;
    unsigned m = 0;
    for (long long r = blockIdx.x * kWarps + warp; r < rows; r += gridDim.x * kWarps) {
        const T * row = x + r * ldx;
        for (int c0 = blockIdx.y * 32 * kDeep<T> + lane; c0 - lane < pieces; c0 += gridDim.y * 32 * kDeep<T>) {
            Piece<T> v[kDeep<T>];
#pragma unroll
            for (int d = 0; d < kDeep<T>; ++d)
                if (c0 + 32 * d < pieces) load_piece<T, ALIGN>(row + (long long)(c0 + 32 * d) * kPiece, v[d]);
#pragma unroll
            for (int d = 0; d < kDeep<T>; ++d)
                if (c0 + 32 * d < pieces) {
#pragma unroll
                    for (int i = 0; i < kPiece; ++i) m = max(m, __float_as_uint(Elem<T>::to(v[d].e[i])) & 0x7fffffffu);
                }
        }
        if (blockIdx.y == 0 && lane < K - pieces * kPiece)
            m = max(m, __float_as_uint(Elem<T>::to(row[pieces * kPiece + lane])) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) part[warp] = m;
    __syncthreads();
    if (threadIdx.x < kWarps) {
        m = __reduce_max_sync((1u << kWarps) - 1, part[threadIdx.x]);
        if (threadIdx.x == 0 && m) atomicMax(amax, m);
    }
}

// A warp per row (rows of the last row tile past the end too: their scale bytes are zero) and 32 * kDeep<T>
// pieces. The scales of four blocks make a 32-bit word, which one lane collects and writes.
template <typename T, int ALIGN, int FMT>
__global__ void __launch_bounds__(32 * kWarps) quantize_kernel(const T * __restrict__ x, int rows, int K, long long ldx,
                                                               const float * __restrict__ amax, uint8_t * __restrict__ codes,
                                                               uint8_t * __restrict__ scales) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kLanes = FMT == TSD_FP4_MX ? 8 : 4;          // lanes whose scales make a word
    const int lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int kt = fp4_ktiles(K, FMT), pieces = K / kPiece;
    const int c0 = blockIdx.y * 32 * kDeep<T> + lane;
    Piece<T> v[kDeep<T>];
    const T * row = x + (r < rows ? r : rows - 1) * ldx;       // what lies past the end is read from the last row or piece,
#pragma unroll                                                 // and not written
    for (int d = 0; d < kDeep<T>; ++d) load_piece<T, ALIGN>(row + (long long)min(c0 + 32 * d, pieces - 1) * kPiece, v[d]);
    const float enc = fp4_enc(amax);
#pragma unroll
    for (int d = 0; d < kDeep<T>; ++d) {
        const int c = c0 + 32 * d;
        if (c - lane >= kt * kLanes) break;                    // the whole warp
        const bool live = r < rows && c < pieces;
        float z[kPiece];
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
            z[i] = Elem<T>::to(v[d].e[i]) * enc;
            m = max(m, __float_as_uint(z[i]) & 0x7fffffffu);
        }
        uint32_t byte;
        bool zero = false;
        if constexpr (FMT == TSD_FP4_MX) {
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));    // the other half of the block
            // exponent field of the maximum is floor(log2) + 127 (subnormals: far below 2^-125); an infinity
            // or a NaN makes the whole block NaN
            const int b = max((int)(m >> 23) - 2, 0);
            byte = m >= 0x7f800000u ? 255u : (uint32_t)b;
            const float inv = __int_as_float((254 - b) << 23);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) z[i] *= inv;
        } else {
            uint16_t s8;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(s8) : "f"(0.f), "f"(div_to_odd(__uint_as_float(m), 6.0f, 1.0f / 6.0f)));
            byte = m >= 0x7f800000u ? 0x7fu : (uint32_t)s8;
            const float s = fp4_scale_value<FMT>(s8);
            zero = !(s > 0.f);                                 // nothing fits under the scale: codes of zero
            const float b = zero ? 1.0f : s, inv = __frcp_rn(b);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) z[i] = div_to_odd(z[i], b, inv);
        }
        const uint2 q = make_uint2(fp4_codes8(z), fp4_codes8(z + 8));
        if (live) *reinterpret_cast<uint2 *>(codes + r * (K / 2) + (long long)c * 8) = zero ? make_uint2(0, 0) : q;
        byte = live ? byte : 0u;
        // byte j of a word comes from the lane (group of two lanes) j of its kLanes
        uint32_t w = byte << (8 * ((lane / (kLanes / 4)) & 3));
        if constexpr (FMT == TSD_FP4_MX) {
            w |= __shfl_xor_sync(0xffffffffu, w, 2);
            w |= __shfl_xor_sync(0xffffffffu, w, 4);
        } else {
            w |= __shfl_xor_sync(0xffffffffu, w, 1);
            w |= __shfl_xor_sync(0xffffffffu, w, 2);
        }
        if (lane % kLanes == 0 && c < kt * kLanes)
            *reinterpret_cast<uint32_t *>(scales + fp4_scale_at(r, c / kLanes, kt)) = w;
    }
}

template <typename T, int ALIGN, int FMT>
__global__ void __launch_bounds__(32 * kWarps) dequantize_kernel(const uint8_t * __restrict__ codes,
                                                                 const uint8_t * __restrict__ scales,
                                                                 const float * __restrict__ amax, int rows, int K,
                                                                 T * __restrict__ y, long long ldy) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kLanes = FMT == TSD_FP4_MX ? 8 : 4;
    const int lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int kt = fp4_ktiles(K, FMT), pieces = K / kPiece;
    const int c0 = blockIdx.y * 32 * kDeep<T> + lane;
    uint2 q[kDeep<T>];
    uint32_t b[kDeep<T>];
#pragma unroll
    for (int d = 0; d < kDeep<T>; ++d) {
        const int c = c0 + 32 * d;
        if (c < pieces) {
            q[d] = __ldg(reinterpret_cast<const uint2 *>(codes + r * (K / 2) + (long long)c * 8));
            b[d] = __ldg(scales + fp4_scale_at(r, c / kLanes, kt) + c % kLanes / (kLanes / 4));
        }
    }
    const float dec = fp4_dec(amax);
#pragma unroll
    for (int d = 0; d < kDeep<T>; ++d) {
        const int c = c0 + 32 * d;
        if (c >= pieces) break;
        const float s = fp4_scale_value<FMT>(b[d]);
        float f[kPiece];
        fp4_values8(q[d].x, f);
        fp4_values8(q[d].y, f + 8);
        Piece<T> o;
#pragma unroll
        for (int i = 0; i < kPiece; ++i) o.e[i] = Elem<T>::from(f[i] * s * dec);
        store_piece<T, ALIGN>(y + r * ldy + (long long)c * kPiece, o);
    }
}

// The widest access every piece of a tensor allows.
int piece_align(const void * p, long long ld, int es) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * es);
    return at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 0;
}
// f(element type, alignment) for a tensor's type and alignment.
template <typename F> cudaError_t with_type(int type, int align, F && f) {
    const auto with_align = [&](auto elem) {
        return align == 32   ? f(elem, std::integral_constant<int, 32>())
               : align == 16 ? f(elem, std::integral_constant<int, 16>())
                             : f(elem, std::integral_constant<int, 0>());
    };
    return type == TSD_TYPE_F32 ? with_align(float()) : type == TSD_TYPE_F16 ? with_align(__half()) : with_align(__nv_bfloat16());
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int64_t tsd_fp4_scale_bytes(int64_t rows, int64_t K, int fmt) {
    if (rows < 0 || rows > TSD_FP4_MAX_ROWS || K < 32 || K > TSD_FP4_MAX_K || K % 32 || (fmt != TSD_FP4_MX && fmt != TSD_FP4_NV)) return -1;
    return (rows + 127) / 128 * fp4_ktiles((int)K, fmt) * kScaleTile;
}

extern "C" int tsd_op_fp4_absmax(const void * x, int type, int rows, int K, int64_t ldx, float * amax, void * stream) {
    const int xs = float_size(type);
    if (rows < 0 || K < 1 || ldx < K || !xs || !amax || !aligned(amax, 4) || (rows && (!x || !aligned(x, xs)))) return TSD_ERR_ARG;
    OperandDevice dev({rows ? x : nullptr, amax});
    if (dev.rc) return dev.rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // the maximum starts from zero: a kernel of one thread, which the next one's launch overlaps (a memset it would not)
    cudaError_t e = launch_pdl(zero_kernel, dim3(1), dim3(1), 0, st, reinterpret_cast<unsigned *>(amax));
    if (e == cudaSuccess && rows) {
        // a few CTAs per SM, each with one atomic at its end; few rows: their length is split too
        const int span = kPiece * 32 * 8 / xs;
        const int gx = rows / kWarps + 1 < 740 ? rows / kWarps + 1 : 740;
        const int gy = K / span + 1 < 740 / gx ? K / span + 1 : 740 / gx;
        e = with_type(type, piece_align(x, ldx, xs), [&](auto elem, auto align) {
            using T = decltype(elem);
            return launch_pdl(absmax_kernel<T, decltype(align)::value>, dim3(gx, gy), dim3(32 * kWarps), 0, st,
                              static_cast<const T *>(x), rows, K, (long long)ldx, reinterpret_cast<unsigned *>(amax));
        });
    }
    return launch_status("tsd_op_fp4_absmax", e);
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
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t * c = static_cast<uint8_t *>(codes), * s = static_cast<uint8_t *>(scales);
    const unsigned gx = (unsigned)(((long long)rows + 127) / 128 * (128 / kWarps));
    const int lanes = fp4_ktiles(K, fmt) * (fmt == TSD_FP4_MX ? 8 : 4);
    const int span = 32 * 8 / xs;          // pieces a warp takes
    const dim3 grid(gx, (lanes + span - 1) / span);   // y: 32768 at most
    const cudaError_t e = with_type(type, piece_align(x, ldx, xs), [&](auto elem, auto align) {
        using T = decltype(elem);
        constexpr int A = decltype(align)::value;
        return launch_pdl(fmt == TSD_FP4_MX ? quantize_kernel<T, A, TSD_FP4_MX> : quantize_kernel<T, A, TSD_FP4_NV>, grid,
                          dim3(32 * kWarps), 0, st, static_cast<const T *>(x), rows, K, (long long)ldx, amax, c, s);
    });
    return launch_status("tsd_op_fp4_quantize", e);
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
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint8_t * c = static_cast<const uint8_t *>(codes), * s = static_cast<const uint8_t *>(scales);
    const int span = 32 * 8 / ys;          // pieces a warp takes
    const dim3 grid((unsigned)((rows + (long long)kWarps - 1) / kWarps), (K / kPiece + span - 1) / span);   // y: likewise
    const cudaError_t e = with_type(type, piece_align(y, ldy, ys), [&](auto elem, auto align) {
        using T = decltype(elem);
        constexpr int A = decltype(align)::value;
        return launch_pdl(fmt == TSD_FP4_MX ? dequantize_kernel<T, A, TSD_FP4_MX> : dequantize_kernel<T, A, TSD_FP4_NV>, grid,
                          dim3(32 * kWarps), 0, st, c, s, amax, rows, K, static_cast<T *>(y), (long long)ldy);
    });
    return launch_status("tsd_op_fp4_dequantize", e);
}
