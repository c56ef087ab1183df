// fp4.cuh — the microscaled 4-bit format (include/tsd_ops.h): sizes, layout of the scales, conversions.
#pragma once
#include <cfloat>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/tsd_ops.h"

namespace tsd {

constexpr int kScaleTile = 512;   // bytes of a tile of scales: 128 rows x 4 blocks

__host__ __device__ constexpr int fp4_block(int fmt) { return fmt == TSD_FP4_MX ? 32 : 16; }
// Tiles of scales along K.
__host__ __device__ constexpr int fp4_ktiles(int K, int fmt) { return (K / fp4_block(fmt) + 3) / 4; }
// Where the scales of blocks 4 t .. 4 t + 3 of row r lie (four consecutive bytes).
__host__ __device__ constexpr long long fp4_scale_at(long long r, int t, int ktiles) {
    return ((r >> 7) * ktiles + t) * kScaleTile + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// The absolute maximum a tensor is scaled by: 2688 (a factor of 1 both ways) where it has none.
__device__ __forceinline__ float fp4_amax(const float * amax) {
    const float a = amax ? *amax : 2688.0f;
    return a >= 7.88860905e-31f && a <= FLT_MAX ? a : 2688.0f;   // 2^-100
}
// The factors before and after. enc by way of the reciprocal, which is what torch computes for 2688 / amax: with the
// quotient itself a few values of a tensor next to a border between two codes would fall on its other side (2688 by way
// of its own reciprocal is exactly one). Above 2^126 the reciprocal is subnormal and has up to two bits fewer; the bytes are those
// of this definition all the same.
__device__ __forceinline__ float fp4_enc(const float * amax) { return 2688.0f * __frcp_rn(fp4_amax(amax)); }
__device__ __forceinline__ float fp4_dec(const float * amax) { return fp4_amax(amax) / 2688.0f; }

// Value of a scale byte.
template <int FMT> __device__ __forceinline__ float fp4_scale_value(uint32_t b) {
    if constexpr (FMT == TSD_FP4_MX) {
        // the byte is an f32 exponent field; 2^-127 is subnormal
        return b == 255 ? __int_as_float(0x7fffffff) : b == 0 ? __int_as_float(1 << 22) : __int_as_float((int)b << 23);
    } else {
        // e4m3 widened to f16 (exact): sign and exponent moved, then the exponent bias by a factor
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)b));
        float f;
        asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;}" : "=f"(f) : "r"(h2));
        return f;
    }
}

// Eight e2m1 codes from eight floats, v[0] in the low nibble (to nearest even, at most 6 in magnitude).
__device__ __forceinline__ uint32_t fp4_codes8(const float * v) {
    uint32_t r;
    asm("{.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// The values of eight codes (exact).
__device__ __forceinline__ void fp4_values8(uint32_t w, float * v) {
    uint32_t h[4];
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;}"
            : "=f"(v[2 * i]), "=f"(v[2 * i + 1]) : "r"(h[i]));
}

}  // namespace tsd
