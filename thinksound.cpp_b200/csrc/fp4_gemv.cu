// fp4_gemv.cu — microscaled 4-bit weights times a few f32 vectors (sm_100a); format: include/tsd_ops.h.
//
//   y[n][m] = act(dec * sum over blocks b of s[m][b] * sum_{k in b} c[m][k] x[n][k] + bias[m])
//
// Matrices of many rows go to fp4_gemv_tc.cu where their vectors fit; the two kernels here take the rest.
// Bound: the weight bytes for few vectors, instructions for many. A code costs half a conversion (e2m1x2 ->
// f16x2), one f16 -> f32 and N / 2 packed f32 FMAs (fma.rn.f32x2); the block's scale is applied to the
// block's sum. Everything after the (exact) conversion is f32; a sum that is not finite is formed again in f64, since |x| near
// f32's end may overflow before a small scale or factor is applied.
//
// A warp takes R rows and 32 * KL elements of K at a time: a lane's KL elements (a block, or a part of
// one) of its N vectors stay in registers for all R rows, whose codes and scales are all requested
// before the first is used. The rows are those whose scale bytes share sectors: 2 p, 2 p + 1 of
// one or more of the four groups of 32 in a scale tile. At the end a transposing butterfly adds the
// R * N sums over the lanes, in a fixed order.
#include "common.cuh"
#include "fp4.cuh"
#include "fp4_gemv.h"
#include "kernels.h"
#include "op_check.h"

#include <cfloat>

namespace tsd {

namespace {

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

// The scales of two rows' blocks (byte `blk` of either word) as f32.
template <int FMT> __device__ __forceinline__ float2 scale_pair(uint32_t w0, uint32_t w1, int blk) {
    if constexpr (FMT == TSD_FP4_MX) {
        return make_float2(fp4_scale_value<FMT>(w0 >> (8 * blk) & 255u), fp4_scale_value<FMT>(w1 >> (8 * blk) & 255u));
    } else {
        uint32_t h;                        // both bytes in one conversion
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)__byte_perm(w0, w1, blk | (4 + blk) << 4)));
        const __half2 h2 = *reinterpret_cast<const __half2 *>(&h);
        return __half22float2(h2);
    }
}

// SPLIT: the warps of a CTA share the rows of one unit and take turns along K; warp 0 adds their sums up.
template <int FMT, int N, int KL, int R, bool SPLIT>
__global__ void __launch_bounds__(32 * kGemvWarps) fp4_gemv_kernel(const Fp4GemvArgs a) {
    constexpr int G = R / 2;               // groups of 32 rows a unit takes its row pair from
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5, unit = SPLIT ? blockIdx.x : blockIdx.x * kGemvWarps + warp;
    constexpr int kStep = 32 * KL * (SPLIT ? kGemvWarps : 1);
    const int start = SPLIT ? warp * 32 * KL : 0;
    if (unit >= a.units) return;
    const int tile = unit / (64 / G), p = unit % 16, g0 = unit % (64 / G) / 16 * G;
    const int kt = fp4_ktiles(a.K, FMT);
    const int row0 = tile * 128 + g0 * 32 + 2 * p;       // row i of the unit: row0 + i / 2 * 32 + i % 2
    if (row0 >= a.M) return;
    // Rows past the end read the last one's codes, elements past the end the last ones' (under a vector of
    // zeros): no load depends on a condition. 32 bits hold 97 rows' offsets at the largest K.
    const uint32_t pitch = (uint32_t)a.K / 2;
    const uint8_t * base = a.W + (long long)row0 * pitch;
    uint32_t off[R];
#pragma unroll
    for (int i = 0; i < R; ++i) off[i] = (uint32_t)min(i / 2 * 32 + i % 2, a.M - 1 - row0) * pitch;
    const uint8_t * scales = a.Ws + fp4_scale_at(row0, 0, kt);
    const float dec = fp4_dec(a.W_amax);
    float acc[R * N] = {};
    uint32_t w[R][KL / 8], sc[2][G];
    const auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint8_t * c = base + (off[i] + (uint32_t)k / 2);
            if constexpr (KL == 16) {
                const uint2 t = __ldg(reinterpret_cast<const uint2 *>(c));
                w[i][0] = t.x;
                w[i][1] = t.y;
            } else {
                w[i][0] = __ldg(reinterpret_cast<const uint32_t *>(c));
            }
        }
        const int blk = k / fp4_block(FMT);
#pragma unroll
        for (int b = 0; b < 2; ++b) {      // words of the unit's groups: consecutive bytes of the scale tile
            const uint8_t * s = scales + (long long)(blk >> 2) * kScaleTile + 16 * b;
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
    };
    // Few rows: the codes and scales of the next elements are requested before these are used. Many rows have the
    // loads of other warps to hide theirs, and the registers are worth more as warps (6000 x 1536, N = 2 MX: 6.8 us, 7.6 with; N = 1
    // NV 5.0, 5.3).
    const auto at = [&](int k0) { return min(k0 + lane * KL, a.K - KL); };
    fetch(at(start));
    for (int k0 = start; k0 < a.K; k0 += kStep) {
        const bool live = k0 + lane * KL < a.K;
        const int k = at(k0), blk = k / fp4_block(FMT);
        float x[N][KL];
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
        uint32_t u[R][KL / 8], z[2][G];
        if (R > 2 && k0 > start) fetch(k);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < KL / 8; ++e) u[i][e] = w[i][e];
#pragma unroll
        for (int i = 0; i < G; ++i) { z[0][i] = sc[0][i]; z[1][i] = sc[1][i]; }
        if (R == 2 && k0 + kStep < a.K) fetch(at(k0 + kStep));
#pragma unroll
        for (int i = 0; i < R; i += 2) {
            const float2 s = scale_pair<FMT>(z[0][i / 2], z[1][i / 2], blk & 3);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float v[KL];
#pragma unroll
                for (int j = 0; j < KL / 8; ++j) fp4_values8(u[i + r][j], v + 8 * j);
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    float2 t = make_float2(0.f, 0.f);
#pragma unroll
                    for (int e = 0; e < KL; e += 2) t = fma2(make_float2(v[e], v[e + 1]), make_float2(x[n][e], x[n][e + 1]), t);
                    acc[(i + r) * N + n] = fmaf(t.x + t.y, r ? s.y : s.x, acc[(i + r) * N + n]);
                }
            }
        }
    }
    constexpr int V = R * N;
    lanes_sum<V>(acc, lane);
    if constexpr (SPLIT) {                 // in a fixed order
        __shared__ float part[kGemvWarps][32];
        part[warp][lane] = acc[0];
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int i = 1; i < kGemvWarps; ++i) acc[0] += part[i][lane];
    }
    const int i = lane / (32 / V) / N, n = lane / (32 / V) % N;
    const int m = row0 + i / 2 * 32 + i % 2;
    const bool mine = lane % (32 / V) == 0 && n < a.N && m < a.M, finite = fabsf(acc[0]) <= FLT_MAX;
    const auto put = [&](float t) {
        if (a.bias) t += __ldg(a.bias + m);
        if (a.silu) t = silu_f(t);
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.y)[n * a.ldy + m] = __float2bfloat16_rn(t);
        else static_cast<float *>(a.y)[n * a.ldy + m] = t;
    };
    if (mine && finite) put(acc[0] * dec);
    const unsigned lost = __ballot_sync(0xffffffffu, mine && !finite);
    if (lost) sum_again<FMT>(a, lost, m, n, dec, lane, put);
}

// ---------------------------------------------------------------------------------------------
// Three vectors and more, too long for fp4_gemv_tc.cu, on many rows: the same product on the warp-level tensor cores, where converting
// a code and scaling it are all that is left to do per weight, whatever the number of vectors.
//
// A CTA takes the 128 rows of a scale tile, a warp 16 of them as the 16 x 16 A operand of mma.m16n8k16
// (f16 -> f32). e2m1 codes, and codes times an e4m3 scale (at most 6 significant bits), are exact in
// f16. A vector enters as two columns of B, in f16 each: with x' = x * 2^p, the power chosen for each vector
// and 128 elements so that the largest |x'| lies in [2^14, 2^15), hi = f16(x') and lo = f16((x' - hi) * 2^12).
// hi + lo / 2^12 is x' to 2^-22 of its own size down to 2^-29 of the largest of the 128 (below that to
// 2^-51 of it), little beside the roundings of an f32 sum. So eight columns are four vectors; N > 4
// takes two tiles of columns.
// NV: scales are applied to the codes, sums run over 128 elements. MX (scales beyond f16's range):
// sums run over one block, so the four lanes that share a row turn their codes around to hold
// parts of the same block, and the block's scale is applied to its sum.
constexpr int kMmaWarps = 8, kChunk = 128;
template <int NT> constexpr int kSegChunks = 16 / NT;   // chunks of x staged at a time: 32 KB of B

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Eight codes as four f16 pairs.
__device__ __forceinline__ void fp4_halves8(uint32_t w, uint32_t (&h)[4]) {
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t half2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 4 x 4 words among the four lanes of a row: lane t's word b goes to lane b's word t.
__device__ __forceinline__ void turn4(uint32_t (&w)[4], int t) {
    // swap halves with the lane two away, then words with the lane next to it
    const bool h = t & 2, l = t & 1;
    const uint32_t g0 = __shfl_xor_sync(0xffffffffu, h ? w[0] : w[2], 2), g1 = __shfl_xor_sync(0xffffffffu, h ? w[1] : w[3], 2);
    if (h) { w[0] = g0; w[1] = g1; } else { w[2] = g0; w[3] = g1; }
    const uint32_t g2 = __shfl_xor_sync(0xffffffffu, l ? w[0] : w[1], 1), g3 = __shfl_xor_sync(0xffffffffu, l ? w[2] : w[3], 1);
    if (l) { w[0] = g2; w[2] = g3; } else { w[1] = g2; w[3] = g3; }
}

// CTAs to an SM: three keep up to four vectors fastest (60000 x 8192, N = 3: 110 us, with two 114); with eight, three would spill
// registers (19000 x 8192, N = 8: 87.8 us, with three 90).
template <int FMT, int NT>
__global__ void __launch_bounds__(32 * kMmaWarps, NT == 1 ? 3 : 2) fp4_gemv_mma_kernel(const Fp4GemvArgs a) {
    constexpr bool NV = FMT == TSD_FP4_NV;
    constexpr int SEG = kSegChunks<NT>, kDeep = 4;
    // B fragments: [chunk][column tile][pair of MMAs][lane] of 16 bytes; the powers of two to undo: [chunk][vector]
    __shared__ uint4 sb[SEG][NT][4][32];
    __shared__ float sf[SEG][4 * NT];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int kt = fp4_ktiles(a.K, FMT), chunks = (a.K + kChunk - 1) / kChunk;
    const float dec = fp4_dec(a.W_amax);
    // rows of this lane: i = g and g + 8 of the warp's 16, row i being 4 warp + i % 4 of group i / 4
    const int ra = blockIdx.x * 128 + 4 * warp + (g & 3) + 32 * (g >> 2), rb = ra + 64;
    const uint8_t * ca = a.W + (long long)ra * (a.K / 2) + t * 16, * cb = a.W + (long long)rb * (a.K / 2) + t * 16;
    const uint8_t * sa = a.Ws + fp4_scale_at(ra, 0, kt);         // rb's scales lie 8 bytes on
    float acc[NT][2] = {};
    for (int c0 = 0; c0 < chunks; c0 += SEG) {
        const int nc = min(SEG, chunks - c0);
        if (c0) __syncthreads();           // the segment before has been used
        for (int u = warp; u < nc * NT; u += kMmaWarps) {
            const int c = u / NT, tile = u % NT, n = 4 * tile + (g >> 1);
            const float * xr = a.x + n * a.ldx;
            float4 v[8];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // four elements for MMA i: of this lane's 32 (NV), of its part of block i / 2 (MX)
                const int k = (c0 + c) * kChunk + (NV ? t * 32 + i * 4 : (i >> 1) * 32 + t * 8 + (i & 1) * 4);
                v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (n < a.N && k < a.K) {
                    if (a.x_vec) v[i] = __ldg(reinterpret_cast<const float4 *>(xr + k));
                    else v[i] = make_float4(__ldg(xr + k), __ldg(xr + k + 1), __ldg(xr + k + 2), __ldg(xr + k + 3));
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t b = __float_as_uint(e[j]) & 0x7fffffffu;
                    m = max(m, b < 0x7f800000u ? b : 0u);
                }
            }
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const int up = min(268 - (int)(m >> 23), 253);   // exponent field of the power that brings the largest to 2^14
            const float p = __uint_as_float((uint32_t)up << 23);
            uint32_t h[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e[4] = {v[i].x * p, v[i].y * p, v[i].z * p, v[i].w * p};
                __half q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    q[j] = __float2half_rn(e[j]);
                    if (g & 1) {           // the low column; nothing is left of an infinity or a NaN
                        const float rest = (e[j] - __half2float(q[j])) * 4096.0f;
                        q[j] = __float2half_rn(fabsf(e[j]) <= FLT_MAX ? rest : 0.f);
                    }
                }
                h[2 * i] = __half_as_ushort(q[0]) | (uint32_t)__half_as_ushort(q[1]) << 16;
                h[2 * i + 1] = __half_as_ushort(q[2]) | (uint32_t)__half_as_ushort(q[3]) << 16;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sb[c][tile][i][lane] = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
            if (t == 0 && !(g & 1)) sf[c][n] = __uint_as_float((uint32_t)(254 - up) << 23);
        }
        __syncthreads();
        for (int c = 0; c < nc; c += kDeep) {
            uint4 wa[kDeep], wb[kDeep];
            uint32_t za[kDeep], zb[kDeep];
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                const int k = (c0 + c + d) * kChunk;
                const bool live = c + d < nc && k + t * 32 < a.K;
                wa[d] = wb[d] = make_uint4(0, 0, 0, 0);
                za[d] = zb[d] = 0;
                if (live && ra < a.M) wa[d] = __ldg(reinterpret_cast<const uint4 *>(ca + k / 2));
                if (live && rb < a.M) wb[d] = __ldg(reinterpret_cast<const uint4 *>(cb + k / 2));
                if constexpr (NV) {        // the two bytes of this lane's blocks
                    if (live) {
                        const uint8_t * s = sa + (k / 64 + (t >> 1)) * (long long)kScaleTile + (t & 1) * 2;
                        za[d] = __ldg(reinterpret_cast<const uint16_t *>(s));
                        zb[d] = __ldg(reinterpret_cast<const uint16_t *>(s + 8));
                    }
                } else if (c + d < nc) {   // the four of the chunk
                    const uint8_t * s = sa + (k / 128) * (long long)kScaleTile;
                    za[d] = __ldg(reinterpret_cast<const uint32_t *>(s));
                    zb[d] = __ldg(reinterpret_cast<const uint32_t *>(s + 8));
                }
            }
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                if (c + d >= nc) break;
                uint32_t xa[4] = {wa[d].x, wa[d].y, wa[d].z, wa[d].w}, xb[4] = {wb[d].x, wb[d].y, wb[d].z, wb[d].w};
                uint32_t fa = 0, fb = 0;
                if constexpr (NV) {
                    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(fa) : "h"((uint16_t)za[d]));
                    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(fb) : "h"((uint16_t)zb[d]));
                } else {
                    turn4(xa, t);
                    turn4(xb, t);
                }
                float s[NT][4] = {};
#pragma unroll
                for (int w = 0; w < 4; ++w) {      // word w of the lane's codes: two MMAs
                    uint32_t ha[4], hb[4];
                    fp4_halves8(xa[w], ha);
                    fp4_halves8(xb[w], hb);
                    if constexpr (NV) {
                        const uint32_t qa = __byte_perm(fa, 0, w < 2 ? 0x1010 : 0x3232), qb = __byte_perm(fb, 0, w < 2 ? 0x1010 : 0x3232);
#pragma unroll
                        for (int e = 0; e < 4; ++e) { ha[e] = half2_mul(ha[e], qa); hb[e] = half2_mul(hb[e], qb); }
                    }
                    const uint32_t a0[4] = {ha[0], hb[0], ha[1], hb[1]}, a1[4] = {ha[2], hb[2], ha[3], hb[3]};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 b = sb[c + d][n][w][lane];
                        mma_f16(s[n], a0, b.x, b.y);
                        mma_f16(s[n], a1, b.z, b.w);
                        if constexpr (!NV) {       // one block is done
                            const float f = sf[c + d][4 * n + t];
                            const float ua = fp4_scale_value<FMT>(za[d] >> (8 * w) & 255u), ub = fp4_scale_value<FMT>(zb[d] >> (8 * w) & 255u);
                            acc[n][0] = fmaf(fmaf(s[n][1], 1.0f / 4096.0f, s[n][0]) * f, ua, acc[n][0]);
                            acc[n][1] = fmaf(fmaf(s[n][3], 1.0f / 4096.0f, s[n][2]) * f, ub, acc[n][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
                        }
                    }
                }
                if constexpr (NV) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float f = sf[c + d][4 * n + t];
                        acc[n][0] = fmaf(fmaf(s[n][1], 1.0f / 4096.0f, s[n][0]), f, acc[n][0]);
                        acc[n][1] = fmaf(fmaf(s[n][3], 1.0f / 4096.0f, s[n][2]), f, acc[n][1]);
                    }
                }
            }
        }
    }
    const auto put = [&](int m, int v, float y) {
        if (a.bias) y += __ldg(a.bias + m);
        if (a.silu) y = silu_f(y);
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.y)[v * a.ldy + m] = __float2bfloat16_rn(y);
        else static_cast<float *>(a.y)[v * a.ldy + m] = y;
    };
    unsigned lost = 0;                     // bit 2 n + i: acc[n][i] is not finite
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = i ? rb : ra, v = 4 * n + t;
            if (v < a.N && m < a.M) {
                if (fabsf(acc[n][i]) <= FLT_MAX) put(m, v, acc[n][i] * dec);
                else lost |= 1u << (2 * n + i);
            }
        }
    if (__any_sync(0xffffffffu, lost))
        for (int e = 0; e < 2 * NT; ++e) {
            const int m = e & 1 ? rb : ra, v = 4 * (e >> 1) + t;
            sum_again<FMT>(a, __ballot_sync(0xffffffffu, lost >> e & 1), m, v, dec, lane, [&](float y) { put(m, v, y); });
        }
}

template <int FMT, int N, int KL, int R> cudaError_t launch(Fp4GemvArgs & a, int sms, cudaStream_t st) {
    const long long units = (long long)((a.M + 127) / 128) * (128 / R);
    a.units = (int)units;
    // Few rows: the warps of a CTA share them (shared / a warp on its own, MX, us: 149 x 10080 N = 1 4.0 / 10.3, N = 8
    // 8.9 / 26.1; 1000 x 2080 N = 3 4.2 / 5.7; 2500 x 2592 N = 1 4.5 / 6.9, N = 8 13.6 / 16.5; 4000 x 1536 N = 1
    // 4.5 / 5.7, N = 3 6.6 / 7.0, but N = 8 12.2 / 9.7; 4000 x 768 N = 1 4.5 / 4.3, N = 8 8.1 / 5.9).
    if constexpr (R == 2)
        if (a.M <= 20 * sms || (N <= 4 && a.K >= 1536))
            return launch_pdl(fp4_gemv_kernel<FMT, N, KL, R, true>, dim3((unsigned)units), dim3(32 * kGemvWarps), 0, st, a);
    return launch_pdl(fp4_gemv_kernel<FMT, N, KL, R, false>, dim3((unsigned)((units + kGemvWarps - 1) / kGemvWarps)),
                      dim3(32 * kGemvWarps), 0, st, a);
}

template <int FMT> cudaError_t launch_fmt(Fp4GemvArgs & a, int sms, cudaStream_t st) {
    // What fp4_gemv_tc.cu does not take (rule below). Rows per warp: eight (four with more than four vectors) share the
    // vectors' loads, two make enough warps of a small matrix. MX, us at two / at more, K = 1536: N = 1, 2000 rows 3.9 / 4.8, 4608 rows 6.3 / 5.1; N = 2, 4608
    // rows 8.2 / 5.9; N = 3, 9400 rows 11.3 / 8.4; N = 8, 4608 rows 9.7 / 11.7, 9400 rows 17.9 / 13.2. Other lengths at 4000
    // rows: K = 512 N = 1 3.1 / 2.9, N = 2 4.1 / 3.1, N = 8 4.9 / 5.7; K = 4096 N = 1 7.6 / 10.4, N = 8 22.7 / 28.5; K = 12288 N = 1
    // 18.8 / 27.3, N = 8 61 / 80. Three vectors and more go to the tensor cores where 128 rows to a CTA leave one for every SM (on them / at more rows a warp, MX and
    // NV: 19000 x 4256 N = 8 61.8 / 76.2 and 48.6 / 73.2, 60000 x 8192 N = 3 138 / 200 and 109 / 167; 9400 x 1536 N = 3
    // 11.0 / 8.4, N = 8 16.7 / 13.2).
    const bool some = a.M >= 28 * sms, more = a.M >= 56 * sms, many = a.M >= 128 * sms;
    if (a.N <= 1) return some ? launch<FMT, 1, 16, 8>(a, sms, st) : launch<FMT, 1, 16, 2>(a, sms, st);
    if (a.N <= 2) return some ? launch<FMT, 2, 16, 8>(a, sms, st) : launch<FMT, 2, 16, 2>(a, sms, st);
    if (many) {
        const dim3 grid((a.M + 127) / 128), block(32 * kMmaWarps);
        return a.N <= 4 ? launch_pdl(fp4_gemv_mma_kernel<FMT, 1>, grid, block, 0, st, a)
                        : launch_pdl(fp4_gemv_mma_kernel<FMT, 2>, grid, block, 0, st, a);
    }
    if (a.N <= 4) return some ? launch<FMT, 4, 8, 8>(a, sms, st) : launch<FMT, 4, 8, 2>(a, sms, st);
    return more ? launch<FMT, 8, 8, 4>(a, sms, st) : launch<FMT, 8, 8, 2>(a, sms, st);
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
    // The tensor-core form pays from 56 rows to an SM on, for vectors of the models' widths (it / the kernels here, K = 1536, us, MX and NV): 4608 rows
    // N = 1 4.7 / 5.2 and 4.7 / 4.5, N = 2 6.1 / 5.8 and 6.0 / 5.7, N = 8 11.2 / 9.8 and 11.4 / 9.9; 9400 rows N = 1
    // 4.7 / 5.6 and 4.9 / 4.8, N = 2 5.9 / 6.2 and 6.1 / 6.1, N = 8 11.1 / 13.4 and 11.1 / 12.9; 129024 rows N = 1
    // 19.8 / 34.6 and 20.3 / 31.4, N = 8 29.3 / 82.6 and 30.0 / 63.5. Shorter vectors leave its stages empty and keep its start: K = 512,
    // MX, 9400 rows N = 1 3.8 / 3.1, N = 8 7.0 / 6.4, 19000 rows 4.1 / 4.9 and 8.4 / 8.9, 129024 rows 7.2 / 12.9 and
    // 18.7 / 28.3; K = 128, 19000 rows N = 1 4.0 / 4.6, N = 8 7.4 / 4.5, 129024 rows 6.6 / 12.8 and 16.3 / 13.7.
    // Vectors that do not fit in one launch of it: two launches pay from 128 rows to an SM on (two / the kernels here, MX and
    // NV: 9400 x 2080 N = 8 20.1 / 18.9 and 20.0 / 17.9, 19000 x 2080 N = 8 23.3 / 31.6 and 23.9 / 25.1, 19000 x 4256
    // N = 3 26.2 / 40.3 and 29.3 / 31.5, 19000 x 7168 N = 2 36.2 / 43.7 and 39.8 / 43.9), three or more do not (three,
    // 60000 x 7168 N = 3 123 / 122 and 135 / 96).
    const int group = fp4_gemv_tc_group(fmt, N, K), most = M >= 128 * (long long)sms ? 2 : M >= 56 * (long long)sms ? 1 : 0;
    const bool tc = group && N <= most * group;
    const cudaError_t e = tc                  ? fp4_gemv_tc(fmt, a, group, cur, sms, st)
                          : fmt == TSD_FP4_MX ? launch_fmt<TSD_FP4_MX>(a, sms, st)
                                              : launch_fmt<TSD_FP4_NV>(a, sms, st);
    return launch_status("tsd_op_fp4_gemv", e);
}
