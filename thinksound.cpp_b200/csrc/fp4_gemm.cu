// fp4_gemm.cu — product of two microscaled 4-bit tensors on the tensor cores (sm_100a); format:
// include/tsd_ops.h.
//
//   acc[n][m] = sum over blocks b of (sum_{k in b} cx[n][k] cw[m][k]) sx[n][b] sw[m][b]
//
// tcgen05.mma.kind::mxf4nvf4 takes both operands' e2m1 codes from shared memory and their block scales
// from tensor memory, multiplies exactly and accumulates in f32. Tokens are the rows of a tile
// (128 tensor-memory lanes), features its columns, so a thread of the epilogue holds consecutive
// features of one token: bias, SwiGLU pairs (w1 / w3 rows alternate) and wide stores need no
// exchange between threads.
//
// Persistent CTAs, one per SM, walk 128-token x BN-feature tiles. A stage holds 256 elements of K:
// 128-byte rows of codes of both operands (TMA, 128-byte swizzle; rows and K past the end read as
// zero) and their tiles of scales (untiled bulk copies; the tiles lie in memory as the tensor
// cores want them). Issuing a copy costs its thread ~300 cycles, so codes and scales of either
// operand have a warp each (0 X codes, 6 W codes, 7 X scales, 8 W scales). Warp 1 copies a
// stage's scales to tensor memory (each stage has its own columns, which are free again when the
// stage is) and issues its MMAs; warps 2-5 drain one of two accumulators while the other fills.
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "op_check.h"

#include <atomic>
#include <cstdio>

namespace tsd {

namespace {

struct Fp4GemmArgs {
    const uint8_t * Ws, * Xs;
    const float * W_amax, * X_amax, * bias;
    void * out;
    int * err;
    long long ldo;
    int M, N, K, swiglu, silu, bf16;
    int vec;           // bytes of a store: 32, 16, or one element
    int mtiles, ntiles;
};

constexpr int kStageK = 256;               // elements of K per stage: one 128-byte row of codes
constexpr int kTN = 128;                   // tokens per tile
constexpr int kThreads = 288;
constexpr int kMaxDevices = 64;            // devices whose kernel attributes are remembered

template <int FMT, int BN> struct Cfg {
    static constexpr int kSfTiles = kStageK / (4 * fp4_block(FMT));   // scale tiles per stage along K: 4 (NV) or 2 (MX)
    static constexpr int kWTiles = (BN + 127) / 128;                  // row tiles of W scales per stage
    static constexpr int kA = kTN * 128, kB = BN * 128;
    static constexpr int kSA = kSfTiles * kScaleTile, kSB = kWTiles * kSA;
    static constexpr int kStage = kA + kB + kSA + kSB;
    static constexpr int kBars = 256;
    static constexpr int kStages = (227 * 1024 - 1024 - kBars) / kStage < 8 ? (227 * 1024 - 1024 - kBars) / kStage : 8;
    static constexpr int kSmem = kStages * kStage + kBars + 1024;
    static constexpr int kSfCols = 4 * kSfTiles * (1 + kWTiles);      // tensor-memory columns of a stage's scales
    static_assert(2 * BN + kStages * kSfCols <= 512, "tensor memory");
    static_assert(kStage % 1024 == 0, "swizzle atoms");
};

// One row segment of NE finished values (consecutive features of one token).
template <int NE> __device__ __forceinline__ void store_row(const Fp4GemmArgs & a, long long at, int left, const float (&v)[NE]) {
    if (a.bf16) {
        __nv_bfloat16 * o = static_cast<__nv_bfloat16 *>(a.out) + at;
        uint32_t p[NE / 2];
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        if (left >= NE && a.vec >= 16) {
#pragma unroll
            for (int i = 0; i < NE / 8; ++i)
                *reinterpret_cast<uint4 *>(o + 8 * i) = make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (i < left) o[i] = __ushort_as_bfloat16((unsigned short)(p[i / 2] >> (16 * (i & 1))));
        }
    } else {
        float * o = static_cast<float *>(a.out) + at;
        if (left >= NE && a.vec >= 16) {
#pragma unroll
            for (int i = 0; i < NE / 4; ++i)
                *reinterpret_cast<float4 *>(o + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (i < left) o[i] = v[i];
        }
    }
}

template <int FMT, int BN>
__global__ void __launch_bounds__(kThreads, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const Fp4GemmArgs a) {
    using C = Cfg<FMT, BN>;
    constexpr int ST = C::kStages;
    pdl_launch_dependents();   // let the next kernel in the stream start its prologue
    extern __shared__ uint8_t smem_raw[];
    uint8_t * smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t * bars = reinterpret_cast<uint64_t *>(smem + ST * C::kStage);
    uint64_t * full = bars;                    // [ST] a stage's four copies have landed
    uint64_t * empty = bars + ST;              // [ST] its MMAs are done
    uint64_t * acc_full = bars + 2 * ST;       // [2]
    uint64_t * acc_empty = bars + 2 * ST + 2;  // [2] 128 arrivals
    uint64_t * drained = bars + 2 * ST + 4;    // after a failed wait: no MMA in flight
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * ST + 5);
    volatile int * s_abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) { mbar_init(&full[s], 4); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 128); }
        mbar_init(drained, 1);
        *s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int nk = (a.K + kStageK - 1) / kStageK;
    const int kt = fp4_ktiles(a.K, FMT);
    const int tiles = a.mtiles * a.ntiles;
    pdl_wait();                // launched with PDL: the operands' writers have finished after this

    if (warp == 0 || warp >= 6) {
        // ---------------- producers: one thread of each warp, one operand part ----------------
        if (lane == 0) {
            if (warp == 0) tma_prefetch(&tmX);
            if (warp == 6) tma_prefetch(&tmW);
            int it = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                const int n0 = tile / a.mtiles * kTN, m0 = tile % a.mtiles * BN;
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % ST;
                    if (it >= ST && !mbar_wait(&empty[s], ((it / ST) & 1) ^ 1, s_abort, a.err, DEV_TIMEOUT_EMPTY)) {
                        ok = false;
                        break;
                    }
                    uint8_t * st = smem + s * C::kStage;
                    if (warp == 0) {
                        mbar_arrive_expect_tx(&full[s], C::kA);
                        tma_load_2d(st, &tmX, &full[s], kb * 128, n0);
                    } else if (warp == 6) {
                        mbar_arrive_expect_tx(&full[s], C::kB);
                        tma_load_2d(st + C::kA, &tmW, &full[s], kb * 128, m0);
                    } else {
                        // whole scale tiles along K; the stage's last ones may not exist
                        const int t0 = kb * C::kSfTiles;
                        const uint32_t bytes = (uint32_t)(kt - t0 < C::kSfTiles ? kt - t0 : C::kSfTiles) * kScaleTile;
                        if (warp == 7) {
                            mbar_arrive_expect_tx(&full[s], bytes);
                            bulk_load_g2s(st + C::kA + C::kB, a.Xs + ((long long)(n0 / 128) * kt + t0) * kScaleTile, bytes, &full[s]);
                        } else {
                            const int r0 = m0 / 128;
                            const int nr = min((a.M + 127) / 128 - r0, C::kWTiles);
                            mbar_arrive_expect_tx(&full[s], bytes * nr);
                            for (int r = 0; r < nr; ++r)
                                bulk_load_g2s(st + C::kA + C::kB + C::kSA + r * C::kSA,
                                              a.Ws + ((long long)(r0 + r) * kt + t0) * kScaleTile, bytes, &full[s]);
                        }
                    }
                }
            }
            if (!ok) {   // let the copies still in flight land before the CTA exits
                for (int i = it > ST ? it - ST : 0; i < it; ++i) {
                    const unsigned long long t0 = globaltimer();
                    while (!mbar_try_wait(&full[i % ST], (i / ST) & 1) && globaltimer() - t0 < wait_ns()) {}
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            constexpr bool NV = FMT == TSD_FP4_NV;
            int it = 0, local = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++local) {
                const int b = local & 1;
                if (local >= 2 && !mbar_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1, s_abort, a.err, DEV_TIMEOUT_ACC)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + b * BN;
                // with BN = 64 an odd tile's rows are the upper half of a scale tile: columns 2 and 3 of its four
                const uint32_t w_col = (tile % a.mtiles * BN % 128) / 32;
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % ST;
                    if (!mbar_wait(&full[s], (it / ST) & 1, s_abort, a.err, DEV_TIMEOUT_FULL)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t base = smem_u32(smem + s * C::kStage);
                    const uint32_t sa = tmem + 2 * BN + s * C::kSfCols, sb = sa + 4 * C::kSfTiles;
#pragma unroll
                    for (int t = 0; t < C::kSfTiles; ++t) {
                        umma_copy_scales(sa + 4 * t, make_sdesc_scales(base + C::kA + C::kB + t * kScaleTile));
#pragma unroll
                        for (int r = 0; r < C::kWTiles; ++r)
                            umma_copy_scales(sb + 4 * (t * C::kWTiles + r),
                                             make_sdesc_scales(base + C::kA + C::kB + C::kSA + r * C::kSA + t * kScaleTile));
                    }
                    const int steps = min(4, (a.K - kb * kStageK + 63) / 64);
                    const uint64_t ad = make_sdesc_sw128(base), bd = make_sdesc_sw128(base + C::kA);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (k >= steps) break;
                        const int t = NV ? k : k / 2;
                        umma_fp4_ss<NV>(d, ad + 2 * k, bd + 2 * k, make_idesc_fp4(kTN, BN, !NV, NV ? 0 : (k & 1) * 2), sa + 4 * t,
                                        sb + 4 * t * C::kWTiles + w_col, kb > 0 || k > 0);
                    }
                    umma_commit(&empty[s]);
                }
                if (ok) umma_commit(&acc_full[b]);
            }
            if (!ok) {   // nothing may run on this CTA's memory once it is given back
                umma_commit(drained);
                const unsigned long long t0 = globaltimer();
                while (!mbar_try_wait(drained, 0) && globaltimer() - t0 < wait_ns()) {}
            }
        }
    } else {
        // ---------------- epilogue (warps 2..5): thread = token ----------------
        const int q = warp & 3;
        const float alpha = fp4_dec(a.W_amax) * fp4_dec(a.X_amax);
        int local = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++local) {
            const int b = local & 1;
            const int n = tile / a.mtiles * kTN + q * 32 + lane, m0 = tile % a.mtiles * BN;
            const bool ok = mbar_wait(&acc_full[b], (local >> 1) & 1, s_abort, a.err, DEV_TIMEOUT_ACC);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                if (m0 + c >= a.M) break;
                __syncwarp();                                 // lanes past the last token rejoin
                float v[32];
                tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + b * BN + c, v);
                if (c + 32 >= BN || m0 + c + 32 >= a.M) {     // the accumulator is read: the next tile may have it
                    tc_fence_before();
                    mbar_arrive(&acc_empty[b]);
                }
                if (n >= a.N) continue;
                const int left = a.M - m0 - c;
                if (a.swiglu) {
                    float o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float u = v[2 * i] * alpha;
                        o[i] = (a.bf16 ? silu_fast(u) : silu_f(u)) * (v[2 * i + 1] * alpha);
                    }
                    store_row<16>(a, n * a.ldo + (m0 + c) / 2, left / 2, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        v[i] *= alpha;
                        if (a.bias && i < left) v[i] += __ldg(a.bias + m0 + c + i);
                        if (a.silu) v[i] = a.bf16 ? silu_fast(v[i]) : silu_f(v[i]);
                    }
                    store_row<32>(a, n * a.ldo + m0 + c, left, v);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int FMT, int BN>
cudaError_t launch(const void * W, const void * X, Fp4GemmArgs & a, int dev, int sms, cudaStream_t st) {
    using C = Cfg<FMT, BN>;
    CUtensorMap tmX, tmW;
    if (!make_tmap_2d(&tmX, X, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K / 2, a.N, a.K / 2, 128, kTN) ||
        !make_tmap_2d(&tmW, W, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K / 2, a.M, a.K / 2, 128, BN))
        return cudaErrorInvalidValue;
    static std::atomic<bool> attr_set[kMaxDevices];
    const bool known = dev < kMaxDevices;
    if (!known || !attr_set[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e =
            cudaFuncSetAttribute(fp4_gemm_kernel<FMT, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (known) attr_set[dev].store(true, std::memory_order_relaxed);
    }
    a.mtiles = (a.M + BN - 1) / BN;
    a.ntiles = (a.N + kTN - 1) / kTN;
    const long long tiles = (long long)a.mtiles * a.ntiles;
    if (tiles > INT32_MAX - 65536) return cudaErrorInvalidValue;
    return launch_pdl(fp4_gemm_kernel<FMT, BN>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(kThreads), C::kSmem, st, tmX, tmW, a);
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int tsd_op_fp4_gemm(const void * W, const void * W_scales, const float * W_amax, int M, const void * X,
                               const void * X_scales, const float * X_amax, int N, int K, int fmt, int mode, int act,
                               const float * bias, void * out, int out_type, int64_t ldo, int * err, void * stream) {
    const int es = float_size(out_type);
    if (tsd_fp4_scale_bytes(M, K, fmt) < 0 || tsd_fp4_scale_bytes(N, K, fmt) < 0 || M < 1 ||
        (mode != TSD_EPI_STORE && mode != TSD_EPI_SWIGLU) || (act != TSD_ACT_NONE && act != TSD_ACT_SILU) ||
        (mode == TSD_EPI_SWIGLU && (M % 2 || bias || act != TSD_ACT_NONE)) || (fmt == TSD_FP4_MX && (W_amax || X_amax)) ||
        (out_type != TSD_TYPE_F32 && out_type != TSD_TYPE_BF16) || ldo < (mode == TSD_EPI_SWIGLU ? M / 2 : M))
        return TSD_ERR_ARG;
    if (N == 0) return TSD_OK;
    if (!W || !W_scales || !X || !X_scales || !out || !aligned(W, 16) || !aligned(W_scales, 16) || !aligned(X, 16) ||
        !aligned(X_scales, 16) || !aligned(out, es) || !aligned(bias, 4) || !aligned(W_amax, 4) || !aligned(X_amax, 4) ||
        !aligned(err, 4))
        return TSD_ERR_ARG;
    OperandDevice od({W, W_scales, W_amax, X, X_scales, X_amax, bias, out, err});
    if (od.rc) return od.rc;
    Fp4GemmArgs a;
    a.Ws = static_cast<const uint8_t *>(W_scales); a.Xs = static_cast<const uint8_t *>(X_scales);
    a.W_amax = W_amax; a.X_amax = X_amax; a.bias = bias; a.out = out; a.ldo = ldo; a.err = err;
    a.M = M; a.N = N; a.K = K; a.swiglu = mode == TSD_EPI_SWIGLU; a.silu = act == TSD_ACT_SILU;
    a.bf16 = out_type == TSD_TYPE_BF16;
    const uintptr_t at = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * es);
    a.vec = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : es;
    int cur = 0, sms = 148;
    cudaGetDevice(&cur);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cur);
    const bool wide = (long long)((M + 127) / 128) * ((N + 127) / 128) >= sms;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (fmt == TSD_FP4_MX) e = wide ? launch<TSD_FP4_MX, 128>(W, X, a, cur, sms, st) : launch<TSD_FP4_MX, 64>(W, X, a, cur, sms, st);
    else e = wide ? launch<TSD_FP4_NV, 128>(W, X, a, cur, sms, st) : launch<TSD_FP4_NV, 64>(W, X, a, cur, sms, st);
    if (e == cudaErrorInvalidValue) return TSD_ERR_ARG;
    if (e != cudaSuccess) {
        fprintf(stderr, "tsd_op_fp4_gemm: %s\n", cudaGetErrorString(e));
        return TSD_ERR_CUDA;
    }
    return TSD_OK;
}
