// fp4_gemm.cu — product of two microscaled 4-bit tensors on the tensor cores (sm_100a); format:
// include/tsd_ops.h.
//
//   acc[n][m] = sum over blocks b of (sum_{k in b} cx[n][k] cw[m][k]) sx[n][b] sw[m][b]
//
// tcgen05.mma.kind::mxf4nvf4 takes both operands' e2m1 codes from shared memory and their block scales
// from tensor memory, multiplies exactly and accumulates in f32. Tokens are the rows of a tile
// (tensor-memory lanes), features its columns, so a thread of the epilogue holds consecutive
// features of one token: bias, SwiGLU pairs (w1 / w3 rows alternate) and stores need no exchange
// between threads.
//
// Persistent CTAs, one per SM, walk tiles of 128 tokens x BN features, or as CTA pairs
// (cta_group::2) of 256 tokens x 256 features: each CTA loads its 128 tokens and half of the
// features, so an SM takes 38 KB in for 512 cycles of MMAs instead of 36 KB for 256 (128 x 128).
// A stage holds 256 elements of K: 128-byte rows of codes of both operands (TMA, 128-byte swizzle)
// and their tiles of scales, which lie in memory as the tensor cores want them (TMA too); rows and
// K past the end read as zero. Warps 0 / 2 / 3 issue the X codes / W codes / scales; warp 1 copies a
// stage's scales to tensor memory (each stage has its own columns, free again when the stage is)
// and issues its MMAs. Warps 4-11 are the epilogue: a warp takes 32 tokens and half of the
// columns into registers in one go, which frees the accumulator, and then finishes them 64 bytes of
// a row at a time through its own staging buffers and TMA stores (or plain stores where the
// output is not aligned to 16 bytes).
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "op_check.h"

#include <atomic>
#include <cstdio>

namespace tsd {

namespace {

struct Fp4GemmArgs {
    const float * W_amax, * X_amax, * bias;
    void * out;
    int * err;
    long long ldo;
    int M, N, K, swiglu, silu, bf16;
    int tma_out;       // TMA stores; else plain ones
    int bias_vec;      // bias is 16-byte aligned
    int mtiles, ntiles;
};

constexpr int kStageK = 256;               // elements of K per stage: one 128-byte row of codes
constexpr int kTN = 128;                   // tokens per CTA
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8, kEpiBuf = 32 * 64;   // epilogue staging: 32 rows x 64 bytes, two per warp
constexpr int kMaxDevices = 64;            // devices whose kernel attributes are remembered

template <int FMT, int BN, bool PAIR> struct Cfg {
    static constexpr int kSfTiles = kStageK / (4 * fp4_block(FMT));   // scale tiles per stage along K: 4 (NV) or 2 (MX)
    static constexpr int kWTiles = (BN + 127) / 128;                  // row tiles of W scales per stage
    static constexpr int kWRows = PAIR ? BN / 2 : BN;                 // W rows this CTA loads
    static constexpr int kA = kTN * 128, kB = kWRows * 128;
    static constexpr int kSA = kSfTiles * kScaleTile, kSB = kWTiles * kSA;
    static constexpr int kStage = kA + kB + kSA + kSB;
    static constexpr int kOut = kEpiWarps * 2 * kEpiBuf;
    static constexpr int kBars = 256;
    static constexpr int kFit = (227 * 1024 - 1024 - kBars - kOut) / kStage;
    static constexpr int kStages = kFit < 6 ? kFit : 6;
    static constexpr int kSmem = kStages * kStage + kOut + kBars + 1024;
    static constexpr int kAccs = BN <= 128 ? 2 : 1;                   // accumulators in tensor memory
    static constexpr int kSfCols = 4 * kSfTiles * (1 + kWTiles);      // tensor-memory columns of a stage's scales
    static_assert(kAccs * BN + kStages * kSfCols <= 512, "tensor memory");
    static_assert(kStage % 1024 == 0, "swizzle atoms");
    static_assert(!PAIR || BN == 256, "a pair's W scales are two whole row tiles");
};

// The W tile's features m0 + c .. + NC - 1 of one token (v: raw sums) -> finished values, 64 bytes of them.
template <int NC, int NE>
__device__ __forceinline__ void finish(const Fp4GemmArgs & a, float alpha, int m, const float * v, float (&o)[NE]) {
    if constexpr (NC == 2 * NE) {           // SwiGLU
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const float u = v[2 * i] * alpha;
            o[i] = (a.bf16 ? silu_fast(u) : silu_f(u)) * (v[2 * i + 1] * alpha);
        }
    } else {
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < NE; i += 4) {
                float4 b;
                if (a.bias_vec && m + i + 4 <= a.M) {
                    b = __ldg(reinterpret_cast<const float4 *>(a.bias + m + i));
                } else {
                    const int last = a.M - 1;
                    b = make_float4(__ldg(a.bias + min(m + i, last)), __ldg(a.bias + min(m + i + 1, last)),
                                    __ldg(a.bias + min(m + i + 2, last)), __ldg(a.bias + min(m + i + 3, last)));
                }
                o[i] = fmaf(v[i], alpha, b.x); o[i + 1] = fmaf(v[i + 1], alpha, b.y);
                o[i + 2] = fmaf(v[i + 2], alpha, b.z); o[i + 3] = fmaf(v[i + 3], alpha, b.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i) o[i] = v[i] * alpha;
        }
        if (a.silu) {
#pragma unroll
            for (int i = 0; i < NE; ++i) o[i] = a.bf16 ? silu_fast(o[i]) : silu_f(o[i]);
        }
    }
}

// NCOL raw sums of one token (features m0 ..) -> output, in pieces of 64 bytes a row. NC sums make
// one piece: 16 (f32) or 32 (bf16), twice that for SwiGLU.
template <int NCOL, int NC, int NE>
__device__ __forceinline__ void put_row(const Fp4GemmArgs & a, const CUtensorMap * tmO, uint8_t * buf, float alpha, int n0w,
                                        int lane, int m0, const float (&v)[NCOL], int & pieces) {
    constexpr int kDiv = NC / NE;           // 2 for SwiGLU
    const int cols = a.M / kDiv;            // columns of the output
#pragma unroll
    for (int c = 0; c < NCOL; c += NC) {
        if (m0 + c >= a.M) break;
        float o[NE];
        finish<NC, NE>(a, alpha, m0 + c, v + c, o);
        const int col = (m0 + c) / kDiv;
        if (a.tma_out) {
            uint8_t * dst = buf + (pieces & 1) * kEpiBuf;
            if (pieces >= 2) {              // the store issued two pieces ago has read this buffer
                if (lane == 0) bulk_wait_read<1>();
                __syncwarp();
            }
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if constexpr (NE == 32) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
                    p[i] = *reinterpret_cast<const uint32_t *>(&h);
                } else {
                    p[i] = __float_as_uint(o[i]);
                }
            }
            // 64-byte swizzle: 16-byte chunk j of row l at chunk j ^ ((l / 2) % 4)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4 *>(dst + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(tmO, dst, col, n0w);
                bulk_commit();
            }
            ++pieces;
        } else if (n0w + lane < a.N) {
            const long long at = (n0w + lane) * a.ldo + col;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                if (col + i >= cols) break;
                if constexpr (NE == 32) static_cast<__nv_bfloat16 *>(a.out)[at + i] = __float2bfloat16_rn(o[i]);
                else static_cast<float *>(a.out)[at + i] = o[i];
            }
        }
    }
}

template <int FMT, int BN, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                const __grid_constant__ CUtensorMap tmXs, const __grid_constant__ CUtensorMap tmWs,
                const __grid_constant__ CUtensorMap tmO, const Fp4GemmArgs a) {
    using C = Cfg<FMT, BN, PAIR>;
    constexpr int ST = C::kStages;
    constexpr int kCtas = PAIR ? 2 : 1;
    pdl_launch_dependents();   // let the next kernel in the stream start its prologue
    extern __shared__ uint8_t smem_raw[];
    uint8_t * smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t * outbuf = smem + ST * C::kStage;
    uint64_t * bars = reinterpret_cast<uint64_t *>(outbuf + C::kOut);
    uint64_t * full = bars;                    // [ST] the stage's copies (a pair: both CTAs', on the leader) have landed
    uint64_t * empty = bars + ST;              // [ST] its MMAs are done
    uint64_t * acc_full = bars + 2 * ST;       // [2]
    uint64_t * acc_empty = bars + 2 * ST + 2;  // [2] every epilogue thread (a pair: of both CTAs, on the leader)
    uint64_t * drained = bars + 2 * ST + 4;    // after a failed wait: no MMA in flight
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * ST + 5);
    volatile int * s_abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) { mbar_init(&full[s], 3); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], kCtas * kEpiWarps * 32); }
        mbar_init(drained, 1);
        *s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
        else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int nk = (a.K + kStageK - 1) / kStageK;
    const int tiles = a.mtiles * a.ntiles;
    const int first = blockIdx.x / kCtas, stride = gridDim.x / kCtas;
    pdl_wait();                // launched with PDL: the operands' writers have finished after this

    if (warp == 0 || warp == 2 || warp == 3) {
        // ---------------- producers: one thread each; a pair's leader arms the barrier for both CTAs ----------------
        if (lane == 0) {
            tma_prefetch(warp == 0 ? &tmX : warp == 2 ? &tmW : &tmXs);
            const uint32_t bytes = kCtas * (warp == 0 ? C::kA : warp == 2 ? C::kB : C::kSA + C::kSB);
            int it = 0;
            bool ok = true;
            for (int tile = first; ok && tile < tiles; tile += stride) {
                const int n0 = tile / a.mtiles * (kCtas * kTN) + rank * kTN, m0 = tile % a.mtiles * BN;
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % ST;
                    if (it >= ST && !mbar_wait(&empty[s], ((it / ST) & 1) ^ 1, s_abort, a.err, DEV_TIMEOUT_EMPTY)) {
                        ok = false;
                        break;
                    }
                    uint8_t * st = smem + s * C::kStage;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
                    if constexpr (PAIR) {
                        const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
                        if (warp == 0) {
                            tma_load_2d_pair(st, &tmX, bar, kb * 128, n0);
                        } else if (warp == 2) {
                            tma_load_2d_pair(st + C::kA, &tmW, bar, kb * 128, m0 + rank * C::kWRows);
                        } else {
                            tma_load_3d_pair(st + C::kA + C::kB, &tmXs, bar, 0, kb * C::kSfTiles, n0 / 128);
                            tma_load_3d_pair(st + C::kA + C::kB + C::kSA, &tmWs, bar, 0, kb * C::kSfTiles, m0 / 128);
                        }
                    } else if (warp == 0) {
                        tma_load_2d(st, &tmX, &full[s], kb * 128, n0);
                    } else if (warp == 2) {
                        tma_load_2d(st + C::kA, &tmW, &full[s], kb * 128, m0);
                    } else {
                        tma_load_3d(st + C::kA + C::kB, &tmXs, &full[s], 0, kb * C::kSfTiles, n0 / 128);
                        tma_load_3d(st + C::kA + C::kB + C::kSA, &tmWs, &full[s], 0, kb * C::kSfTiles, m0 / 128);
                    }
                }
            }
            if (!ok) {   // let the copies still in flight land before the CTA exits
                const int n_wait = it < ST ? it : ST;
                const unsigned long long t0 = globaltimer();
                for (int i = it - n_wait; i < it; ++i)
                    while (rank == 0 && !mbar_try_wait(&full[i % ST], (i / ST) & 1) && globaltimer() - t0 < wait_ns()) {}
                while (rank != 0 && globaltimer() - t0 < 1000000ull) {}   // its bytes are counted by the leader
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (a pair: the leader's) ----------------
        if (lane == 0 && rank == 0) {
            constexpr bool NV = FMT == TSD_FP4_NV;
            int it = 0, local = 0;
            bool ok = true;
            for (int tile = first; ok && tile < tiles; tile += stride, ++local) {
                const int b = local % C::kAccs, use = local / C::kAccs;
                if (use > 0 && !mbar_wait(&acc_empty[b], (use & 1) ^ 1, s_abort, a.err, DEV_TIMEOUT_ACC)) {
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
                    const uint32_t sa = tmem + C::kAccs * BN + s * C::kSfCols, sb = sa + 4 * C::kSfTiles;
#pragma unroll
                    for (int t = 0; t < C::kSfTiles; ++t) {
                        umma_copy_scales<PAIR>(sa + 4 * t, make_sdesc_scales(base + C::kA + C::kB + t * kScaleTile));
#pragma unroll
                        for (int r = 0; r < C::kWTiles; ++r)
                            umma_copy_scales<PAIR>(sb + 4 * (t * C::kWTiles + r),
                                                   make_sdesc_scales(base + C::kA + C::kB + C::kSA + r * C::kSA + t * kScaleTile));
                    }
                    const int steps = min(4, (a.K - kb * kStageK + 63) / 64);
                    const uint64_t ad = make_sdesc_sw128(base), bd = make_sdesc_sw128(base + C::kA);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (k >= steps) break;
                        const int t = NV ? k : k / 2;
                        umma_fp4_ss<NV, PAIR>(d, ad + 2 * k, bd + 2 * k, make_idesc_fp4(kCtas * kTN, BN, !NV, NV ? 0 : (k & 1) * 2),
                                              sa + 4 * t, sb + 4 * t * C::kWTiles + w_col, kb > 0 || k > 0);
                    }
                    if constexpr (PAIR) umma_commit_pair(&empty[s], 3);
                    else umma_commit(&empty[s]);
                }
                if (ok) {
                    if constexpr (PAIR) umma_commit_pair(&acc_full[b], 3);
                    else umma_commit(&acc_full[b]);
                }
            }
            if (!ok) {   // nothing may run on this CTA's memory once it is given back
                if constexpr (PAIR) umma_commit_pair(drained, 1);
                else umma_commit(drained);
                const unsigned long long t0 = globaltimer();
                while (!mbar_try_wait(drained, 0) && globaltimer() - t0 < wait_ns()) {}
            }
        }
    } else {
        // ---------------- epilogue (warps 4..11): thread = token, half of the tile's columns ----------------
        constexpr int kCols = BN / 2;
        const int q = warp & 3, half = (warp - 4) >> 2;
        uint8_t * buf = outbuf + (warp - 4) * 2 * kEpiBuf;
        const float alpha = fp4_dec(a.W_amax) * fp4_dec(a.X_amax);
        if (lane == 0 && a.tma_out) tma_prefetch(&tmO);
        int local = 0, pieces = 0;
        for (int tile = first; tile < tiles; tile += stride, ++local) {
            const int b = local % C::kAccs, use = local / C::kAccs;
            const int n0w = tile / a.mtiles * (kCtas * kTN) + rank * kTN + q * 32, m0 = tile % a.mtiles * BN + half * kCols;
            const bool ok = mbar_wait(&acc_full[b], use & 1, s_abort, a.err, DEV_TIMEOUT_ACC);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            float v[kCols];
            {
                uint32_t r[kCols / 32][32];
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c)
                    tmem_ld32_async(tmem + ((uint32_t)(q * 32) << 16) + b * BN + half * kCols + 32 * c, r[c]);
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    tmem_wait_ld(r[c]);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[32 * c + i] = __uint_as_float(r[c][i]);
                }
            }
            tc_fence_before();
            if constexpr (PAIR) mbar_arrive_remote(mapa_shared(smem_u32(&acc_empty[b]), 0));
            else mbar_arrive(&acc_empty[b]);
            if (n0w >= a.N || m0 >= a.M) continue;          // the whole warp
            if (a.bf16) {
                if (a.swiglu) {
                    if constexpr (kCols >= 64) put_row<kCols, 64, 32>(a, &tmO, buf, alpha, n0w, lane, m0, v, pieces);
                } else {
                    put_row<kCols, 32, 32>(a, &tmO, buf, alpha, n0w, lane, m0, v, pieces);
                }
            } else {
                if (a.swiglu) put_row<kCols, 32, 16>(a, &tmO, buf, alpha, n0w, lane, m0, v, pieces);
                else put_row<kCols, 16, 16>(a, &tmO, buf, alpha, n0w, lane, m0, v, pieces);
            }
        }
        if (lane == 0) bulk_wait<0>();          // the stores have left shared memory and arrived
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    // a pair's CTAs signal each other's barriers and share MMAs: neither leaves before both are done
    if constexpr (PAIR) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

template <int FMT, int BN, bool PAIR>
cudaError_t launch(const void * W, const void * Ws, const void * X, const void * Xs, Fp4GemmArgs & a, int dev, int sms,
                   cudaStream_t st) {
    using C = Cfg<FMT, BN, PAIR>;
    constexpr int kCtas = PAIR ? 2 : 1;
    const uint64_t kt = fp4_ktiles(a.K, FMT), row = a.K / 2;
    const uint64_t nt = (a.N + 127) / 128, mt = (a.M + 127) / 128;
    CUtensorMap tmX, tmW, tmXs, tmWs, tmO;
    const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const auto u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
    if (!make_tmap_2d(&tmX, X, u8, 1, row, a.N, row, 128, kTN) || !make_tmap_2d(&tmW, W, u8, 1, row, a.M, row, 128, C::kWRows) ||
        !make_tmap_3d(&tmXs, Xs, u32, 4, 128, kt, nt, kScaleTile, kt * kScaleTile, 128, C::kSfTiles, 1) ||
        !make_tmap_3d(&tmWs, Ws, u32, 4, 128, kt, mt, kScaleTile, kt * kScaleTile, 128, C::kSfTiles, C::kWTiles))
        return cudaErrorInvalidValue;
    const int es = a.bf16 ? 2 : 4;
    const uint64_t cols = a.swiglu ? a.M / 2 : a.M;
    a.tma_out = aligned(a.out, 16) && a.ldo * es % 16 == 0 &&
                make_tmap_2d(&tmO, a.out, a.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, es, cols,
                             a.N, a.ldo * es, 64 / es, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    if (!a.tma_out) tmO = tmX;   // not read
    static std::atomic<bool> attr_set[kMaxDevices];
    const bool known = dev < kMaxDevices;
    if (!known || !attr_set[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e =
            cudaFuncSetAttribute(fp4_gemm_kernel<FMT, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (known) attr_set[dev].store(true, std::memory_order_relaxed);
    }
    a.mtiles = (a.M + BN - 1) / BN;
    a.ntiles = (a.N + kCtas * kTN - 1) / (kCtas * kTN);
    const long long tiles = (long long)a.mtiles * a.ntiles;
    if (tiles > INT32_MAX - 65536) return cudaErrorInvalidValue;
    const int units = sms / kCtas;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles < units ? tiles : units) * kCtas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int na = 0;
    if (pdl_enabled()) {
        at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[na++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (PAIR) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim.x = 2;
        at[na].val.clusterDim.y = at[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = at;
    cfg.numAttrs = na;
    return cudaLaunchKernelEx(&cfg, fp4_gemm_kernel<FMT, BN, PAIR>, tmX, tmW, tmXs, tmWs, tmO, a);
}

template <int FMT>
cudaError_t launch_fmt(int form, const void * W, const void * Ws, const void * X, const void * Xs, Fp4GemmArgs & a, int dev,
                       int sms, cudaStream_t st) {
    if (form == 2) return launch<FMT, 256, true>(W, Ws, X, Xs, a, dev, sms, st);
    if (form == 1) return launch<FMT, 128, false>(W, Ws, X, Xs, a, dev, sms, st);
    return launch<FMT, 64, false>(W, Ws, X, Xs, a, dev, sms, st);
}

// Tile form: 2 CTA pairs (256 x 256), 1 128 x 128, 0 128 x 64. The time of a form is its waves of
// tiles times the K loop of a tile, which the operand bytes of a stage bound (38 / 36 / 28 KB).
int pick_form(int N, int M, bool no64, int sms) {
    const auto waves = [&](int tn, int tm, int units) {
        const long long t = (long long)((N + tn - 1) / tn) * ((M + tm - 1) / tm);
        return (double)((t + units - 1) / units);
    };
    const double t2 = waves(256, 256, sms / 2) * 38, t1 = waves(128, 128, sms) * 36, t0 = no64 ? 1e30 : waves(128, 64, sms) * 28;
    return t2 <= t1 && t2 <= t0 ? 2 : t1 <= t0 ? 1 : 0;
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
    a.W_amax = W_amax; a.X_amax = X_amax; a.bias = bias; a.out = out; a.ldo = ldo; a.err = err;
    a.M = M; a.N = N; a.K = K; a.swiglu = mode == TSD_EPI_SWIGLU; a.silu = act == TSD_ACT_SILU;
    a.bf16 = out_type == TSD_TYPE_BF16;
    a.bias_vec = aligned(bias, 16);
    int cur = 0, sms = 148;
    cudaGetDevice(&cur);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cur);
    const int form = pick_form(N, M, a.swiglu && a.bf16, sms);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = fmt == TSD_FP4_MX ? launch_fmt<TSD_FP4_MX>(form, W, W_scales, X, X_scales, a, cur, sms, st)
                                            : launch_fmt<TSD_FP4_NV>(form, W, W_scales, X, X_scales, a, cur, sms, st);
    if (e == cudaErrorInvalidValue) return TSD_ERR_ARG;
    if (e != cudaSuccess) {
        fprintf(stderr, "tsd_op_fp4_gemm: %s\n", cudaGetErrorString(e));
        return TSD_ERR_CUDA;
    }
    return TSD_OK;
}
