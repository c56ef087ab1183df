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
// features. A stage holds 256 elements of K (single CTAs: 512, whose smaller tiles would otherwise
// spend more on a stage's waits than on its MMAs): 128-byte rows of codes of both operands (TMA, 128-byte
// swizzle) and their tiles of scales (TMA); rows and K past the end read as zero. Warp 0 loads
// the codes, warp 2 the scales, warp 3 copies a stage's scales to tensor memory, warp 1 issues the
// MMAs. Warps 4-11 are the epilogue: a warp takes 32 tokens and half of the columns into registers in
// one go, which frees the accumulator, finishes them and stores 32 bytes of a row at a time straight
// from registers, or, where another tile follows, 128 bytes of a row at a time through a staging
// buffer and TMA, so that it does not wait for memory to take them.
//
// What a stage costs is the latency of its steps more than its 512 cycles of MMAs; measured on 8192^3 (MX / NV):
//  - issue loops in a branch on the lane number (operands moved to uniform registers for every
//    tcgen05 instruction, ~100 cycles each) against whole-warp loops with elect_one: 286 / 313 -> 219 / 241 us;
//  - scale copies issued by the MMA warp, in order with the MMAs, against a warp of their own: 282 / 289 -> 218 / 229 us;
//  - four warps writing the scales with tcgen05.st instead of tcgen05.cp: 212 / 242 us (each re-reads
//    them from shared memory, whose bandwidth the MMAs need);
//  - a release at cluster scope on each arrival at the pair's leader: 565 / 638 us instead of 359 / 379.
// 256 features leave tensor memory for one accumulator only, so a tile's last MMAs wait for the
// registers of the epilogue; 192 features with two accumulators take as long per stage.
#include "common.cuh"
#include "fp4.cuh"
#include "fp4_tc.cuh"
#include "kernels.h"
#include "op_check.h"

#include <atomic>
#include <cfloat>

namespace tsd {

namespace {

struct Fp4GemmArgs {
    const float * W_amax, * X_amax, * bias;
    void * out;
    int * err;
    long long ldo;
    int M, N, K, swiglu, silu, bf16;
    int vec;           // bytes a store may have by the output's alignment: 32, 16 or one element
    int staged;        // output through staging buffers and TMA
    int mtiles, ntiles;
};

constexpr int kTN = 128;                   // tokens per CTA
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8, kOutBuf = 32 * 128;
constexpr int kMaxDevices = 64;            // devices whose kernel attributes are remembered

template <int FMT, int BN, bool PAIR> struct Cfg {
    static constexpr int kAtoms = PAIR ? 1 : 2;                       // 128-byte atoms of K per stage
    static constexpr int kStageK = kAtoms * kAtomK, kSteps = kStageK / 64;    // elements of K and MMAs per stage
    static constexpr int kSfTiles = kStageK / (4 * fp4_block(FMT));   // scale tiles per stage along K
    static constexpr int kWTiles = (BN + 127) / 128;                  // row tiles of W scales per stage
    static constexpr int kWRows = PAIR ? BN / 2 : BN;                 // W rows this CTA loads
    static constexpr int kAtomA = kTN * 128, kAtomB = kWRows * 128;
    static constexpr int kA = kAtoms * kAtomA, kB = kAtoms * kAtomB;
    static constexpr int kSA = kSfTiles * kScaleTile, kSB = kWTiles * kSA;
    static constexpr int kStage = kA + kB + kSA + kSB;
    static constexpr int kBars = 256;
    static constexpr int kEpi = PAIR ? kOutBuf : BN / 2 * 4;          // an epilogue warp's bias, then (pairs) its output
    static constexpr int kOut = kEpiWarps * kEpi;
    static constexpr int kFit = (227 * 1024 - 1024 - kBars - kOut) / kStage;
    static constexpr int kStages = kFit < 6 ? kFit : 6;
    static constexpr int kSmem = kStages * kStage + kBars + kOut + 1024;
    // Tensor-memory columns of a stage's scales: four to a tile (a copy writes whole, aligned fours)
    static constexpr int kACols = 4 * kSfTiles, kWCols = 4 * kWTiles * kSfTiles;
    static constexpr int kAccs = BN <= 128 ? 2 : 1;                   // accumulators in tensor memory
    static constexpr int kSlotFit = (512 - kAccs * BN) / (kACols + kWCols);
    static constexpr int kSlots = kSlotFit < kStages ? kSlotFit : kStages;     // stages whose scales tensor memory holds
    static_assert(kSlots >= 3, "the scales of a stage are written while the two before it are multiplied");
    static_assert(kStage % 1024 == 0, "swizzle atoms");
    static_assert(BN == 64 || BN % 128 == 0, "a tile starts on the first or third column of its scale tile");
};

// A position in a ring of N stages, and the parity of its current turn.
template <int N> struct Ring {
    int s = 0;
    uint32_t turn = 0;
    __device__ __forceinline__ void next() {
        if (++s == N) { s = 0; turn ^= 1; }
    }
};

// SiLU of a value that stays f32: expf in full, the division to two ulp (a result below 1.1e-36 in magnitude may
// come out as zero).
__device__ __forceinline__ float silu_f32(float x) { return __fdividef(x, 1.0f + expf(-x)); }

// Sums of one token, scaled and with their bias -> finished values, NE of them.
template <int NC, int NE>
__device__ __forceinline__ void finish(const Fp4GemmArgs & a, const float * v, float (&o)[NE]) {
    if constexpr (NC == 2 * NE) {           // SwiGLU
#pragma unroll
        for (int i = 0; i < NE; ++i) o[i] = (a.bf16 ? silu_fast(v[2 * i]) : silu_f32(v[2 * i])) * v[2 * i + 1];
    } else if (a.silu) {
#pragma unroll
        for (int i = 0; i < NE; ++i) o[i] = a.bf16 ? silu_fast(v[i]) : silu_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NE; ++i) o[i] = v[i];
    }
}

// 32 bytes of a row in one store: a whole sector of each of the 32 rows a warp holds.
__device__ __forceinline__ void store32(void * p, const uint32_t * v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// NCOL raw sums of token n (features m0 ..) -> output, in pieces of NE values of a row; NC sums make one
// piece: NE, or twice that for SwiGLU.
template <int NC, int NE, typename T>
__device__ __forceinline__ void make_piece(const Fp4GemmArgs & a, const float * v, uint32_t (&p)[NE * sizeof(T) / 4]) {
    float o[NE];
    finish<NC, NE>(a, v, o);
#pragma unroll
    for (int i = 0; i < NE * (int)sizeof(T) / 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            p[i] = __float_as_uint(o[i]);
        }
    }
}
// Straight from registers, 32 bytes at a time where the alignment allows it.
template <int NCOL, int NC, int NE, typename T>
__device__ __forceinline__ void put_row(const Fp4GemmArgs & a, int n, int m0, const float (&v)[NCOL]) {
    constexpr int kDiv = NC / NE, kWords = NE * (int)sizeof(T) / 4;
    if (n >= a.N) return;
#pragma unroll
    for (int c = 0; c < NCOL; c += NC) {
        const int left = (a.M - m0 - c) / kDiv;   // values of the row from here on
        if (left <= 0) break;
        uint32_t p[kWords];
        make_piece<NC, NE, T>(a, v + c, p);
        T * at = static_cast<T *>(a.out) + n * a.ldo + (m0 + c) / kDiv;
        if (left >= NE && a.vec == 32) {
#pragma unroll
            for (int j = 0; j < kWords; j += 8) store32(reinterpret_cast<uint32_t *>(at) + j, p + j);
        } else if (left >= NE && a.vec == 16) {
#pragma unroll
            for (int j = 0; j < kWords; j += 4)
                *(reinterpret_cast<uint4 *>(at) + j / 4) = make_uint4(p[j], p[j + 1], p[j + 2], p[j + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (i < left) {
                    if constexpr (sizeof(T) == 2) at[i] = __ushort_as_bfloat16((unsigned short)(p[i / 2] >> (16 * (i & 1))));
                    else at[i] = __uint_as_float(p[i]);
                }
        }
    }
}
// Rows that no 16-byte store may start on: eight lanes turn their eight values around, so that a store writes eight
// neighbours of each of four rows instead of one value of 32 (18360 x 1490 x 224 SwiGLU to bf16: 133 -> 40 us).
template <int NCOL, int DIV, typename T>
__device__ __forceinline__ void put_turned(const Fp4GemmArgs & a, int lane, int n0w, int m0, const float (&v)[NCOL]) {
#pragma unroll
    for (int c = 0; c < NCOL; c += 8 * DIV) {
        if (m0 + c >= a.M) break;
        float o[8];
        finish<8 * DIV, 8>(a, v + c, o);
#pragma unroll
        for (int s = 4; s >= 1; s /= 2) {
            const bool up = lane & s;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(i & s)) {
                    const float got = __shfl_xor_sync(0xffffffffu, up ? o[i] : o[i + s], s);
                    if (up) o[i] = got;
                    else o[i + s] = got;
                }
        }
        const int m = (m0 + c) / DIV + (lane & 7), n = n0w + (lane & 24);   // o[i]: of row n + i
        T * at = static_cast<T *>(a.out) + n * a.ldo + m;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (m < a.M / DIV && n + i < a.N) {
                if constexpr (sizeof(T) == 2) at[i * a.ldo] = __float2bfloat16_rn(o[i]);
                else at[i * a.ldo] = o[i];
            }
    }
}
// By TMA, 128 bytes of 32 rows at a time, through a staging buffer: the warp does not wait for
// memory to take the output. The map clips what lies past the end.
template <int NCOL, int NC, int NE, typename T>
__device__ __forceinline__ void put_rows_tma(const Fp4GemmArgs & a, const CUtensorMap * tmO, uint8_t * buf, int lane,
                                             int n0w, int m0, const float (&v)[NCOL]) {
    constexpr int kDiv = NC / NE;
    static_assert(NE * sizeof(T) == 128, "one swizzled row");
#pragma unroll
    for (int c = 0; c < NCOL; c += NC) {
        if (m0 + c >= a.M) break;
        uint32_t p[32];
        make_piece<NC, NE, T>(a, v + c, p);
        if (c > 0) {                               // the store before has read the buffer
            if (elect_one()) bulk_wait_read<0>();
            __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4 *>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {                         // the same lane for all of a warp's stores and waits
            tma_store_2d(tmO, buf, (m0 + c) / kDiv, n0w);
            bulk_commit();
        }
        __syncwarp();
    }
}

// After a wait for sums that ran out: NaN in an epilogue warp's part of this tile and of those to come, its 32 tokens and `cols`
// columns from m_off on of each tile of 128 tokens a CTA x tm.
__device__ __forceinline__ void put_nan(const Fp4GemmArgs & a, int tile, int tm, int ctas, int m_off, int cols) {
    const int div = a.swiglu ? 2 : 1, lane = threadIdx.x & 31;
    const int n_off = (int)(blockIdx.x % ctas) * kTN + (int)(threadIdx.x >> 5 & 3) * 32;
    for (; tile < a.mtiles * a.ntiles; tile += (int)gridDim.x / ctas) {
        const int n0 = tile / a.mtiles * (ctas * kTN) + n_off, m0 = tile % a.mtiles * tm + m_off;
        for (int i = 0; i < 32 && n0 + i < a.N; ++i)
            for (int c = lane; c < cols / div && m0 / div + c < a.M / div; c += 32) {
                const long long at = (n0 + i) * a.ldo + m0 / div + c;
                if (a.bf16) static_cast<uint16_t *>(a.out)[at] = 0x7fff;
                else static_cast<uint32_t *>(a.out)[at] = 0x7fffffff;
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
    // [ST] the stage's codes have landed and its scales are in tensor memory (a pair: both CTAs', on the leader)
    uint64_t * full = bars;
    uint64_t * sf_full = bars + ST;            // [ST] its scales have landed (likewise)
    uint64_t * empty = bars + 2 * ST;          // [ST] its MMAs are done
    uint64_t * acc_full = bars + 3 * ST;       // [2]
    uint64_t * acc_empty = acc_full + 2;       // [2] every epilogue warp (a pair: of both CTAs, on the leader)
    uint64_t * drained = acc_empty + 2;        // after a wait that ran out: no MMA in flight
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int * s_abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile float * factors = reinterpret_cast<volatile float *>(tmem_slot + 2);   // [2] what sums are multiplied by
    volatile Progress * progress = reinterpret_cast<volatile Progress *>(tmem_slot + 4);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp: uniform
    const uint32_t rank = PAIR ? cluster_ctarank() : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&sf_full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], kCtas * kEpiWarps); }
        mbar_init(drained, 1);
        *s_abort = 0;
        progress->codes = progress->scales = progress->copied = -1;
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
    const int nk = (a.K + C::kStageK - 1) / C::kStageK;
    const int tiles = a.mtiles * a.ntiles;
    const int first = blockIdx.x / kCtas, stride = gridDim.x / kCtas;
    pdl_wait();                // launched with PDL: the operands' writers have finished after this

    if (warp == 0 || warp == 2) {
        // ---------------- producers: one thread of a warp issues; a pair's leader arms the barriers for both CTAs ----------------
        if (elect_one()) {
            tma_prefetch(warp == 0 ? &tmX : &tmXs);
            tma_prefetch(warp == 0 ? &tmW : &tmWs);
        }
        int it = 0;                            // stages issued
        uint64_t * landed = warp == 0 ? full : sf_full;
        const uint32_t bytes = kCtas * (warp == 0 ? C::kA + C::kB : C::kSA + C::kSB);
        Ring<ST> ring;
        bool ok = true;
        for (int tile = first; ok && tile < tiles; tile += stride) {
            const int n0 = tile / a.mtiles * (kCtas * kTN) + rank * kTN, m0 = tile % a.mtiles * BN;
            const int m0w = m0 + (PAIR ? rank * C::kWRows : 0);
            for (int kb = 0; kb < nk; ++kb, ++it) {
                if (it >= ST && (warp_aborted(s_abort) ||
                                 !warp_wait(&empty[ring.s], ring.turn ^ 1, s_abort, a.err, DEV_TIMEOUT_EMPTY))) {
                    ok = false;
                    break;
                }
                uint8_t * st = smem + ring.s * C::kStage;
                if (elect_one()) {
                    if (rank == 0) mbar_arrive_expect_tx(&landed[ring.s], bytes);
                    if constexpr (PAIR) {
                        const uint32_t bar = mapa_shared(smem_u32(&landed[ring.s]), 0);
                        if (warp == 0) {
                            tma_load_2d_pair(st, &tmX, bar, kb * 128, n0);
                            tma_load_2d_pair(st + C::kA, &tmW, bar, kb * 128, m0w);
                        } else {
                            tma_load_3d_pair(st + C::kA + C::kB, &tmXs, bar, 0, kb * C::kSfTiles, n0 / 128);
                            tma_load_3d_pair(st + C::kA + C::kB + C::kSA, &tmWs, bar, 0, kb * C::kSfTiles, m0 / 128);
                        }
                    } else if (warp == 0) {
#pragma unroll
                        for (int i = 0; i < C::kAtoms; ++i) {
                            tma_load_2d(st + i * C::kAtomA, &tmX, &landed[ring.s], (kb * C::kAtoms + i) * 128, n0);
                            tma_load_2d(st + C::kA + i * C::kAtomB, &tmW, &landed[ring.s], (kb * C::kAtoms + i) * 128, m0w);
                        }
                    } else {
                        tma_load_3d(st + C::kA + C::kB, &tmXs, &landed[ring.s], 0, kb * C::kSfTiles, n0 / 128);
                        tma_load_3d(st + C::kA + C::kB + C::kSA, &tmWs, &landed[ring.s], 0, kb * C::kSfTiles, m0 / 128);
                    }
                }
                __syncwarp();
                ring.next();
            }
        }
        if (lane == 0) *(warp == 0 ? &progress->codes : &progress->scales) = it;
    } else if (warp == 1) {
        if (rank == 0) {
            // ---------------- MMA issuer (a pair: the leader's) ----------------
            // The warp's instructions bound the stage (wait, 4 MMAs, commit): no divisions, descriptors by
            // increments, and the whole warp in the loop (elect_one) so that they stay in uniform registers.
            constexpr bool NV = FMT == TSD_FP4_NV;
            constexpr uint32_t kIdesc[2] = {make_idesc_fp4(kCtas * kTN, BN, !NV, 0), make_idesc_fp4(kCtas * kTN, BN, !NV, NV ? 0 : 2)};
            const uint64_t ad0 = make_sdesc_sw128(smem_u32(smem)), bd0 = make_sdesc_sw128(smem_u32(smem) + C::kA);
            const int last_steps = (a.K - (nk - 1) * C::kStageK + 63) / 64;   // MMAs of a tile's last stage
            Ring<ST> ring;
            int slot = 0;
            Ring<C::kAccs> acc, last;          // this tile's accumulator, and the one before
            bool ok = true;
            for (int tile = first, local = 0; ok && tile < tiles; tile += stride, ++local) {
                if (local >= C::kAccs && !warp_wait(&acc_empty[acc.s], acc.turn ^ 1, s_abort, a.err, DEV_TIMEOUT_ACC)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc.s * BN;
                const uint32_t w_off = BN % 128 && tile % a.mtiles % 2 ? 2 : 0;   // an odd tile of 64: the upper half of its scale tile
                for (int kb = 0; kb < nk; ++kb) {
                    if (!warp_wait(&full[ring.s], ring.turn, s_abort, a.err, DEV_TIMEOUT_FULL)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = ad0 + (uint32_t)(ring.s * (C::kStage / 16)), bd = bd0 + (uint32_t)(ring.s * (C::kStage / 16));
                    const uint32_t sa = tmem + C::kAccs * BN + slot * (C::kACols + C::kWCols), sb = sa + C::kACols + w_off;
                    const auto step = [&](int k, uint32_t accumulate) {
                        const int t = NV ? k : k / 2;
                        const int i = k / 4;   // atom
                        umma_fp4_ss<NV, PAIR>(d, ad + i * (C::kAtomA / 16) + 2 * (k & 3), bd + i * (C::kAtomB / 16) + 2 * (k & 3), kIdesc[k & 1],
                                              sa + 4 * t, sb + 4 * C::kWTiles * t, accumulate);
                    };
                    if (elect_one()) {
                        step(0, kb > 0);
                        if (kb + 1 < nk || last_steps == C::kSteps) {
#pragma unroll
                            for (int k = 1; k < C::kSteps; ++k) step(k, 1);
                        } else {
#pragma unroll
                            for (int k = 1; k < C::kSteps - 1; ++k)
                                if (k < last_steps) step(k, 1);
                        }
                        if constexpr (PAIR) umma_commit_pair(&empty[ring.s], 3);
                        else umma_commit(&empty[ring.s]);
                        if (kb + 1 == nk) {
                            if constexpr (PAIR) umma_commit_pair(&acc_full[acc.s], 3);
                            else umma_commit(&acc_full[acc.s]);
                        }
                    }
                    __syncwarp();
                    ring.next();
                    if (++slot == C::kSlots) slot = 0;
                }
                last = acc;
                acc.next();
            }
            if (ok) drain_wait(&acc_full[last.s], last.turn, globaltimer());
            else wind_down<PAIR>(drained, full, sf_full, ST, progress, C::kA + C::kB, C::kSA + C::kSB, s_abort);
        }
    } else if (warp == 3) {
        // ---------------- scales to tensor memory (a pair: the leader's warp, for both CTAs) ----------------
        if (rank == 0) {
            const uint64_t sd0 = make_sdesc_scales(smem_u32(smem) + C::kA + C::kB);
            Ring<ST> ring, freed;              // this stage; the stage whose slot this one takes over
            int slot = 0, filled = 0, copied = 0;
            bool ok = true;
            for (int tile = first; ok && tile < tiles; tile += stride) {
                for (int kb = 0; kb < nk; ++kb, ++copied) {
                    ok = warp_wait(&sf_full[ring.s], ring.turn, s_abort, a.err, DEV_TIMEOUT_FULL);
                    if (ok && filled == C::kSlots) {      // the MMAs that read this slot before are done
                        ok = warp_wait(&empty[freed.s], freed.turn, s_abort, a.err, DEV_TIMEOUT_EMPTY);
                        freed.next();
                    } else {
                        ++filled;
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t sd = sd0 + (uint32_t)(ring.s * (C::kStage / 16));
                    const uint32_t sa = tmem + C::kAccs * BN + slot * (C::kACols + C::kWCols), sb = sa + C::kACols;
                    if (elect_one()) {
#pragma unroll
                        for (int t = 0; t < C::kSfTiles; ++t) umma_copy_scales<PAIR>(sa + 4 * t, sd + t * (kScaleTile / 16));
#pragma unroll
                        for (int t = 0; t < C::kSfTiles; ++t)
#pragma unroll
                            for (int r = 0; r < C::kWTiles; ++r)
                                umma_copy_scales<PAIR>(sb + 4 * (t * C::kWTiles + r), sd + C::kSA / 16 + r * (C::kSA / 16) + t * (kScaleTile / 16));
                        if constexpr (PAIR) umma_commit_pair(&full[ring.s], 1);
                        else umma_commit(&full[ring.s]);
                    }
                    __syncwarp();
                    ring.next();
                    if (++slot == C::kSlots) slot = 0;
                }
            }
            if (lane == 0) progress->copied = copied;
        }
    } else {
        // ---------------- epilogue (warps 4..11): thread = token, half of the tile's columns ----------------
        constexpr int kCols = BN / 2;
        const int q = warp & 3, half = (warp - 4) >> 2;
        // The tensors' factors in one where an f32 holds their product, else one after the other: a sum is at least 2^-20 and
        // far below 2^64, so the first step leaves f32's normal range only where the second ends beyond it too. They wait in
        // shared memory (every warp writes the same): the registers are full of sums.
        {
            const float dec_w = fp4_dec(a.W_amax), dec_x = fp4_dec(a.X_amax), both = dec_w * dec_x;
            const bool apart = !(both >= FLT_MIN && both <= FLT_MAX);
            if (lane == 0) { factors[0] = apart ? dec_w : 1.0f; factors[1] = apart ? dec_x : both; }
            __syncwarp();
        }
        Ring<C::kAccs> acc;
        int tile = first;
        for (; tile < tiles; tile += stride, acc.next()) {
            const int n0w = tile / a.mtiles * (kCtas * kTN) + rank * kTN + q * 32, m0 = tile % a.mtiles * BN + half * kCols;
            // the tile's bias is on its way while the MMAs run
            float bias[kCols / 32];
            if (a.bias) {
                const float * p = a.bias + m0 + lane * (kCols / 32);
                const int left = a.M - m0 - lane * (kCols / 32);
#pragma unroll
                for (int i = 0; i < kCols / 32; ++i) bias[i] = i < left ? __ldg(p + i) : 0.f;
            }
            if (!warp_wait(&acc_full[acc.s], acc.turn, s_abort, a.err, DEV_TIMEOUT_ACC)) break;
            tc_fence_after();
            float v[kCols];
            {
                uint32_t r[kCols / 32][32];
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c)
                    tmem_ld32_async(tmem + ((uint32_t)(q * 32) << 16) + acc.s * BN + half * kCols + 32 * c, r[c]);
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    tmem_wait_ld(r[c]);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[32 * c + i] = __uint_as_float(r[c][i]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_remote_tmem(mapa_shared(smem_u32(&acc_empty[acc.s]), 0));
                else mbar_arrive(&acc_empty[acc.s]);
            }
            if (n0w >= a.N || m0 >= a.M) continue;          // the whole warp
            const int n = n0w + lane;
            uint8_t * buf = outbuf + (warp - 4) * C::kEpi;
            if (PAIR && a.staged) {                         // the last tile's store has read the buffer
                if (elect_one()) bulk_wait_read<0>();
                __syncwarp();
            }
            if (factors[0] != 1.0f) {
                const float first = factors[0];
#pragma unroll
                for (int i = 0; i < kCols; ++i) v[i] *= first;
            }
            const float alpha = factors[1];
            if (a.bias) {
                float * w = reinterpret_cast<float *>(buf);
#pragma unroll
                for (int i = 0; i < kCols / 32; ++i) w[lane * (kCols / 32) + i] = bias[i];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kCols; i += 4) {
                    const float4 t = *reinterpret_cast<const float4 *>(w + i);
                    v[i] = fmaf(v[i], alpha, t.x); v[i + 1] = fmaf(v[i + 1], alpha, t.y);
                    v[i + 2] = fmaf(v[i + 2], alpha, t.z); v[i + 3] = fmaf(v[i + 3], alpha, t.w);
                }
                __syncwarp();
            } else {
#pragma unroll
                for (int i = 0; i < kCols; ++i) v[i] *= alpha;
            }
            if constexpr (PAIR) {
                if (a.staged) {
                    if (a.bf16) {
                        if (a.swiglu) put_rows_tma<kCols, 128, 64, __nv_bfloat16>(a, &tmO, buf, lane, n0w, m0, v);
                        else put_rows_tma<kCols, 64, 64, __nv_bfloat16>(a, &tmO, buf, lane, n0w, m0, v);
                    } else {
                        if (a.swiglu) put_rows_tma<kCols, 64, 32, float>(a, &tmO, buf, lane, n0w, m0, v);
                        else put_rows_tma<kCols, 32, 32, float>(a, &tmO, buf, lane, n0w, m0, v);
                    }
                    continue;
                }
            }
            if (a.vec < 16) {
                if (a.bf16) {
                    if (a.swiglu) put_turned<kCols, 2, __nv_bfloat16>(a, lane, n0w, m0, v);
                    else put_turned<kCols, 1, __nv_bfloat16>(a, lane, n0w, m0, v);
                } else {
                    if (a.swiglu) put_turned<kCols, 2, float>(a, lane, n0w, m0, v);
                    else put_turned<kCols, 1, float>(a, lane, n0w, m0, v);
                }
                continue;
            }
            if (a.bf16) {
                if (a.swiglu) put_row<kCols, 32, 16, __nv_bfloat16>(a, n, m0, v);
                else put_row<kCols, 32, 32, __nv_bfloat16>(a, n, m0, v);
            } else {
                if (a.swiglu) put_row<kCols, 32, 16, float>(a, n, m0, v);
                else put_row<kCols, 16, 16, float>(a, n, m0, v);
            }
            __syncwarp();                                   // lanes past the last token rejoin
        }
        if (tile < tiles) put_nan(a, tile, BN, kCtas, half * kCols, kCols);
        if (PAIR && elect_one()) bulk_wait<0>();            // the stores have arrived
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
    a.mtiles = (a.M + BN - 1) / BN;
    a.ntiles = (a.N + kCtas * kTN - 1) / (kCtas * kTN);
    const long long tiles = (long long)a.mtiles * a.ntiles;
    if (tiles > INT32_MAX - 65536) return cudaErrorInvalidValue;
    const int units = sms / kCtas;
    // Staged stores pay where a pair goes on to another tile meanwhile (24832 x 8192 x 1536 with bias: 166 us straight
    // from registers, 146 staged); with one tile each they only come later (388 x 8192 x 1536: 7.5 against 8.1 us).
    a.staged = PAIR && a.vec >= 16 && tiles > units;
    const int es = a.bf16 ? 2 : 4;
    if (!a.staged) tmO = tmX;   // not read
    else if (!make_tmap_2d(&tmO, a.out, a.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, es,
                           a.swiglu ? a.M / 2 : a.M, a.N, a.ldo * es, 128 / es, 32))
        return cudaErrorInvalidValue;
    static std::atomic<bool> attr_set[kMaxDevices];
    const bool known = dev < kMaxDevices;
    if (!known || !attr_set[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e =
            cudaFuncSetAttribute(fp4_gemm_kernel<FMT, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (known) attr_set[dev].store(true, std::memory_order_relaxed);
    }
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
// tiles times the K loop of a tile, which a CTA's operand bytes bound (38 / 36 / 28 KB for 256 elements of K).
int pick_form(int N, int M, int sms) {
    const auto waves = [&](int tn, int tm, int units) {
        const long long t = (long long)((N + tn - 1) / tn) * ((M + tm - 1) / tm);
        return (double)((t + units - 1) / units);
    };
    const double t2 = waves(256, 256, sms / 2) * 38, t1 = waves(128, 128, sms) * 36, t0 = waves(128, 64, sms) * 28;
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
    const uintptr_t at = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * es);
    a.vec = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : es;
    int cur = 0, sms = 148;
    cudaGetDevice(&cur);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cur);
    const int form = pick_form(N, M, sms);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = fmt == TSD_FP4_MX ? launch_fmt<TSD_FP4_MX>(form, W, W_scales, X, X_scales, a, cur, sms, st)
                                            : launch_fmt<TSD_FP4_NV>(form, W, W_scales, X, X_scales, a, cur, sms, st);
    if (e == cudaErrorInvalidValue) return TSD_ERR_ARG;
    return launch_status("tsd_op_fp4_gemm", e);
}
