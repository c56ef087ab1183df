// fp4_gemv_tc.cu — microscaled 4-bit weights with many rows times a few f32 vectors on the tensor cores (sm_100a).
//
// The other forms (fp4_gemv.cu) turn every code into a float and are bound by those instructions. Here the
// codes go from memory to tcgen05.mma.kind::mxf4nvf4 as they are, and the vectors are written in digits that the
// same format holds. Within a block with largest magnitude below 2^(E+1), x is rounded to a multiple of
// 2^(E-44) and written to base 8 with digits -4 .. 3, all of them (halved) e2m1 values:
//
//   x = 2 sum_{j<16} c_j 8^-j 2^E,   c_j in {-2, -1.5, .. 1.5}
//
// (adding 4 (8^16 - 1) / 7 to the integer x 2^(45-E) turns its base-8 digits 0 .. 7 into these). So a vector is
// 16 rows of a 4-bit operand that share the scales 2^E, products are exact and summed in f32, and
// y = sum_j 8^-j (row j's sum). An element keeps 22 bits of its own down to 2^-23 of the largest of its block and
// is off by 2^-45 of that at most below. MX scales are 2^E itself (a vector whose largest lies beyond 2^+-64
// is scaled to about one first); NV scales hold 18 powers of two, so there E is at least the vector's
// largest less 17. (With MX a row's sum holds terms as large as 2^(E+2) |w| whatever the element: weights within
// 2^7 / 2^E of f32's end may overflow it.) Sums that are not finite, and vectors with an infinity or a NaN, which digits cannot
// hold, are multiplied again in f64.
//
// Vectors whose digits do not fit into shared memory together go in two groups, each a launch.
//
// Bound: the weight bytes. Persistent CTAs walk tiles of 128 rows. Each first writes the digits of all
// vectors into its shared memory (16 N K / 2 bytes and their scales), where they stay, while the first
// weights are on their way. Warp 0 loads codes (TMA, 512 elements of K a stage), warp 2 scales, warp 3 copies
// scales to tensor memory, warp 1 issues the MMAs (128 rows x 16 N digits), warps 4-7 add up the digits' sums
// (a thread has a row of W: no exchange) and store. 129024 x 1536: 19.8 us MX (5.4 TB/s), 20.3 NV (5.5 TB/s); eight
// vectors 29.3 / 30.0, of which writing their digits takes about 7.
#include "common.cuh"
#include "fp4.cuh"
#include "fp4_gemv.h"
#include "fp4_tc.cuh"
#include "kernels.h"

#include <atomic>
#include <cfloat>

namespace tsd {

namespace {

constexpr int kDigits = 16, kRows = 128, kStageK = 512, kThreads = 384;
constexpr int kMaxStages = 6, kMinStages = 3;
constexpr int kConverters = 256;                  // warps 4-11
constexpr int kMaxDevices = 64;
constexpr int kTail = 1024;                       // barriers and the vectors' factors

template <int FMT, int BN> struct Cfg {
    static constexpr int kSfTiles = kStageK / (4 * fp4_block(FMT)), kSteps = kStageK / 64;
    static constexpr int kAtomA = kRows * 128, kAtomB = BN * 128;
    static constexpr int kA = kStageK / kAtomK * kAtomA, kSA = kSfTiles * kScaleTile, kStage = kA + kSA;
    static constexpr int kCols = 4 * kSfTiles;    // tensor-memory columns of a stage's scales, of either operand
    static constexpr int kSlotFit = (512 - 2 * BN) / (2 * kCols);
    static_assert(kStage % 1024 == 0 && kAtomB % 1024 == 0, "swizzle atoms");
    static_assert(kSlotFit >= kMinStages, "the scales of a stage are written while those before it are multiplied");
    // Shared memory for the digits of vectors of K elements.
    static __host__ __device__ long long resident(int K) {
        return (long long)((K + kAtomK - 1) / kAtomK) * kAtomB + (long long)fp4_ktiles(K, FMT) * kScaleTile;
    }
    static __host__ int stages(int K) {
        const long long n = (227 * 1024 - 1024 - kTail - resident(K)) / kStage;
        return n < kMinStages ? 0 : n > kMaxStages ? kMaxStages : (int)n;
    }
};

// A position in a ring, and the parity of its current turn.
struct Place {
    int s = 0;
    uint32_t turn = 0;
    __device__ __forceinline__ void next(int n) {
        if (++s == n) { s = 0; turn ^= 1; }
    }
};

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// x[n][k .. k + 7], zeros past the end.
__device__ __forceinline__ void load8(const Fp4GemvArgs & a, int n, int k, bool live, float (&v)[8]) {
    const float * p = a.x + n * a.ldx + k;
    if (live && a.x_vec) {
        const float4 t = __ldg(reinterpret_cast<const float4 *>(p)), u = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        v[4] = u.x; v[5] = u.y; v[6] = u.z; v[7] = u.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = live ? __ldg(p + i) : 0.f;
    }
}
__device__ __forceinline__ unsigned max_bits(const float (&v)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// 8 x 8 nibbles: nibble p of word i -> nibble i of word p.
__device__ __forceinline__ void transpose8(uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = w[i], b = w[i + 4];
        w[i] = __byte_perm(a, b, 0x5410);
        w[i + 4] = __byte_perm(a, b, 0x7632);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (!(i & 2)) {
            const uint32_t a = w[i], b = w[i + 2];
            w[i] = __byte_perm(a, b, 0x6240);
            w[i + 2] = __byte_perm(a, b, 0x7351);
        }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t a = w[i], b = w[i + 1];
        w[i] = (a & 0x0f0f0f0fu) | (b << 4 & 0xf0f0f0f0u);
        w[i + 1] = (a >> 4 & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u);
    }
}

// The digits of all vectors, by warps 4-11 (thread t of them). exps[n]: the power of two the row sums of vector
// n are to be multiplied by, or kNotFinite.
constexpr int kNotFinite = 1 << 20;
template <int FMT, int BN>
__device__ __forceinline__ void write_digits(const Fp4GemvArgs & a, int t, uint8_t * digits, uint8_t * scales, unsigned * part, int * exps) {
    constexpr int kLanes = fp4_block(FMT) / 8;                     // lanes that share a block
    constexpr int kWarps = 8 * kDigits / BN;                       // warps that share a vector
    const int lane = t & 31, n = (t >> 5) / kWarps, first = ((t >> 5) % kWarps) * 32 + lane;
    const int chunks = (a.K + 63) / 64 * 8;                        // of eight elements: whole MMAs
    float next[8];
    load8(a, min(n, a.N - 1), first * 8, first * 8 < a.K, next);
    unsigned top = 0;
    if (n < a.N) {
        for (int c = first; c * 8 < a.K; c += 4 * 32 * kWarps) {   // four requests at a time
            float v[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) load8(a, n, (c + i * 32 * kWarps) * 8, (c + i * 32 * kWarps) * 8 < a.K, v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max_bits(v[i]));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (kWarps > 1 && lane == 0) part[t >> 5] = top;
    }
    if constexpr (kWarps > 1) {
        bar_sync(2, kConverters);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) top = max(top, part[n * kWarps + i]);
    }
    if (n >= a.N) return;
    const int V = max((int)(top >> 23), 1);                        // exponent field of the vector's largest
    const bool unit = FMT == TSD_FP4_NV || V < 127 - 64 || V > 127 + 64;
    if (first == 0) exps[n] = top >= 0x7f800000u ? kNotFinite : 1 + (FMT == TSD_FP4_NV ? V - 135 : unit ? V - 127 : 0);
    for (int c = first; c - lane < chunks; c += 32 * kWarps) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = next[i];
        load8(a, n, (c + 32 * kWarps) * 8, (c + 32 * kWarps) * 8 < a.K, next);
        unsigned m = max_bits(v);
#pragma unroll
        for (int o = 1; o < kLanes; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int E = max(max((int)(m >> 23), 1), V - (FMT == TSD_FP4_NV ? 17 : 100));
        // the scales of four blocks, collected by the 4 kLanes lanes that hold them, for the vector's 16 rows
        const int e8 = E - V + 8;
        uint32_t word = FMT == TSD_FP4_NV ? (uint32_t)(e8 >= -6 ? (e8 + 7) << 3 : 1 << (e8 + 9)) : (uint32_t)(unit ? E - V + 127 : E);
        word <<= 8 * (lane / kLanes & 3);
        word |= __shfl_xor_sync(0xffffffffu, word, kLanes);
        word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanes);
        if (c - lane % (4 * kLanes) < chunks) {
            uint8_t * sc = scales + c / (4 * kLanes) * kScaleTile + (n * kDigits >> 5) * 4 + (n * kDigits & 31) * 16;
#pragma unroll
            for (int i = 0; i < 16; i += 4 * kLanes) *reinterpret_cast<uint32_t *>(sc + (lane % (4 * kLanes) + i) * 16) = word;
        }
        if (c >= chunks) continue;
        // x = (h 2^24 + l) 2^(E - 172): h to nearest, then l of what is left, as integers in the low bits of sums with
        // 1.5 * 2^23 and (to a multiple of two) 1.5 * 2^24; nothing else rounds
        const float pre = E < 64 ? 1.8446744e19f : 1.0f, s1 = __int_as_float((127 + 148 - E - (E < 64 ? 64 : 0)) << 23);
        uint32_t lo[8], hi[8];                                     // digits 8-15 and 0-7
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = v[i] * pre, t = fmaf(x, s1, 12582912.0f);
            const float left = fmaf(x, s1, 12582912.0f - t);       // at most a half
            const int l = 2 * (__float_as_int(fmaf(left, 16777216.0f, 25165824.0f)) - 0x4bc00000) + 044444444;
            lo[i] = l & 0xffffff;
            hi[i] = __float_as_int(t) - 0x4b400000 + 044444444 + (l >> 24);
        }
        uint8_t * row = digits + (c >> 5) * (BN * 128) + n * kDigits * 128 + (c & 3) * 4;
        const int q16 = (c & 31) >> 2;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t u = hi[i];                                // three bits a digit, then four
                u += (u & 0xfff000u) * 15u;
                u += (u & 0x0fc00fc0u) * 3u;
                u += u & 0x38383838u;
                // digit u - 4 -> code: u - 4 or, negative, 8 | 4 - u
                const uint32_t pos = (u >> 2 & 0x11111111u) * 15u;
                w[i] = (pos & u & 0x33333333u) | (~pos & (0xccccccccu - u));
            }
            transpose8(w);
#pragma unroll
            for (int j = 0; j < 8; ++j) *reinterpret_cast<uint32_t *>(row + j * 128 + ((q16 ^ j) << 4)) = w[7 - j];
            row += 8 * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i) hi[i] = lo[i];
        }
    }
}

template <int FMT, int BN>
__global__ void __launch_bounds__(kThreads, 1)
fp4_gemv_tc_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmWs, const Fp4GemvArgs a, int ST) {
    using C = Cfg<FMT, BN>;
    constexpr bool NV = FMT == TSD_FP4_NV;
    pdl_launch_dependents();
    extern __shared__ uint8_t smem_raw[];
    uint8_t * smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int kt = fp4_ktiles(a.K, FMT);
    uint8_t * digits = smem + ST * C::kStage;
    uint8_t * xscales = digits + (a.K + kAtomK - 1) / kAtomK * C::kAtomB;
    uint64_t * full = reinterpret_cast<uint64_t *>(xscales + kt * kScaleTile);   // codes landed, scales in tensor memory
    uint64_t * sf_full = full + kMaxStages;           // scales landed
    uint64_t * empty = sf_full + kMaxStages;          // MMAs done
    uint64_t * acc_full = empty + kMaxStages;         // [2]
    uint64_t * acc_empty = acc_full + 2;              // [2] four epilogue warps
    uint64_t * drained = acc_empty + 2;               // after a wait that ran out: no MMA in flight
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int * s_abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    unsigned * part = reinterpret_cast<unsigned *>(tmem_slot + 2);   // [8] converters' maxima
    int * exps = reinterpret_cast<int *>(part + 8);                  // [8]
    volatile Progress * progress = reinterpret_cast<volatile Progress *>(exps + 8);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&sf_full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 4); }
        mbar_init(drained, 1);
        *s_abort = 0;
        progress->codes = progress->scales = progress->copied = -1;
        fence_mbar_init();
    }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int nk = (a.K + kStageK - 1) / kStageK, tiles = (a.M + kRows - 1) / kRows, slots = min(ST, C::kSlotFit);
    pdl_wait();

    if (warp == 0 || warp == 2) {
        // ---------------- producers ----------------
        const CUtensorMap * map = warp == 0 ? &tmW : &tmWs;
        if (elect_one()) tma_prefetch(map);
        uint64_t * landed = warp == 0 ? full : sf_full;
        int it = 0;
        Place ring;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x)
            for (int kb = 0; kb < nk; ++kb, ++it) {
                if (it >= ST && (warp_aborted(s_abort) ||
                                 !warp_wait(&empty[ring.s], ring.turn ^ 1, s_abort, nullptr, DEV_TIMEOUT_EMPTY))) {
                    ok = false;
                    break;
                }
                uint8_t * st = smem + ring.s * C::kStage;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&landed[ring.s], warp == 0 ? C::kA : C::kSA);
                    if (warp == 0) {
#pragma unroll
                        for (int i = 0; i < kStageK / kAtomK; ++i)
                            tma_load_2d(st + i * C::kAtomA, &tmW, &landed[ring.s], kb * (kStageK / 2) + i * 128, tile * kRows);
                    } else {
                        tma_load_3d(st + C::kA, &tmWs, &landed[ring.s], 0, kb * C::kSfTiles, tile);
                    }
                }
                __syncwarp();
                ring.next(ST);
            }
        if (lane == 0) *(warp == 0 ? &progress->codes : &progress->scales) = it;
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        constexpr uint32_t kIdesc[2] = {make_idesc_fp4(kRows, BN, !NV, 0), make_idesc_fp4(kRows, BN, !NV, NV ? 0 : 2)};
        const uint64_t ad0 = make_sdesc_sw128(smem_u32(smem)), bd0 = make_sdesc_sw128(smem_u32(digits));
        const int last_steps = (a.K - (nk - 1) * kStageK + 63) / 64;
        bar_sync(1, kConverters + 64);             // the digits are written
        Place ring, acc, last;
        int slot = 0;
        bool ok = true;
        for (int tile = blockIdx.x, local = 0; ok && tile < tiles; tile += gridDim.x, ++local) {
            if (local >= 2 && !warp_wait(&acc_empty[acc.s], acc.turn ^ 1, s_abort, nullptr, DEV_TIMEOUT_ACC)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t d = tmem + acc.s * BN;
            for (int kb = 0; kb < nk; ++kb) {
                if (!warp_wait(&full[ring.s], ring.turn, s_abort, nullptr, DEV_TIMEOUT_FULL)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t ad = ad0 + (uint32_t)(ring.s * (C::kStage / 16)), bd = bd0 + (uint32_t)(kb * (kStageK / kAtomK) * (C::kAtomB / 16));
                const uint32_t sa = tmem + 2 * BN + slot * (2 * C::kCols), sb = sa + C::kCols;
                const int steps = kb + 1 < nk ? C::kSteps : last_steps;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < C::kSteps; ++k)
                        if (k < steps) {
                            const int t = NV ? k : k / 2, i = k / 4;
                            umma_fp4_ss<NV, false>(d, ad + i * (C::kAtomA / 16) + 2 * (k & 3), bd + i * (C::kAtomB / 16) + 2 * (k & 3),
                                                   kIdesc[k & 1], sa + 4 * t, sb + 4 * t, k > 0 || kb > 0);
                        }
                    umma_commit(&empty[ring.s]);
                    if (kb + 1 == nk) umma_commit(&acc_full[acc.s]);
                }
                __syncwarp();
                ring.next(ST);
                if (++slot == slots) slot = 0;
            }
            last = acc;
            acc.next(2);
        }
        if (ok) drain_wait(&acc_full[last.s], last.turn, globaltimer());
        else wind_down<false>(drained, full, sf_full, ST, progress, 0, 0, s_abort);
    } else if (warp == 3) {
        // ---------------- scales to tensor memory ----------------
        const uint64_t ad0 = make_sdesc_scales(smem_u32(smem) + C::kA), bd0 = make_sdesc_scales(smem_u32(xscales));
        bar_sync(1, kConverters + 64);
        Place ring, freed;
        int slot = 0, filled = 0, copied = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x)
            for (int kb = 0; kb < nk; ++kb, ++copied) {
                ok = warp_wait(&sf_full[ring.s], ring.turn, s_abort, nullptr, DEV_TIMEOUT_FULL);
                if (ok && filled == slots) {          // the MMAs that read this slot before are done
                    ok = warp_wait(&empty[freed.s], freed.turn, s_abort, nullptr, DEV_TIMEOUT_EMPTY);
                    freed.next(ST);
                } else {
                    ++filled;
                }
                if (!ok) break;
                tc_fence_after();
                const uint64_t ad = ad0 + (uint32_t)(ring.s * (C::kStage / 16)), bd = bd0 + (uint32_t)(kb * C::kSfTiles * (kScaleTile / 16));
                const uint32_t sa = tmem + 2 * BN + slot * (2 * C::kCols), sb = sa + C::kCols;
                if (elect_one()) {
#pragma unroll
                    for (int t = 0; t < C::kSfTiles; ++t)
                        if (kb * C::kSfTiles + t < kt) {
                            umma_copy_scales<false>(sa + 4 * t, ad + t * (kScaleTile / 16));
                            umma_copy_scales<false>(sb + 4 * t, bd + t * (kScaleTile / 16));
                        }
                    umma_commit(&full[ring.s]);
                }
                __syncwarp();
                ring.next(ST);
                if (++slot == slots) slot = 0;
            }
        if (lane == 0) progress->copied = copied;
    } else {
        write_digits<FMT, BN>(a, threadIdx.x - 128, digits, xscales, part, exps);
        fence_proxy_async_smem();
        bar_sync(1, kConverters + 64);
        if (warp < 8) {
            // ---------------- epilogue: thread = row of W ----------------
            const int q = warp & 3;
            const double dec = fp4_dec(a.W_amax);
            Place acc;
            bool ok = true;                        // a wait that ran out leaves NaN in what is still to come
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, acc.next(2)) {
                const int m = tile * kRows + q * 32 + lane;
                const float bias = a.bias && m < a.M ? __ldg(a.bias + m) : 0.f;
                ok = ok && warp_wait(&acc_full[acc.s], acc.turn, s_abort, nullptr, DEV_TIMEOUT_ACC);
                float s[BN / kDigits];
                if (ok) {                          // else the accumulator may be another's by now, and is not given back
                    tc_fence_after();
#pragma unroll
                    for (int n = 0; n < BN / kDigits; ++n) {
                        float v[kDigits];
                        tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + acc.s * BN + n * kDigits, v);
                        s[n] = v[kDigits - 1];
#pragma unroll
                        for (int j = kDigits - 2; j >= 0; --j) s[n] = fmaf(s[n], 0.125f, v[j]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[acc.s]);
                }
                const auto put = [&](int n, float y) {
                    if (a.bias) y += bias;
                    if (a.silu) y = silu_f(y);
                    if (a.bf16) static_cast<__nv_bfloat16 *>(a.y)[n * a.ldy + m] = __float2bfloat16_rn(y);
                    else static_cast<float *>(a.y)[n * a.ldy + m] = y;
                };
                unsigned lost = 0;                 // bit n: vector n's sum is not finite, or the vector is not
#pragma unroll
                for (int n = 0; n < BN / kDigits; ++n)
                    if (n < a.N && m < a.M) {
                        // in f64: neither factor alone need keep an f32 in range
                        if (!ok) put(n, __int_as_float(0x7fffffff));
                        else if (exps[n] != kNotFinite && fabsf(s[n]) <= FLT_MAX)
                            put(n, (float)(s[n] * dec * __hiloint2double((exps[n] + 1023) << 20, 0)));
                        else lost |= 1u << n;
                    }
                if (__any_sync(0xffffffffu, lost))
                    for (int n = 0; n < a.N; ++n)
                        sum_again<FMT>(a, __ballot_sync(0xffffffffu, lost >> n & 1), m, n, dec, lane, [&](float y) { put(n, y); });
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int FMT, int BN> cudaError_t launch(const Fp4GemvArgs & a, int dev, int sms, cudaStream_t st) {
    using C = Cfg<FMT, BN>;
    const uint64_t kt = fp4_ktiles(a.K, FMT), row = a.K / 2, tiles = (a.M + kRows - 1) / kRows;
    CUtensorMap tmW, tmWs;
    if (!make_tmap_2d(&tmW, a.W, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, a.M, row, 128, kRows) ||
        !make_tmap_3d(&tmWs, a.Ws, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, 128, kt, tiles, kScaleTile, kt * kScaleTile, 128, C::kSfTiles, 1))
        return cudaErrorInvalidValue;
    const int stages = C::stages(a.K);
    const int smem = 1024 + stages * C::kStage + (int)C::resident(a.K) + kTail;
    static std::atomic<bool> attr_set[kMaxDevices];
    const bool known = dev < kMaxDevices;
    if (!known || !attr_set[dev].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(fp4_gemv_tc_kernel<FMT, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        if (known) attr_set[dev].store(true, std::memory_order_relaxed);
    }
    return launch_pdl(fp4_gemv_tc_kernel<FMT, BN>, dim3(tiles < (uint64_t)sms ? (unsigned)tiles : sms), dim3(kThreads), smem, st, tmW, tmWs, a, stages);
}

template <int FMT> cudaError_t launch_fmt(const Fp4GemvArgs & a, int dev, int sms, cudaStream_t st) {
    return a.N <= 1   ? launch<FMT, 16>(a, dev, sms, st)
           : a.N <= 2 ? launch<FMT, 32>(a, dev, sms, st)
           : a.N <= 4 ? launch<FMT, 64>(a, dev, sms, st)
                      : launch<FMT, 128>(a, dev, sms, st);
}
template <int FMT> int group_of(int N, int K) {
    return N > 4 && Cfg<FMT, 128>::stages(K)  ? 8
           : N > 2 && Cfg<FMT, 64>::stages(K) ? 4
           : N > 1 && Cfg<FMT, 32>::stages(K) ? 2
           : Cfg<FMT, 16>::stages(K)          ? 1
                                              : 0;
}

}  // namespace

int fp4_gemv_tc_group(int fmt, int N, int K) { return fmt == TSD_FP4_MX ? group_of<TSD_FP4_MX>(N, K) : group_of<TSD_FP4_NV>(N, K); }

cudaError_t fp4_gemv_tc(int fmt, const Fp4GemvArgs & all, int group, int dev, int sms, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    for (int n = 0; n < all.N && e == cudaSuccess; n += group) {
        Fp4GemvArgs a = all;
        a.x += n * a.ldx;
        a.y = static_cast<char *>(a.y) + n * a.ldy * (a.bf16 ? 2 : 4);
        a.N = all.N - n < group ? all.N - n : group;
        e = fmt == TSD_FP4_MX ? launch_fmt<TSD_FP4_MX>(a, dev, sms, st) : launch_fmt<TSD_FP4_NV>(a, dev, sms, st);
    }
    return e;
}

}  // namespace tsd
