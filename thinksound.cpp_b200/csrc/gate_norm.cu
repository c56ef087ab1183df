// gate_norm.cu — the boundary between two transformer blocks in one pass (sm_100a): norm of the
// block's output, gate and residual scales, and the norm and modulation that feed the next block.
//
//   b  = post(y) * post_gain                       post, pre: none, LayerNorm or RMS norm over the row
//   x' = x_scale * x + y_scale * (gate * b)
//   h  = (pre(x') * pre_gain) * (1 + scale) + shift
//
// With y absent x' is x_scale * x, so the call is then a plain norm + modulation. The reference
// does the parts as separate nodes (gate + residual src/mmdit.cpp:231,:234, norm + modulate
// :55-59,:218,:232); its blocks have no post-norm and no residual scales.
//
// Bound: memory. A row costs 4 H (x) + s_y H + 4 H (x') + s_h H bytes, and 4 H more for each of
// gate, scale and shift that is given per token; a few operations per element.
//
// One CTA holds one row: every thread keeps its elements of x' in registers from the first load to
// the last store, so nothing is read twice whichever norms are on. LayerNorm takes the mean first
// and then the sum of squared deviations (both over registers), so a row with a large mean loses
// nothing. Statistics, gate and residual are f32; x' is rounded only by being stored as f32 and the
// pre-norm reads the same f32 values, h is rounded once.
#include "common.cuh"
#include "kernels.h"
#include "op_check.h"
#include "../../include/tsd_ops.h"


namespace tsd {

namespace {

struct GateNormArgs {
    const float * x;
    const void * y;
    float * x_out;
    void * h;
    const float * post_gain, * pre_gain, * gate, * shift, * scale;
    long long ldx, ldy, ldxo, ldh, ldg, ld_mod;
    int H, rows, gate_div, mod_div;
    int y_type, h_type, post, pre;
    float post_eps, pre_eps, x_scale, y_scale;
};

// The threads that hold a row: T of them, this one t.
struct Team { int t, T; };

// Sum over a row's threads of one float each, in a fixed order: butterflies within the warps, then over
// the warps' sums (each warp on its own, so that one barrier does). red: 2 x 32 floats, used in turn.
__device__ __forceinline__ float row_sum(float v, Team team, float * red, int & turn) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int nw = team.T >> 5, lane = threadIdx.x & 31;
    if (nw == 1) return v;
    float * r = red + 32 * (turn++ & 1);   // the other half may still be read by a slower warp
    if (lane == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < nw ? r[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int V> __device__ __forceinline__ void load_f32(const float * p, float (&v)[V]) {
    if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
        v[0] = *p;
    }
}
template <int V> __device__ __forceinline__ void store_f32(float * p, const float (&v)[V]) {
    if constexpr (V == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *p = v[0];
}
__device__ __forceinline__ float from16(uint16_t u, bool bf16) {
    return bf16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}
__device__ __forceinline__ uint16_t to16(float v, bool bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
template <int V> __device__ __forceinline__ void load_16(const uint16_t * p, bool bf16, float (&v)[V]) {
    if constexpr (V == 4) {
        const ushort4 t = *reinterpret_cast<const ushort4 *>(p);
        v[0] = from16(t.x, bf16); v[1] = from16(t.y, bf16); v[2] = from16(t.z, bf16); v[3] = from16(t.w, bf16);
    } else {
        v[0] = from16(*p, bf16);
    }
}
template <int V> __device__ __forceinline__ void store_16(uint16_t * p, bool bf16, const float (&v)[V]) {
    if constexpr (V == 4)
        *reinterpret_cast<ushort4 *>(p) = make_ushort4(to16(v[0], bf16), to16(v[1], bf16), to16(v[2], bf16), to16(v[3], bf16));
    else *p = to16(v[0], bf16);
}

// Norm of the row held as v[S][V] (elements at or past H are zero and stay it), in place.
template <int V, int S>
__device__ __forceinline__ void row_norm(float (&v)[S][V], int kind, float eps, int H, float inv_H, Team team, float * red, int & turn) {
    if (kind == TSD_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[k][e];
        const float mean = row_sum(s, team, red, turn) / (float)H;   // exact for a row of one value
#pragma unroll
        for (int k = 0; k < S; ++k)
            if ((team.t + k * team.T) * V < H) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[k][e] -= mean;
            }
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) q = fmaf(v[k][e], v[k][e], q);
    const float r = __frsqrt_rn(fmaf(row_sum(q, team, red, turn), inv_H, eps));
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] *= r;
}

// A parameter's V elements from i on, or a constant where there is none.
template <int V> __device__ __forceinline__ void load_param(const float * p, int i, float none, float (&v)[V]) {
    if (p) {
        load_f32<V>(p + i, v);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = none;
    }
}

// One CTA per row, or (WARP) one warp; thread t of T holds V elements at (t + k T) * V for k < S. EARLY: the gate and
// the modulation are requested with x and y, before the first reduction (registers permitting).
template <int V, int S, int MAX, bool WARP, bool EARLY>
__global__ void __launch_bounds__(MAX) gate_norm_kernel(const GateNormArgs a) {
    __shared__ float red[64];
    const Team team = {WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x, WARP ? 32 : (int)blockDim.x};
    int turn = 0;
    pdl_launch_dependents();   // let the next kernel in the stream start its prologue
    pdl_wait();                // launched with PDL: the predecessor's writes are visible after this
    const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x, H = a.H;
    if (WARP && row >= a.rows) return;
    const float inv_H = 1.0f / (float)H;
    float v[S][V], b[S][V], g[EARLY ? S : 1][V], c[EARLY ? S : 1][V], d[EARLY ? S : 1][V];
    const float * xr = a.x + row * a.ldx;
    const float * gr = a.gate ? a.gate + (a.gate_div == 1 ? row : row / a.gate_div) * a.ldg : nullptr;
    const long long mrow = (a.mod_div == 1 ? row : row / a.mod_div) * a.ld_mod;
    const float * cr = a.scale ? a.scale + mrow : nullptr, * dr = a.shift ? a.shift + mrow : nullptr;
#pragma unroll
    for (int k = 0; k < S; ++k) {
        const int i = (team.t + k * team.T) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] = b[k][e] = 0.f;
        if (i < H) load_f32<V>(xr + i, v[k]);
    }
    if (a.y_type == TSD_TYPE_F32) {
        const float * yr = static_cast<const float *>(a.y) + row * a.ldy;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int i = (team.t + k * team.T) * V;
            if (a.y && i < H) load_f32<V>(yr + i, b[k]);
        }
    } else {
        const uint16_t * yr = static_cast<const uint16_t *>(a.y) + row * a.ldy;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int i = (team.t + k * team.T) * V;
            if (a.y && i < H) load_16<V>(yr + i, a.y_type == TSD_TYPE_BF16, b[k]);
        }
    }
    if constexpr (EARLY) {
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int i = (team.t + k * team.T) * V;
            if (i < H) {
                load_param<V>(gr, i, 1.f, g[k]);
                load_param<V>(cr, i, 0.f, c[k]);
                load_param<V>(dr, i, 0.f, d[k]);
            }
        }
    }
    if (a.y) {
        if (a.post != TSD_NORM_NONE) row_norm<V, S>(b, a.post, a.post_eps, H, inv_H, team, red, turn);
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int i = (team.t + k * team.T) * V;
            if (i < H) {
                float t[V];
                if (a.post_gain) {
                    load_f32<V>(a.post_gain + i, t);
#pragma unroll
                    for (int e = 0; e < V; ++e) b[k][e] *= t[e];
                }
                if constexpr (!EARLY) load_param<V>(gr, i, 1.f, g[0]);
#pragma unroll
                for (int e = 0; e < V; ++e) v[k][e] = fmaf(a.y_scale, b[k][e] * g[EARLY ? k : 0][e], a.x_scale * v[k][e]);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) v[k][e] *= a.x_scale;
    }
    if (a.x_out) {
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int i = (team.t + k * team.T) * V;
            if (i < H) store_f32<V>(a.x_out + row * a.ldxo + i, v[k]);
        }
    }
    if (!a.h) return;
    if (a.pre != TSD_NORM_NONE) row_norm<V, S>(v, a.pre, a.pre_eps, H, inv_H, team, red, turn);
#pragma unroll
    for (int k = 0; k < S; ++k) {
        const int i = (team.t + k * team.T) * V;
        if (i >= H) continue;
        if (a.pre_gain) {
            float t[V];
            load_f32<V>(a.pre_gain + i, t);
#pragma unroll
            for (int e = 0; e < V; ++e) v[k][e] *= t[e];
        }
        if constexpr (!EARLY) {
            load_param<V>(cr, i, 0.f, c[0]);
            load_param<V>(dr, i, 0.f, d[0]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] = fmaf(v[k][e], 1.0f + c[EARLY ? k : 0][e], d[EARLY ? k : 0][e]);
        if (a.h_type == TSD_TYPE_F32) store_f32<V>(static_cast<float *>(a.h) + row * a.ldh + i, v[k]);
        else store_16<V>(static_cast<uint16_t *>(a.h) + row * a.ldh + i, a.h_type == TSD_TYPE_BF16, v[k]);
    }
}

template <int V, int S, int MAX = 512> cudaError_t launch(const GateNormArgs & a, cudaStream_t st) {
    const int per = V * S;
    const int threads = ((a.H + per - 1) / per + 31) / 32 * 32;
    return launch_pdl(gate_norm_kernel<V, S, MAX, false, (S * V < 16)>, dim3(a.rows), dim3(threads), 0, st, a);
}
template <int V, int S> cudaError_t launch_warps(const GateNormArgs & a, cudaStream_t st) {
    return launch_pdl(gate_norm_kernel<V, S, 128, true, true>, dim3((unsigned)((a.rows + 3ll) / 4)), dim3(128), 0, st, a);
}

}  // namespace
}  // namespace tsd

using namespace tsd;

extern "C" int tsd_op_gate_norm(const float * x, int64_t ldx, const void * y, int y_type, int64_t ldy, int rows, int H,
                                int post_norm, const float * post_gain, float post_eps, const float * gate, int64_t ldg,
                                int gate_div, float x_scale, float y_scale, float * x_out, int64_t ldxo, int pre_norm,
                                const float * pre_gain, float pre_eps, const float * shift, const float * scale,
                                int64_t ld_mod, int mod_div, void * h, int h_type, int64_t ldh, void * stream) {
    if (rows < 0 || H < 1 || H > TSD_GATE_NORM_MAX_H || post_norm < 0 || post_norm > TSD_NORM_RMS || pre_norm < 0 ||
        pre_norm > TSD_NORM_RMS || gate_div < 1 || mod_div < 1 || !(post_eps >= 0.f) || !(pre_eps >= 0.f))
        return TSD_ERR_ARG;
    if (rows == 0) return TSD_OK;
    const int ys = float_size(y_type), hs = float_size(h_type);
    if (!x || (!x_out && !h) || ldx < H || (y && (!ys || ldy < H)) || (x_out && ldxo < H) || (h && (!hs || ldh < H)) ||
        (gate && ldg != 0 && ldg < H) || ((shift || scale) && ld_mod != 0 && ld_mod < H))
        return TSD_ERR_ARG;
    if (!y && (post_norm != TSD_NORM_NONE || post_gain || gate)) return TSD_ERR_ARG;
    if (!h && (pre_norm != TSD_NORM_NONE || pre_gain || shift || scale)) return TSD_ERR_ARG;
    // each row is read whole before it is written, so x_out may be x itself, row for row; nothing else may be shared
    if ((x_out == x && ldxo != ldx) || (h && (h == (const void *)x_out || h == (const void *)x || h == y)) ||
        (x_out && (const void *)x_out == y))
        return TSD_ERR_ARG;
    if (!aligned(x, 4) || !aligned(x_out, 4) || !aligned(post_gain, 4) || !aligned(pre_gain, 4) || !aligned(gate, 4) ||
        !aligned(shift, 4) || !aligned(scale, 4) || (y && !aligned(y, ys)) || (h && !aligned(h, hs)))
        return TSD_ERR_ARG;
    OperandDevice dev({x, y, post_gain, gate, x_out, pre_gain, shift, scale, h});
    if (dev.rc) return dev.rc;
    GateNormArgs a;
    a.x = x; a.y = y; a.x_out = x_out; a.h = h;
    a.post_gain = post_gain; a.pre_gain = pre_gain; a.gate = gate; a.shift = shift; a.scale = scale;
    a.ldx = ldx; a.ldy = ldy; a.ldxo = ldxo; a.ldh = ldh; a.ldg = ldg; a.ld_mod = ld_mod;
    a.H = H; a.rows = rows; a.gate_div = gate_div; a.mod_div = mod_div;
    a.y_type = y_type; a.h_type = h_type; a.post = post_norm; a.pre = pre_norm;
    a.post_eps = post_eps; a.pre_eps = pre_eps; a.x_scale = x_scale; a.y_scale = y_scale;
    // four elements to an access where every row starts on a boundary of four, else one
    const bool vec = H % 4 == 0 && ldx % 4 == 0 && aligned(x, 16) && (!y || (ldy % 4 == 0 && aligned(y, 4 * ys))) &&
                     (!x_out || (ldxo % 4 == 0 && aligned(x_out, 16))) && (!h || (ldh % 4 == 0 && aligned(h, 4 * hs))) &&
                     aligned(post_gain, 16) && aligned(pre_gain, 16) && aligned(gate, 16) && (!gate || ldg % 4 == 0) &&
                     aligned(shift, 16) && aligned(scale, 16) && (!(shift || scale) || ld_mod % 4 == 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    // Elements per thread: few rows are a matter of latency and take as many threads as a CTA may have; many
    // rows are a matter of instructions and bytes in flight, and 12 elements a thread serve both
    // (24832 x 1536: 175 us at 4 elements, 170 at 8, 166 at 12; 1 x 1536: 2.8 / 3.7 / 4.1 us, 388 x 1536:
    // 4.0 / 4.3 / 4.5 us). Many short rows go to a warp each (20008 x 16: 22 us with a CTA for each, 14 us; 11021 x 53:
    // 12.0, 8.0). Unaligned rows: up to 1024 threads (11 x 4734: 27 us at 32 elements a thread, 9.3 at 8).
    const bool many = rows >= 1024;
    if (vec) {
        e = many && H <= 384         ? launch_warps<4, 3>(a, st)
            : H > 8192               ? launch<4, 4, 1024>(a, st)
            : H > 6144               ? launch<4, 4>(a, st)
            : many || H > 4096       ? launch<4, 3>(a, st)
            : H > 2048               ? launch<4, 2>(a, st)
                                     : launch<4, 1>(a, st);
    } else {
        e = many && H <= 256 ? launch_warps<1, 8>(a, st)
            : H <= 1024      ? launch<1, 2>(a, st)
            : H <= 4096      ? launch<1, 4, 1024>(a, st)
            : H <= 8192      ? launch<1, 8, 1024>(a, st)
                             : launch<1, 16, 1024>(a, st);
    }
    return launch_status("tsd_op_gate_norm", e);
}
