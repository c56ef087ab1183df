"""The microscaled 4-bit operators (tsd_op_fp4_*): codes and scales byte for byte against a plain
implementation in 64 bits, products against 64-bit products of the values the bytes stand for,
and the refusals.

Tolerances. u = 2^-24 is half an f32 step. The products of two codes and their scales are exact, and a
sum of K of them in f32, in any order, is off by at most 2 K u sum|x w| (twice, for additions that
truncate); gemv's x enters with 24 bits, another u (for many rows as two f16 parts: 2^-22, 4 u). dec_W dec_X, its product with the sum and the bias
are single roundings; SiLU(v) = v / (1 + exp(-v)) has slope 1.1 at most and costs 8 u of its value in
f32 (exp and the division, a few ulp each), or 2^-20 where the result is rounded to bf16 afterwards.
A sum of K roundings of random sign is about sqrt(K) u, so the 2-norm of the error is also held to
8 sqrt(K) u of the norm of sum|x w|, far below the worst case."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tsd_b200 import tsd

DEV = "cuda:0"
U = 2.0 ** -24
MX, NV = tsd.FP4_MX, tsd.FP4_NV
BLOCK = {MX: 32, NV: 16}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m / 512 for m in range(8)] +
                [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)])


# ------------------------------------------------------------------------------------ plain implementation, numpy f64
def nearest(a, table):
    """Index of the nearest entry of an ascending table (ties to the even index, the last beyond the end)."""
    mid = (table[1:] + table[:-1]) / 2
    i = np.searchsorted(mid, a, side="left")
    tie = (i < len(mid)) & (a == mid[np.minimum(i, len(mid) - 1)])
    return np.where(tie & (i % 2 == 1), i + 1, i)


def tiles_of(b, rows, K, fmt):
    """Scale bytes [rows][nb] in their tiles."""
    nb = K // BLOCK[fmt]
    kt = -(-nb // 4)
    p = np.zeros((-(-rows // 128) * 128, kt * 4), np.uint8)
    p[:rows, :nb] = b
    return p.reshape(-1, 4, 32, kt, 4).transpose(0, 3, 2, 1, 4).reshape(-1)


def rows_of_tiles(t, rows, K, fmt):
    nb = K // BLOCK[fmt]
    kt = -(-nb // 4)
    return t.reshape(-1, kt, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(-1, kt * 4)[:rows, :nb]


def factors(amax):
    """(enc, dec) in f32."""
    a = np.float32(0 if amax is None else amax)
    if amax is None or not (a >= np.float32(2.0 ** -100)) or not np.isfinite(a):
        return np.float32(1), np.float32(1)
    return np.float32(2688) * (np.float32(1) / a), a / np.float32(2688)   # enc: the reciprocal, rounded, times 2688


def quantize(x, fmt, amax=None):
    """x f32 -> (codes [rows][K/2], scale tiles)."""
    rows, K = x.shape
    with np.errstate(all="ignore"):
        z = (x.astype(np.float32) * factors(amax)[0]).astype(np.float64).reshape(rows, -1, BLOCK[fmt])
        bad = ~np.isfinite(z).all(-1)
        top = np.where(bad, 0, np.abs(np.where(bad[..., None], 0, z)).max(-1))
        if fmt == MX:
            e = np.maximum(np.frexp(top)[1] - 1 - 2, -127)
            e = np.where(top > 0, e, -127)
            byte, s = (e + 127).astype(np.uint8), np.ldexp(1.0, e)
        else:
            byte = nearest(top / 6, E4M3).astype(np.uint8)
            s = E4M3[byte]
        q = np.where(s[..., None] > 0, np.abs(z) / np.where(s > 0, s, 1)[..., None], 0)
        code = nearest(q, GRID).astype(np.uint8)
        code |= np.where((s[..., None] > 0) & np.signbit(z), 8, 0).astype(np.uint8)
    byte = np.where(bad, 255 if fmt == MX else 0x7F, byte).astype(np.uint8)
    code = code.reshape(rows, K)
    return code[:, 0::2] | (code[:, 1::2] << 4), tiles_of(byte, rows, K, fmt), bad


def values(codes, tiles, fmt):
    """code * scale, f64."""
    rows, K = codes.shape[0], 2 * codes.shape[1]
    c = np.stack([codes & 15, codes >> 4], -1).reshape(rows, K)
    v = np.where(c & 8, -1, 1) * GRID[c & 7]
    b = rows_of_tiles(tiles, rows, K, fmt).astype(int)
    s = np.where(b == 255, np.nan, np.ldexp(1.0, b - 127)) if fmt == MX else np.append(E4M3, np.nan)[np.minimum(b, 127)]
    return v * np.repeat(s, BLOCK[fmt], axis=1)


def make4(x, fmt, amax=None):
    """A device 4-bit tensor of f32 numpy values, made by the plain implementation."""
    c, t, _ = quantize(x, fmt, amax)
    return torch.from_numpy(c).to(DEV), torch.from_numpy(t).to(DEV), values(c, t, fmt) * float(factors(amax)[1])


def amax_of(x):
    return torch.tensor([np.abs(x).max()], device=DEV)


def dev_quantize(x, fmt, amax=None, stream=0):
    rows, K = x.shape
    c = torch.full((rows, K // 2), 0xAA, device=DEV, dtype=torch.uint8)
    t = torch.full((tsd.fp4_scale_bytes(rows, K, fmt),), 0xAA, device=DEV, dtype=torch.uint8)
    tsd.op_fp4_quantize(x, fmt, c, t, amax=amax, stream=stream)
    return c, t


def dev_empty(rows, K):
    return (torch.empty(rows, K // 2, device=DEV, dtype=torch.uint8), torch.empty(tsd.fp4_scale_bytes(rows, K, MX), device=DEV, dtype=torch.uint8))


def spread(rng, rows, K):
    """Values over many magnitudes, with zeros of both signs and whole blocks of zeros."""
    x = (rng.standard_normal((rows, K)) * np.exp2(rng.uniform(-12, 12, (rows, 1)))).astype(np.float32)
    x[rng.random((rows, K)) < 0.05] = 0
    x[rng.random((rows, K)) < 0.05] *= -0.0
    x[rows // 2, : K // 2] = 0
    return x


# ------------------------------------------------------------------------------------ quantisation
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("src", list(DT))
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 64), (31, 96), (127, 160), (128, 256), (129, 2080), (400, 1536)])
def test_quantize_bytes(fmt, src, rows, K):
    x = spread(np.random.default_rng(rows * K), rows, K)
    xt = torch.from_numpy(x).to(DEV).clamp(-6e4, 6e4).to(DT[src])
    c, t = dev_quantize(xt, fmt)
    rc, rt, _ = quantize(xt.float().cpu().numpy(), fmt)
    assert np.array_equal(t.cpu().numpy(), rt)
    assert np.array_equal(c.cpu().numpy(), rc)


@pytest.mark.gpu
@pytest.mark.parametrize("amax", [1.0, 0.731, 2688.0, 1e-20, 1e25, 0.0, 2.0 ** -101, float("inf"), float("nan")])
def test_quantize_with_a_tensor_scale(amax):
    rng = np.random.default_rng(5)
    top = amax if np.isfinite(amax) and amax > 1e-30 else 1.0
    x = (rng.uniform(-1, 1, (70, 512)) * top).astype(np.float32)
    x[0, 0] = top
    a = torch.tensor([amax], device=DEV)
    c, t = dev_quantize(torch.from_numpy(x).to(DEV), NV, a)
    rc, rt, _ = quantize(x, NV, amax)
    assert np.array_equal(t.cpu().numpy(), rt) and np.array_equal(c.cpu().numpy(), rc)
    y = torch.empty(70, 512, device=DEV)
    tsd.op_fp4_dequantize(c, t, NV, y, amax=a)
    want = (values(rc, rt, NV).astype(np.float32) * factors(amax)[1])
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("amax", [2.0 ** 126, 1.7e38, 3.4e38])
def test_quantize_with_a_tensor_scale_at_the_end_of_the_range(amax):
    """Maxima whose reciprocal is subnormal (fewer bits, the same ones here, in the plain implementation and in torch)."""
    x = (np.random.default_rng(5).uniform(-1, 1, (70, 512)) * amax).astype(np.float32)
    x[0, 0] = amax
    a, xt = torch.tensor([amax], device=DEV), torch.from_numpy(x).to(DEV)
    c, t = dev_quantize(xt, NV, a)
    rc, rt, _ = quantize(x, NV, np.float32(amax))
    assert np.array_equal(t.cpu().numpy(), rt) and np.array_equal(c.cpu().numpy(), rc)
    c1, t1 = dev_quantize(xt * (2688.0 / a), NV)
    assert torch.equal(c, c1) and torch.equal(t, t1)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_quantize_next_to_every_border(fmt):
    """Elements at, one step above and one below each border between codes, under many scales; maxima at the
    borders between scales."""
    rng = np.random.default_rng(6)
    rows = []
    mids = (GRID[1:] + GRID[:-1]) / 2
    scales = E4M3[8:] if fmt == NV else np.exp2(np.arange(-126, 122, 3.0))
    for s in scales:
        at = np.concatenate([mids * s, -mids * s]).astype(np.float32)
        near = np.concatenate([at, np.nextafter(at, np.float32(0)), np.nextafter(at, np.float32(np.inf)), np.nextafter(at, np.float32(-np.inf))])
        for part in np.array_split(rng.permutation(near), -(-len(near) // (BLOCK[fmt] - 1))):
            b = np.zeros(BLOCK[fmt], np.float32)
            b[: len(part)] = part
            b[-1] = 6 * s                                       # fixes the scale
            rows.append(b)
    if fmt == NV:
        m = (((E4M3[1:] + E4M3[:-1]) / 2) * 6).astype(np.float32)
        for v in np.concatenate([m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(1e9)), [2687.9, 2688, 2689, 1e6, 1e38]]):
            b = (rng.uniform(-1, 1, BLOCK[fmt]) * v).astype(np.float32)
            b[3] = v
            rows.append(b)
    rows += [np.zeros(BLOCK[fmt], np.float32)] * (-len(rows) % 2)
    x = np.stack(rows).reshape(-1, 2 * BLOCK[fmt])
    if x.shape[1] % 32:
        x = x[: x.shape[0] // 2 * 2].reshape(-1, 32)
    c, t = dev_quantize(torch.from_numpy(x).to(DEV), fmt)
    rc, rt, _ = quantize(x, fmt)
    assert np.array_equal(t.cpu().numpy(), rt) and np.array_equal(c.cpu().numpy(), rc)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_quantize_extremes(fmt):
    x = np.zeros((12, 64), np.float32)
    x[0] = -0.0
    x[1, 0], x[1, 1] = 2.0 ** -149, -(2.0 ** -149)
    x[2, 5], x[2, 6] = 2.0 ** -126, -(2.0 ** -140)
    x[3, 0], x[3, 1] = 3.4e38, -1e30
    x[4, 40] = np.inf
    x[5, 2] = np.nan
    x[6] = np.linspace(-1, 1, 64)
    x[7, 0] = 2.0 ** -12
    x[8, 0], x[8, 1] = 2.0 ** -10 * 6, -(2.0 ** -11)
    x[9, 0], x[9, 1:8] = 7.9, 6.9
    x[10, 0], x[10, 17] = 448 * 6, -5e-39
    x[11, 0], x[11, 1:9] = 6, -(2.0 ** -149)
    c, t = dev_quantize(torch.from_numpy(x).to(DEV), fmt)
    rc, rt, bad = quantize(x, fmt)
    assert np.array_equal(t.cpu().numpy(), rt)
    ok = ~np.repeat(bad, BLOCK[fmt] // 2, axis=1)
    assert np.array_equal(c.cpu().numpy()[ok], rc[ok])
    y = torch.empty(12, 64, device=DEV)
    tsd.op_fp4_dequantize(c, t, fmt, y)
    want = values(rc, rt, fmt).astype(np.float32)
    got = y.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.repeat(bad, BLOCK[fmt], axis=1))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(got)])


@pytest.mark.gpu
@pytest.mark.parametrize("pad,off", [(16, 0), (3, 0), (8, 1), (7, 5)])
@pytest.mark.parametrize("src", list(DT))
def test_quantize_and_dequantize_strides(pad, off, src):
    """x and y in wider buffers at any alignment; nothing around y is written."""
    rows, K = 37, 224
    x = spread(np.random.default_rng(8), rows, K)
    buf = torch.zeros((rows + 1) * (K + pad), device=DEV, dtype=DT[src])
    v = buf[off:off + rows * (K + pad)].view(rows, K + pad)[:, :K]
    v.copy_(torch.from_numpy(x).clamp(-6e4, 6e4))
    for fmt in (MX, NV):
        c, t = dev_quantize(v, fmt)
        rc, rt, _ = quantize(v.float().cpu().numpy(), fmt)
        assert np.array_equal(t.cpu().numpy(), rt) and np.array_equal(c.cpu().numpy(), rc)
        out = torch.full_like(buf, 9.0)
        o = out[off:off + rows * (K + pad)].view(rows, K + pad)[:, :K]
        tsd.op_fp4_dequantize(c, t, fmt, o)
        want = torch.from_numpy(values(rc, rt, fmt).astype(np.float32)).to(DT[src])
        assert torch.equal(o.cpu(), want)
        o.fill_(9.0)
        assert (out == 9.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("src", list(DT))
@pytest.mark.parametrize("rows,K,pad,off", [(1, 1, 0, 0), (3, 7, 2, 1), (200, 1536, 0, 0), (5, 4099, 5, 3), (3000, 64, 8, 0)])
def test_absmax(src, rows, K, pad, off):
    g = torch.Generator(device=DEV).manual_seed(rows)
    buf = torch.full(((rows + 1) * (K + pad),), 99.0, device=DEV, dtype=DT[src])   # larger than anything in x
    v = buf[off:off + rows * (K + pad)].view(rows, K + pad)[:, :K]
    v.copy_(torch.randn(rows, K, device=DEV, generator=g))
    v[rows - 1, K - 1] = -8.5
    a = torch.full((1,), 1e30, device=DEV)
    tsd.op_fp4_absmax(v, a)
    assert a.item() == 8.5
    v[0, 0] = float("inf")
    tsd.op_fp4_absmax(v, a)
    assert a.item() == float("inf")
    v[0, K // 2] = float("nan")
    tsd.op_fp4_absmax(v, a)
    assert np.isnan(a.item())
    v.zero_()
    tsd.op_fp4_absmax(v, a)
    assert a.item() == 0.0
    a.fill_(5.0)
    tsd.op_fp4_absmax(torch.empty(0, K, device=DEV), a)
    assert a.item() == 0.0


# ------------------------------------------------------------------------------------ products
def silu64(v):
    return v / (1 + torch.exp(-v))


def check_product(out, xv, wv, mode, act, bias, xerr=0.0):
    """out against act(xv wv' + bias) with the bounds derived above (the 64-bit products on the GPU: they are many)."""
    K = xv.shape[1]
    bf16 = out.dtype == torch.bfloat16
    xv, wv = torch.from_numpy(xv).to(DEV), torch.from_numpy(wv).to(DEV)
    acc = xv @ wv.T
    mag = xv.abs() @ wv.abs().T
    err = (2 * K * U + xerr + 3 * U) * mag
    rms = (8 * np.sqrt(K) * U + xerr + 3 * U) * mag.norm()
    if bias is not None:
        acc = acc + torch.from_numpy(bias).to(DEV).double()
        err, rms = err + U * acc.abs(), rms + U * acc.norm()
    f = 2.0 ** -20 if bf16 else 8 * U
    if mode == tsd.EPI_SWIGLU:
        a, b, ea, eb = acc[:, 0::2], acc[:, 1::2], err[:, 0::2], err[:, 1::2]
        acc = silu64(a) * b
        err = 1.1 * ea * b.abs() + silu64(a).abs() * eb + 1.1 * ea * eb + (f + U) * acc.abs()
        rms = None
    elif act == tsd.ACT_SILU:
        s = silu64(acc)
        err, rms = 1.1 * err + f * s.abs(), 1.1 * rms + f * s.norm()
        acc = s
    got = out.double()
    half = torch.finfo(out.dtype).eps / 2 if bf16 else 0.0
    err = err + half * (acc.abs() + err) + 1e-38
    bad = ~((got - acc).abs() <= err)
    assert not bad.any(), (int(bad.sum()), bad.numel(), bad.nonzero()[:4].tolist(), float(((got - acc).abs() / err).max()))
    if rms is not None:
        assert (got - acc).norm() <= rms + half * acc.norm()


def operands(rng, N, M, K, fmt, amax):
    x = (rng.standard_normal((N, K)) * np.exp2(rng.uniform(-3, 3, (1, K)))).astype(np.float32)
    w = (0.05 * rng.standard_normal((M, K))).astype(np.float32)
    xa, wa = (np.abs(x).max(), np.abs(w).max()) if amax else (None, None)
    t = lambda a: None if a is None else torch.tensor([a], device=DEV)   # noqa: E731
    return make4(x, fmt, xa), make4(w, fmt, wa), t(xa), t(wa), x


def gemm(X, W, fmt, out, stream=0, **kw):
    tsd.op_fp4_gemm(W[0], W[1], X[0], X[1], fmt, out, stream=stream, **kw)


GEMM_SHAPES = [(1, 1, 32), (1, 64, 64), (5, 7, 96), (16, 200, 128), (63, 65, 160), (64, 64, 256), (77, 1000, 2080),
               (128, 128, 512), (129, 257, 288), (200, 384, 1536), (388, 1536, 4096), (257, 770, 544), (1, 8192, 1536),
               (600, 130, 320)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", GEMM_SHAPES)
def test_gemm_store(fmt, N, M, K):
    rng = np.random.default_rng(N + M + K)
    X, W, xa, wa, _ = operands(rng, N, M, K, fmt, fmt == NV)
    out = torch.full((N, M), float("nan"), device=DEV)
    gemm(X, W, fmt, out, x_amax=xa, w_amax=wa)
    check_product(out, X[2], W[2], tsd.EPI_STORE, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", [(3, 2, 64), (77, 1000, 288), (300, 512, 1536), (130, 66, 96)])
@pytest.mark.parametrize("kind", ["bias", "silu", "swiglu", "bf16", "silu_bf16", "swiglu_f32"])
def test_gemm_epilogues(fmt, N, M, K, kind):
    rng = np.random.default_rng(N * M + K)
    X, W, _, _, _ = operands(rng, N, M, K, fmt, False)
    swiglu, act = "swiglu" in kind, tsd.ACT_SILU if "silu" in kind else tsd.ACT_NONE
    bias = None if swiglu else rng.standard_normal(M).astype(np.float32)
    out = torch.full((N, M // 2 if swiglu else M), float("nan"), device=DEV,
                     dtype=torch.bfloat16 if kind in ("bf16", "silu_bf16", "swiglu") else torch.float32)
    mode = tsd.EPI_SWIGLU if swiglu else tsd.EPI_STORE
    gemm(X, W, fmt, out, mode=mode, act=act, bias=None if bias is None else torch.from_numpy(bias).to(DEV))
    check_product(out, X[2], W[2], mode, act, bias)


# One tile form after the other (the sizes choose it): 128 x 128, one 256 x 256 tile for each CTA pair, several
WIDE = [(100, 16384, 96), (128, 12800, 1120), (388, 8192, 288), (300, 8200, 1056), (250, 18944, 544), (2600, 4008, 96), (2305, 4100, 800)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", WIDE)
@pytest.mark.parametrize("kind", ["f32", "bias_bf16", "swiglu", "bias_silu", "swiglu_f32"])
def test_gemm_wide_tiles(fmt, N, M, K, kind):
    rng = np.random.default_rng(N + M + K)
    X, W, xa, wa, _ = operands(rng, N, M, K, fmt, fmt == NV)
    swiglu, act = "swiglu" in kind, tsd.ACT_SILU if "silu" in kind else tsd.ACT_NONE
    bias = rng.standard_normal(M).astype(np.float32) if "bias" in kind else None
    out = torch.full((N, M // 2 if swiglu else M), float("nan"), device=DEV, dtype=torch.bfloat16 if kind in ("bias_bf16", "swiglu") else torch.float32)
    mode = tsd.EPI_SWIGLU if swiglu else tsd.EPI_STORE
    gemm(X, W, fmt, out, mode=mode, act=act, bias=None if bias is None else torch.from_numpy(bias).to(DEV), x_amax=xa, w_amax=wa)
    check_product(out, X[2], W[2], mode, act, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_gemm_wide_scale_of_every_block_counts_in_a_graph(fmt):
    """As above for CTA pairs, and replayed: the operands are those of the moment."""
    N, M, K = 2400, 4352, 288
    rng = np.random.default_rng(3)

    def tensor(rows):
        codes = rng.integers(0, 256, (rows, K // 2), dtype=np.uint8)
        b = rng.integers(120, 135, (rows, K // BLOCK[fmt])) if fmt == MX else rng.integers(40, 90, (rows, K // BLOCK[fmt]))
        t = tiles_of(b.astype(np.uint8), rows, K, fmt)
        return torch.from_numpy(codes).to(DEV), torch.from_numpy(t).to(DEV), values(codes, t, fmt)

    X, W = tensor(N), tensor(M)
    out = torch.empty(N, M, device=DEV)
    graph = torch.cuda.CUDAGraph()
    gemm(X, W, fmt, out)
    with torch.cuda.graph(graph):
        gemm(X, W, fmt, out, stream=torch.cuda.current_stream().cuda_stream)
    Y = tensor(N)
    X[0].copy_(Y[0]), X[1].copy_(Y[1])
    out.fill_(float("nan"))
    graph.replay()
    check_product(out, Y[2], W[2], tsd.EPI_STORE, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", [tsd.EPI_STORE, tsd.EPI_SWIGLU])
@pytest.mark.parametrize("N,M,K", [(77, 58, 64), (150, 1182, 96), (2600, 2990, 64), (33, 16390, 64)])
def test_gemm_rows_without_alignment(dtype, mode, N, M, K):
    """Odd output widths, so that a row starts anywhere, for every tile form."""
    X, W, _, _, _ = operands(np.random.default_rng(N), N, M, K, NV, False)
    cols = (M // 2 if mode == tsd.EPI_SWIGLU else M) | 1
    buf = torch.full((N * cols + 3,), 5.0, device=DEV, dtype=dtype)
    out = buf[1:1 + N * cols].view(N, cols)[:, :M // 2 if mode == tsd.EPI_SWIGLU else M]
    gemm(X, W, NV, out, mode=mode)
    check_product(out, X[2], W[2], mode, 0, None)
    out.fill_(5.0)
    assert (buf == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,off", [(8, 0), (3, 0), (16, 1), (5, 7), (8, 8), (0, 16)])
@pytest.mark.parametrize("N,M,K", [(150, 203, 96), (2500, 4000, 64), (350, 8192, 64)])
def test_gemm_output_strides(dtype, pad, off, N, M, K):
    X, W, _, _, _ = operands(np.random.default_rng(1), N, M, K, MX, False)
    buf = torch.full(((N + 1) * (M + pad) + 8,), 3.0, device=DEV, dtype=dtype)
    out = buf[off:off + N * (M + pad)].view(N, M + pad)[:, :M]
    gemm(X, W, MX, out)
    check_product(out.contiguous(), X[2], W[2], tsd.EPI_STORE, 0, None)
    out.fill_(3.0)
    assert (buf == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_gemm_scale_of_every_block_counts(fmt):
    """One block of K at a time under scales that no other has: a wrong scale, row or block shows."""
    N, M, K = 130, 200, 320
    rng = np.random.default_rng(2)
    nb = K // BLOCK[fmt]

    def tensor(rows):
        codes = rng.integers(0, 256, (rows, K // 2), dtype=np.uint8)
        b = rng.integers(120, 135, (rows, nb)) if fmt == MX else rng.integers(40, 90, (rows, nb))
        t = tiles_of(b.astype(np.uint8), rows, K, fmt)
        return torch.from_numpy(codes).to(DEV), torch.from_numpy(t).to(DEV), values(codes, t, fmt)

    X, W = tensor(N), tensor(M)
    out = torch.empty(N, M, device=DEV)
    gemm(X, W, fmt, out)
    check_product(out, X[2], W[2], tsd.EPI_STORE, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_gemm_extreme_scales_and_nan_blocks(fmt):
    N, M, K = 40, 72, 128
    rng = np.random.default_rng(3)
    x = rng.standard_normal((N, K)).astype(np.float32)
    w = rng.standard_normal((M, K)).astype(np.float32)
    if fmt == MX:
        x *= np.float32(2.0 ** 60)
        w *= np.float32(2.0 ** -90)
    X, W = make4(x, fmt), make4(w, fmt)
    out = torch.empty(N, M, device=DEV)
    gemm(X, W, fmt, out)
    check_product(out, X[2], W[2], tsd.EPI_STORE, 0, None)
    clean = out.clone()
    x[7, 100] = np.nan                                          # row 7 of x, column 9 of the product
    w[9, 3] = np.inf
    X, W = make4(x, fmt), make4(w, fmt)
    gemm(X, W, fmt, out)
    bad = torch.zeros(N, M, dtype=torch.bool, device=DEV)
    bad[7], bad[:, 9] = True, True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("xa,wa", [(1e-18, 1e-18), (3e-19, 3e-19), (2e-30, 5e-9), (1e-24, 1e-24), (1e23, 1e23), (3e38, 3e38), (1e38, 3e-30), (2e-15, 1e38)])
@pytest.mark.parametrize("N,M,K", [(40, 72, 96), (2400, 4352, 96)])
def test_gemm_maxima_at_the_ends_of_the_range(xa, wa, N, M, K):
    """Maxima whose factors' product no f32 holds, or only with fewer bits. Outputs are f32 where they lie in f32's range:
    K additions (2 K u, as above), four single roundings, and half a step of 2^-149 twice below the normal range."""
    rng = np.random.default_rng(9)

    def tensor(rows, top):
        v = rng.uniform(-1, 1, (rows, K)) * top
        v[0, 0] = top
        v[3] = 0
        v[5:8] *= 2.0 ** -19                                    # the smallest codes and scales: products far below the largest
        return make4(v.astype(np.float32), NV, np.float32(top)), torch.tensor([top], device=DEV)

    (X, xt), (W, wt) = tensor(N, xa), tensor(M, wa)
    out = torch.full((N, M), float("nan"), device=DEV)
    gemm(X, W, NV, out, x_amax=xt, w_amax=wt)
    xv, wv = torch.from_numpy(X[2]).to(DEV), torch.from_numpy(W[2]).to(DEV)
    acc, err = xv @ wv.T, (2 * K + 4) * U * (xv.abs() @ wv.abs().T) + 2.0 ** -149
    top = torch.finfo(torch.float32).max
    fits, past = acc.abs() + err < top, acc.abs() - err > top
    got = out.double()
    assert ((got - acc).abs() <= err)[fits].all(), float(((got - acc).abs() / err)[fits].max())
    assert (got == torch.copysign(torch.tensor(float("inf"), device=DEV), acc))[past].all()
    assert (out[3] == 0).all() and (out[:, 3] == 0).all()
    bias = torch.from_numpy((rng.uniform(-1, 1, M) * min(float(acc[fits].abs().max()), 1e38)).astype(np.float32)).to(DEV)
    gemm(X, W, NV, out, x_amax=xt, w_amax=wt, bias=bias)
    sums = acc + bias.double()
    fits = fits & (sums.abs() + err + U * sums.abs() < top)
    assert ((out.double() - sums).abs() <= err + U * sums.abs())[fits].all()


@pytest.mark.gpu
def test_gemm_zero_operands_and_negative_zero_codes():
    X = torch.full((33, 80), 0x88, device=DEV, dtype=torch.uint8), torch.zeros(tsd.fp4_scale_bytes(33, 160, NV), device=DEV, dtype=torch.uint8)
    W = torch.full((50, 80), 0xFF, device=DEV, dtype=torch.uint8), torch.full((tsd.fp4_scale_bytes(50, 160, NV),), 0, device=DEV, dtype=torch.uint8)
    out = torch.full((33, 50), 4.0, device=DEV)
    gemm(X, W, NV, out)
    assert (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 8])
@pytest.mark.parametrize("M,K", [(1, 32), (9, 64), (130, 96), (1000, 2080), (256, 1536), (33, 12288)])
def test_gemv(fmt, N, M, K):
    rng = np.random.default_rng(N + M + K)
    _, W, _, wa, x = operands(rng, N, M, K, fmt, fmt == NV)
    bias = rng.standard_normal(M).astype(np.float32)
    act = tsd.ACT_SILU if N % 2 else tsd.ACT_NONE
    y = torch.full((N, M), float("nan"), device=DEV, dtype=torch.bfloat16 if N % 3 == 0 else torch.float32)
    tsd.op_fp4_gemv(W[0], W[1], fmt, torch.from_numpy(x).to(DEV), y, bias=torch.from_numpy(bias).to(DEV), act=act, w_amax=wa)
    check_product(y, x.astype(np.float64), W[2], tsd.EPI_STORE, act, bias, xerr=U)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", [(1, 19000, 32), (2, 19001, 96), (4, 20000, 416), (5, 18944, 160), (8, 19077, 2080), (3, 19000, 4256), (7, 19200, 1152),
                                   (1, 4201, 544), (2, 4300, 1056), (4, 4222, 288), (8, 8333, 352)])
def test_gemv_many_rows(fmt, N, M, K):
    """The forms for some and for many rows: ragged K and M, more K than is staged at once."""
    rng = np.random.default_rng(N + M + K)
    x = (rng.standard_normal((N, K)) * np.exp2(rng.uniform(-8, 8, (1, K)))).astype(np.float32)
    w = (0.05 * rng.standard_normal((M, K)) * np.exp2(rng.integers(-9, 9, (M, 1)))).astype(np.float32)
    wa = np.abs(w).max() if fmt == NV else None
    W = make4(w, fmt, wa)
    bias = rng.standard_normal(M).astype(np.float32)
    y = torch.full((N, M), float("nan"), device=DEV, dtype=torch.bfloat16 if N == 2 else torch.float32)
    tsd.op_fp4_gemv(W[0], W[1], fmt, torch.from_numpy(x).to(DEV), y, bias=torch.from_numpy(bias).to(DEV),
                    act=tsd.ACT_SILU if N == 4 else tsd.ACT_NONE, w_amax=None if wa is None else torch.tensor([wa], device=DEV))
    check_product(y, x.astype(np.float64), W[2], tsd.EPI_STORE, tsd.ACT_SILU if N == 4 else tsd.ACT_NONE, bias, xerr=4 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", [(1, 1, 32), (1, 149, 4736), (2, 500, 1056), (3, 1000, 288), (8, 2960, 544), (8, 2961, 544), (2, 3500, 1536),
                                   (4, 3333, 2080), (5, 3333, 1536), (6, 63, 5024)])
def test_gemv_few_rows(fmt, N, M, K):
    """Warps that share rows and take turns along K, some of them without a turn, and warps on their own."""
    rng = np.random.default_rng(N * M + K)
    _, W, _, wa, x = operands(rng, N, M, K, fmt, fmt == NV)
    y = torch.full((N, M), float("nan"), device=DEV, dtype=torch.bfloat16 if N == 4 else torch.float32)
    tsd.op_fp4_gemv(W[0], W[1], fmt, torch.from_numpy(x).to(DEV), y, w_amax=wa)
    check_product(y, x.astype(np.float64), W[2], tsd.EPI_STORE, 0, None, xerr=U)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", [(1, 8300, 32), (1, 40001, 1536), (2, 8290, 800), (2, 20000, 1056), (3, 8448, 2080), (4, 38000, 160),
                                   (5, 9000, 96), (6, 19100, 1536), (7, 57000, 544), (8, 8400, 1568), (2, 19000, 6400), (3, 18950, 4256),
                                   (7, 18944, 2080)])
def test_gemv_digits(fmt, N, M, K):
    """Many rows of short vectors: one and several tiles to a CTA, vectors that fill their digits' tile and not, two launches."""
    rng = np.random.default_rng(N + M + K)
    x = (rng.standard_normal((N, K)) * np.exp2(rng.uniform(-8, 8, (1, K)))).astype(np.float32)
    w = (0.05 * rng.standard_normal((M, K)) * np.exp2(rng.integers(-9, 9, (M, 1)))).astype(np.float32)
    wa = np.abs(w).max() if fmt == NV else None
    W = make4(w, fmt, wa)
    bias = rng.standard_normal(M).astype(np.float32) if N % 2 else None
    act = tsd.ACT_SILU if N % 3 == 0 else tsd.ACT_NONE
    y = torch.full((N, M), float("nan"), device=DEV, dtype=torch.bfloat16 if N in (2, 5) else torch.float32)
    tsd.op_fp4_gemv(W[0], W[1], fmt, torch.from_numpy(x).to(DEV), y, bias=None if bias is None else torch.from_numpy(bias).to(DEV),
                    act=act, w_amax=None if wa is None else torch.tensor([wa], device=DEV))
    check_product(y, x.astype(np.float64), W[2], tsd.EPI_STORE, act, bias, xerr=4 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N", [1, 2, 4, 8])
@pytest.mark.parametrize("more", [0, 32])
def test_gemv_longest_vectors_of_a_form(fmt, N, more):
    """The largest K whose digits (128-byte rows of 256 elements, 16 to a vector) and scales (512 bytes to 4 blocks) fit beside
    three stages of weights in shared memory, and the next."""
    room = 227 * 1024 - 2048 - 3 * (32768 + 512 * 512 // (4 * BLOCK[fmt]))
    size = lambda K: -(-K // 256) * N * 2048 + -(-K // (4 * BLOCK[fmt])) * 512   # noqa: E731
    K = max(k for k in range(32, 20000, 32) if size(k) <= room) + more
    M = 8300
    rng = np.random.default_rng(K)
    x = rng.standard_normal((N, K)).astype(np.float32)
    codes = rng.integers(0, 256, (M, K // 2), dtype=np.uint8)
    nb = K // BLOCK[fmt]
    t = tiles_of((rng.integers(120, 135, (M, nb)) if fmt == MX else rng.integers(40, 90, (M, nb))).astype(np.uint8), M, K, fmt)
    y = torch.full((N, M), float("nan"), device=DEV)
    tsd.op_fp4_gemv(torch.from_numpy(codes).to(DEV), torch.from_numpy(t).to(DEV), fmt, torch.from_numpy(x).to(DEV), y)
    check_product(y, x.astype(np.float64), values(codes, t, fmt), tsd.EPI_STORE, 0, None, xerr=4 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("M", [200, 8400])
def test_gemv_unlike_magnitudes(fmt, M):
    """Vectors at the ends of f32's range, blocks and elements far below the largest: an element is off by 2^-22 of
    itself, or 2^-45 of the largest of its 128 and 2^-62 of the vector's, whichever is more."""
    N, K = 8, 512
    rng = np.random.default_rng(31)
    W = make4((0.5 * rng.standard_normal((M, K))).astype(np.float32), fmt)
    x = rng.standard_normal((N, K))
    x[0] *= 2.0 ** 115 / np.abs(x[0]).max()
    x[1] *= 2.0 ** -100
    x[2] *= 2.0 ** -140                                         # subnormal
    x[3] *= np.exp2(rng.integers(-60, 1, K))
    x[4] *= np.exp2(np.repeat(rng.integers(-90, 1, K // 16), 16))
    x[5, 1:] *= 2.0 ** -30
    x[6], x[6, 100] = 0, 2.0 ** -126
    x[7, ::2] = 0
    x = x.astype(np.float32)
    y = torch.full((N, M), float("nan"), device=DEV)
    tsd.op_fp4_gemv(W[0], W[1], fmt, torch.from_numpy(x).to(DEV), y)
    xv = x.astype(np.float64)
    top = np.repeat(np.abs(xv).reshape(N, -1, 128).max(-1), 128, axis=1)
    dx = np.maximum(2.0 ** -22 * np.abs(xv), np.maximum(2.0 ** -45 * top, 2.0 ** -62 * np.abs(xv).max(1, keepdims=True)))
    acc, mag, derr = xv @ W[2].T, np.abs(xv) @ np.abs(W[2]).T, dx @ np.abs(W[2]).T
    err = derr + (2 * K + 3) * U * mag + K * 2.0 ** -148        # products and sums at the end of the range lose up to a step of it each
    bad = ~(np.abs(y.double().cpu().numpy() - acc) <= err)
    assert not bad.any(), np.argwhere(bad)[:4]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", [(8, 200, 512), (1, 200, 512), (8, 8400, 512), (1, 8400, 544), (3, 6000, 512), (8, 10000, 2592), (8, 19000, 4256), (3, 18950, 6400)])
def test_gemv_sums_that_leave_the_range_on_the_way(fmt, N, M, K):
    """Elements up to f32's end under small block scales (MX) or a small maximum (NV), in every form: y is finite and as near as
    elsewhere (bounds of the test above) wherever the exact value lies in f32's range, infinite beyond it."""
    rng = np.random.default_rng(41)
    nb = K // BLOCK[fmt]
    codes = rng.integers(0, 256, (M, K // 2), dtype=np.uint8)
    b = rng.integers(125, 128, (M, nb)) + rng.integers(-100, -1, (M, 1)) if fmt == MX else rng.integers(60, 127, (M, nb))
    t, wa = tiles_of(b.astype(np.uint8), M, K, fmt), None if fmt == MX else 0.02
    W = torch.from_numpy(codes).to(DEV), torch.from_numpy(t).to(DEV), values(codes, t, fmt) * float(factors(wa)[1])
    x = rng.uniform(-1, 1, (8, K))
    x[0] *= 2.0 ** 127.9
    x[1, 1::7] *= 2.0 ** 127.5                                  # few elements at the end, the others near one
    x[2] = np.abs(x[2]) * 2e35
    x[3] *= 2.0 ** 124 * np.exp2(np.repeat(rng.integers(-60, 1, K // 32), 32))
    x[4] = np.repeat(x[4, ::2], 2) * np.tile([1.0, -1.0], K // 2) * 2.0 ** 127   # neighbours of opposite sign
    x[5, 9] = 3.4e38
    x[6] *= 2.0 ** 100
    x = x[:N].astype(np.float32)
    y = torch.full((N, M), float("nan"), device=DEV)
    tsd.op_fp4_gemv(W[0], W[1], fmt, torch.from_numpy(x).to(DEV), y, w_amax=None if wa is None else torch.tensor([wa], device=DEV))
    xv, wv = torch.from_numpy(x).to(DEV).double(), torch.from_numpy(W[2]).to(DEV)
    near = torch.nn.functional.max_pool1d(xv.abs()[None], 255, stride=1, padding=127)[0]         # the largest of any 128 around
    dx = torch.maximum(2.0 ** -22 * xv.abs(), torch.maximum(2.0 ** -45 * near, 2.0 ** -62 * xv.abs().amax(1, keepdim=True)))
    acc, mag, derr = xv @ wv.T, xv.abs() @ wv.abs().T, dx @ wv.abs().T
    err = derr + (2 * K + 3) * U * mag + K * 2.0 ** -148
    got, top = y.double(), torch.finfo(torch.float32).max
    fits, past = acc.abs() + err < top, acc.abs() - err > top
    bad = fits & ~((got - acc).abs() <= err)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
    assert (got == torch.copysign(torch.tensor(float("inf"), device=DEV), acc))[past].all()
    assert fits.double().mean() > 0.8


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(200, 512), (8400, 512), (18950, 6400)])
def test_gemv_weights_near_the_end_of_the_range(M, K):
    """Vectors whose digits, before they are weighed, add up to more than the vector: every element but one of a block is -1/4
    under a largest of 0.9 (its second digit alone is -2 / 8 of the block's power of two), weights 6 * 2^s with the
    largest at a weight of zero. The sums are exact in f32 and in range, those of the second digits are not."""
    codes = np.full((M, K // 2), 0x77, np.uint8)
    codes[:, ::16] = 0x70                                       # element 0 of a block: zero
    s = int(np.floor(np.log2(2.0 ** 128 / (6 * K * 31 / 32 * 0.25)))) - 1
    t = tiles_of(np.full((M, K // 32), 127 + s, np.uint8), M, K, MX)
    x = np.full((3, K), -0.25, np.float32)
    x[:, ::32] = 0.9
    x[1] *= -1
    x[2, K // 2:] *= -1                                         # both ends of the range in one sum of zero
    y = torch.full((3, M), float("nan"), device=DEV)
    tsd.op_fp4_gemv(torch.from_numpy(codes).to(DEV), torch.from_numpy(t).to(DEV), MX, torch.from_numpy(x).to(DEV), y)
    want = 6 * 2.0 ** s * 0.25 * K * 31 / 32
    assert want * 4 > 2.0 ** 128 > want
    assert (y[0] == -want).all() and (y[1] == want).all() and (y[2].abs() <= 2 * K * U * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [77, 9000, 19000])
def test_gemv_strides_magnitudes_and_nan(M):
    N, K = 5, 160
    rng = np.random.default_rng(4)
    W = make4((0.1 * rng.standard_normal((M, K))).astype(np.float32), NV)
    x = rng.standard_normal((N, K)).astype(np.float32)
    x[1] *= np.float32(1e30)                                    # rows of unlike size do not touch each other
    x[2] *= np.float32(1e-30)
    x[3, ::3] *= np.float32(1e-6)                               # small next to large within a row
    x[4] = 0
    buf = torch.zeros(N * (K + 3) + 1, device=DEV)
    xs = buf[1:].view(N, K + 3)[:, :K]
    xs.copy_(torch.from_numpy(x))
    yb = torch.full((N * (M + 5) + 1,), 2.0, device=DEV)
    y = yb[1:].view(N, M + 5)[:, :M]
    tsd.op_fp4_gemv(W[0], W[1], NV, xs, y)
    for n in range(N):
        check_product(y[n:n + 1].contiguous(), x[n:n + 1].astype(np.float64), W[2], tsd.EPI_STORE, 0, None, xerr=4 * U)
    clean = y.clone()
    xs[0, 5], xs[4, 7] = float("nan"), float("inf")
    tsd.op_fp4_gemv(W[0], W[1], NV, xs, y)
    assert torch.isnan(y[0]).all() and torch.equal(y[1:4], clean[1:4]) and not torch.isfinite(y[4]).any()
    y.fill_(2.0)
    assert (yb == 2.0).all()


# ------------------------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_a_block_s_feed_forward_in_four_bits(fmt):
    """norm -> 4 bits -> w1/w3 with SwiGLU -> 4 bits -> w2 -> gate, residual, norm: each stage against the 64-bit
    formula on what the stage before gave, eagerly and as a replayed graph with other inputs."""
    N, H, F = 90, 256, 352
    rng = np.random.default_rng(11)
    w13, w2 = (0.06 * rng.standard_normal((2 * F, H))).astype(np.float32), (0.06 * rng.standard_normal((H, F))).astype(np.float32)
    W13, W2 = make4(w13, fmt), make4(w2, fmt)
    g = torch.Generator(device=DEV).manual_seed(1)
    x, gate = torch.randn(N, H, device=DEV, generator=g), torch.randn(N, H, device=DEV, generator=g)
    shift, scale = torch.randn(H, device=DEV, generator=g), torch.randn(H, device=DEV, generator=g)
    h, hid = torch.empty(N, H, device=DEV, dtype=torch.bfloat16), torch.empty(N, F, device=DEV, dtype=torch.bfloat16)
    y, x2, h2 = torch.empty(N, H, device=DEV), torch.empty_like(x), torch.empty_like(h)
    four = lambda r, k: (torch.empty(r, k // 2, device=DEV, dtype=torch.uint8),   # noqa: E731
                         torch.empty(tsd.fp4_scale_bytes(r, k, fmt), device=DEV, dtype=torch.uint8))
    hq, hidq = four(N, H), four(N, F)
    ha, hida = (torch.empty(1, device=DEV), torch.empty(1, device=DEV)) if fmt == NV else (None, None)

    def block():
        st = torch.cuda.current_stream().cuda_stream
        tsd.op_gate_norm(x, None, None, h, pre_norm=tsd.NORM_LAYER, shift=shift, scale=scale, stream=st)
        if fmt == NV:
            tsd.op_fp4_absmax(h, ha, stream=st)
        tsd.op_fp4_quantize(h, fmt, *hq, amax=ha, stream=st)
        gemm(hq, W13, fmt, hid, mode=tsd.EPI_SWIGLU, x_amax=ha, stream=st)
        if fmt == NV:
            tsd.op_fp4_absmax(hid, hida, stream=st)
        tsd.op_fp4_quantize(hid, fmt, *hidq, amax=hida, stream=st)
        gemm(hidq, W2, fmt, y, x_amax=hida, stream=st)
        tsd.op_gate_norm(x, y, x2, h2, post_norm=tsd.NORM_RMS, gate=gate, pre_norm=tsd.NORM_LAYER, shift=shift, scale=scale, stream=st)

    def look():
        torch.cuda.synchronize()
        for src, q, a in ((h, hq, ha), (hid, hidq, hida)):
            rc, rt, _ = quantize(src.float().cpu().numpy(), fmt, None if a is None else float(src.float().abs().max()))
            assert np.array_equal(q[0].cpu().numpy(), rc) and np.array_equal(q[1].cpu().numpy(), rt)
        hv = [values(q[0].cpu().numpy(), q[1].cpu().numpy(), fmt) * (1.0 if a is None else float(factors(a.item())[1]))
              for q, a in ((hq, ha), (hidq, hida))]
        check_product(hid, hv[0], W13[2], tsd.EPI_SWIGLU, 0, None)
        check_product(y, hv[1], W2[2], tsd.EPI_STORE, 0, None)
        yd = y.double()
        want = x.double() + gate.double() * yd / torch.sqrt((yd * yd).mean(-1, keepdim=True) + 1e-5)
        assert ((x2.double() - want).norm() / want.norm()) < 1e-6
        ref = torch.nn.functional.layer_norm(x2.double(), (H,)) * (1 + scale.double()) + shift.double()
        assert ((h2.double() - ref).norm() / ref.norm()) < 2.0 ** -8

    block()
    look()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
    for k in range(2):
        x.copy_(torch.randn(N, H, device=DEV, generator=g) * (1 + 3 * k))
        graph.replay()
        look()


@pytest.mark.gpu
def test_calls_on_two_streams_and_repeats_give_the_same_bits():
    rng = np.random.default_rng(12)
    X, W, xa, wa, x = operands(rng, 300, 1000, 1536, NV, True)
    xt = torch.from_numpy(x[:4]).to(DEV)
    outs, ys = [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for k in range(4):
        s = streams[k % 2]
        with torch.cuda.stream(s):
            outs.append(torch.empty(300, 1000, device=DEV))
            ys.append(torch.empty(4, 1000, device=DEV))
            gemm(X, W, NV, outs[-1], x_amax=xa, w_amax=wa, stream=s.cuda_stream)
            tsd.op_fp4_gemv(W[0], W[1], NV, xt, ys[-1], w_amax=wa, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o, y in zip(outs[1:], ys[1:]):
        assert torch.equal(o, outs[0]) and torch.equal(y, ys[0])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
def test_row_strides_past_32_bits(fmt):
    """Inputs and outputs whose row strides put offsets, in elements and in bytes, past 32 bits."""
    rng = np.random.default_rng(21)
    N, M, K, ld = 3, 200, 288, 2 ** 30 + 8
    far = lambda cols, dt: torch.empty(2 * ld + cols, device=DEV, dtype=dt).as_strided((3, cols), (ld, 1))   # noqa: E731
    X, W, xa, wa, x = operands(rng, N, M, K, fmt, fmt == NV)
    fx = far(K, torch.float32)
    fx.copy_(torch.from_numpy(x))
    c, t = dev_quantize(fx, fmt, xa)
    assert torch.equal(c, X[0]) and torch.equal(t, X[1])
    m = torch.empty(1, device=DEV)
    tsd.op_fp4_absmax(fx, m)
    assert m.item() == np.abs(x).max()
    fy = far(K, torch.bfloat16)
    tsd.op_fp4_dequantize(c, t, fmt, fy, amax=xa)
    y = torch.empty(N, K, device=DEV, dtype=torch.bfloat16)
    tsd.op_fp4_dequantize(c, t, fmt, y, amax=xa)
    assert torch.equal(fy, y)
    out = far(M, torch.float32)
    gemm(X, W, fmt, out, x_amax=xa, w_amax=wa)
    check_product(out, X[2], W[2], tsd.EPI_STORE, 0, None)
    out.fill_(float("nan"))
    tsd.op_fp4_gemv(W[0], W[1], fmt, fx, out, w_amax=wa)
    check_product(out, x.astype(np.float64), W[2], tsd.EPI_STORE, 0, None, xerr=U)
    # the same through staging buffers (several pair tiles to a CTA pair) and the many-row product
    M = 19000
    _, W, _, wa, _ = operands(rng, 1, M, 96, fmt, fmt == NV)
    X, _, xa, _, _ = operands(rng, 300, 1, 96, fmt, fmt == NV)
    del out
    big = torch.empty(299 * (2 ** 24) + M, device=DEV, dtype=torch.bfloat16).as_strided((300, M), (2 ** 24, 1))
    gemm(X, W, fmt, big, x_amax=xa, w_amax=wa)
    check_product(big, X[2], W[2], tsd.EPI_STORE, 0, None)
    del big
    out = far(M, torch.bfloat16)
    v = torch.from_numpy(rng.standard_normal((3, 96)).astype(np.float32)).to(DEV)
    tsd.op_fp4_gemv(W[0], W[1], fmt, v, out, w_amax=wa)
    check_product(out, v.double().cpu().numpy(), W[2], tsd.EPI_STORE, 0, None, xerr=4 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [MX, NV])
@pytest.mark.parametrize("N,M,K", [(1, 2 ** 19 + 300, 16416), (2, 2 ** 19 + 300, 16416), (5, 2 ** 19 + 300, 16416),
                                   (130, 2 ** 19 + 300, 16416), (1, 2 ** 22 + 300, 2080), (3, 2 ** 22 + 300, 2080)])
def test_codes_past_4_gb(fmt, N, M, K):
    """A weight whose last rows' codes lie past 4 GB; the rows before them are zero."""
    tail = 300
    rng = np.random.default_rng(N)
    codes = torch.zeros(M, K // 2, device=DEV, dtype=torch.uint8)
    scales = torch.zeros(tsd.fp4_scale_bytes(M, K, fmt), device=DEV, dtype=torch.uint8)
    _, W, _, _, _ = operands(rng, 1, tail, K, fmt, False)
    codes[-tail:] = W[0]
    scales[-W[1].numel():] = W[1]                               # 2^19 rows are whole tiles
    out = torch.full((N, M), float("nan"), device=DEV)
    x = rng.standard_normal((N, K)).astype(np.float32)
    if N <= 8:
        tsd.op_fp4_gemv(codes, scales, fmt, torch.from_numpy(x).to(DEV), out)
        check_product(out[:, -tail:], x.astype(np.float64), W[2], tsd.EPI_STORE, 0, None, xerr=4 * U)
    else:
        X = make4(x, fmt)
        gemm(X, (codes, scales), fmt, out)
        check_product(out[:, -tail:], X[2], W[2], tsd.EPI_STORE, 0, None)
    assert not out[:, :-tail].any()


FIRST_CALLS = """
import __graft_entry__
__graft_entry__.load_package()
import torch
from tsd_b200 import tsd
DEV, NV, N, M, K = "cuda:0", tsd.FP4_NV, %d, %d, 288
g = torch.Generator(device=DEV).manual_seed(1)
n = lambda *s: torch.randn(*s, device=DEV, generator=g)
x, y, w, v = n(N, K), n(N, K), n(M, K), n(5, K)
z = lambda *s, dtype=torch.uint8: torch.zeros(*s, device=DEV, dtype=dtype)
xq, xs, wq, ws = z(N, K // 2), z(tsd.fp4_scale_bytes(N, K, NV)), z(M, K // 2), z(tsd.fp4_scale_bytes(M, K, NV))
xa, wa, h, out, back, vec = z(1, dtype=torch.float32), z(1, dtype=torch.float32), z(N, K, dtype=torch.bfloat16), z(N, M, dtype=torch.float32), z(M, K, dtype=torch.bfloat16), z(5, M, dtype=torch.float32)
def step(stream):
    tsd.op_gate_norm(x, y, None, h, pre_norm=tsd.NORM_RMS, stream=stream)
    tsd.op_fp4_absmax(h, xa, stream=stream)
    tsd.op_fp4_quantize(h, NV, xq, xs, amax=xa, stream=stream)
    tsd.op_fp4_absmax(w, wa, stream=stream)
    tsd.op_fp4_quantize(w, NV, wq, ws, amax=wa, stream=stream)
    tsd.op_fp4_gemm(wq, ws, xq, xs, NV, out, w_amax=wa, x_amax=xa, stream=stream)
    tsd.op_fp4_dequantize(wq, ws, NV, back, amax=wa, stream=stream)
    tsd.op_fp4_gemv(wq, ws, NV, v, vec, w_amax=wa, stream=stream)
results = (h, xa, xq, xs, wa, wq, ws, out, back, vec)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step(torch.cuda.current_stream().cuda_stream)
for t in results: t.zero_()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in results]
for t in results: t.zero_()
step(0)
torch.cuda.synchronize()
assert all(torch.equal(a, b) and a.any() for a, b in zip(got, results))
print("same bits")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", [(50, 300), (600, 20000)])
def test_first_calls_of_a_process_can_be_captured(N, M):
    """What an entry point sets up on its first call happens while a stream is being captured."""
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS % (N, M)], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "same bits" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_empty_calls_and_host_memory():
    e = lambda *s, dtype=torch.uint8: torch.empty(*s, device=DEV, dtype=dtype)   # noqa: E731
    W = e(8, 32), e(tsd.fp4_scale_bytes(8, 64, MX))
    none = e(0, 32), e(0)
    gemm(none, W, MX, e(0, 8, dtype=torch.float32))
    tsd.op_fp4_gemv(W[0], W[1], MX, e(0, 64, dtype=torch.float32), e(0, 8, dtype=torch.float32))
    tsd.op_fp4_quantize(e(0, 64, dtype=torch.float32), MX, *none)
    tsd.op_fp4_dequantize(*none, MX, e(0, 64, dtype=torch.float32))
    for call in (lambda: gemm((torch.zeros(4, 32, dtype=torch.uint8), e(tsd.fp4_scale_bytes(4, 64, MX))), W, MX, e(4, 8, dtype=torch.float32)),
                 lambda: tsd.op_fp4_gemv(*W, MX, torch.zeros(1, 64), e(1, 8, dtype=torch.float32)),
                 lambda: tsd.op_fp4_quantize(torch.zeros(8, 64), MX, *W),
                 lambda: tsd.op_fp4_dequantize(*W, MX, torch.zeros(8, 64)),
                 lambda: tsd.op_fp4_absmax(torch.zeros(8, 64), e(1, dtype=torch.float32))):
        with pytest.raises(tsd.TsdError, match="TSD_ERR_ARG"):
            call()


@pytest.mark.gpu
def test_a_refused_launch_leaves_no_error_for_the_next_call():
    """A launch on the legacy stream while a stream that synchronises with it is being captured: the call says so, and the calls
    after the capture are none the wiser."""
    rt = ctypes.CDLL("libcudart.so.12")                         # torch's, already loaded
    x, h = torch.randn(4, 64, device=DEV), torch.empty(4, 64, device=DEV, dtype=torch.bfloat16)
    X, W, _, _, v = operands(np.random.default_rng(0), 4, 64, 64, MX, False)
    out, m, vt = torch.empty(4, 64, device=DEV), torch.zeros(1, 64, device=DEV), torch.from_numpy(v).to(DEV)
    amax = torch.empty(1, device=DEV)
    torch.cuda.synchronize()
    for call in (lambda: tsd.op_gate_norm(x, None, None, h, pre_norm=tsd.NORM_LAYER), lambda: tsd.op_fp4_absmax(x, amax),
                 lambda: tsd.op_fp4_quantize(x, MX, *dev_empty(4, 64)), lambda: tsd.op_fp4_dequantize(X[0], X[1], MX, out),
                 lambda: gemm(X, W, MX, out), lambda: tsd.op_fp4_gemv(W[0], W[1], MX, vt, out)):
        stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
        assert rt.cudaStreamCreate(ctypes.byref(stream)) == 0
        assert rt.cudaStreamBeginCapture(stream, 2) == 0        # relaxed: what this thread may call is not restricted
        with pytest.raises(tsd.TsdError, match="TSD_ERR_CUDA"):
            call()
        rt.cudaStreamEndCapture(stream, ctypes.byref(graph))    # the launch has spoilt it
        rt.cudaGetLastError()
        assert rt.cudaStreamDestroy(stream) == 0
        tsd.op_ln_modulate(x, 4, 64, m, m, 64, 0, 4, h)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------ without a GPU
def test_scale_bytes():
    f = tsd.lib().tsd_fp4_scale_bytes
    assert [f(1, 32, MX), f(128, 128, MX), f(129, 160, MX), f(0, 32, NV), f(1, 64, NV), f(256, 96, NV)] == [512, 512, 2048, 0, 512, 2048]
    assert [f(-1, 32, MX), f(1, 0, MX), f(1, 16, NV), f(1, 48, NV), f(1, 64, 2), f(1, 64, -1), f(2 ** 31, 32, MX)] == [-1] * 7
    assert [f(2 ** 30, 32, NV), f(1, 2 ** 25, MX)] == [2 ** 23 * 512, 2 ** 18 * 512]
    assert [f(2 ** 30 + 1, 32, NV), f(1, 2 ** 25 + 32, MX)] == [-1] * 2


def test_plain_implementation_against_differences_in_direct_form():
    """The oracle itself: every byte's value is the nearest the format has (by trying all codes), scales by their formula."""
    rng = np.random.default_rng(0)
    x = spread(rng, 9, 96)
    for fmt in (MX, NV):
        c, t, bad = quantize(x, fmt)
        v = values(c, t, fmt).reshape(9, -1, BLOCK[fmt])
        b = rows_of_tiles(t, 9, 96, fmt)
        z = x.astype(np.float64).reshape(v.shape)
        for r in range(9):
            for j in range(v.shape[1]):
                top = np.abs(z[r, j]).max()
                s = 2.0 ** (int(b[r, j]) - 127) if fmt == MX else E4M3[b[r, j]]
                if fmt == MX:
                    assert top == 0 or 4 <= top / s < 8
                else:
                    assert np.abs(E4M3 - top / 6).min() == abs(s - top / 6)
                for e in range(BLOCK[fmt]):
                    assert abs(v[r, j, e] - z[r, j, e]) == min(abs(z[r, j, e] - q * s) for q in np.concatenate([GRID, -GRID]))


P = dict(W=4096, Ws=8192, Wa=None, M=64, X=12288, Xs=16384, Xa=None, N=4, K=64, fmt=0, mode=0, act=0, bias=None, out=20480,
         out_type=0, ldo=64, err=None, stream=None)
V = dict(W=4096, Ws=8192, Wa=None, fmt=0, M=64, K=64, x=12288, ldx=64, N=4, bias=None, act=0, y=16384, y_type=0, ldy=64, stream=None)
Q = dict(x=4096, type=30, rows=4, K=64, ldx=64, fmt=1, amax=8192, codes=12288, scales=16384, stream=None)
D = dict(codes=4096, scales=8192, fmt=1, amax=None, rows=4, K=64, y=12288, type=0, ldy=64, stream=None)
A = dict(x=4096, type=0, rows=4, K=64, ldx=64, amax=8192, stream=None)


@pytest.mark.parametrize("fn,base,kw", [
    *[("tsd_op_fp4_gemm", P, k) for k in (
        dict(W=None), dict(Ws=None), dict(X=None), dict(Xs=None), dict(out=None), dict(M=0), dict(M=-4), dict(N=-1), dict(K=0),
        dict(K=48), dict(fmt=2), dict(mode=2), dict(mode=-1), dict(act=2), dict(mode=1, M=63), dict(mode=1, bias=4096),
        dict(mode=1, act=1), dict(Wa=4096), dict(Xa=4096), dict(out_type=1), dict(ldo=63), dict(mode=1, ldo=31), dict(W=4104),
        dict(X=12289), dict(Ws=8200), dict(Xs=16388), dict(out=20482), dict(bias=4097), dict(fmt=1, Wa=4098), dict(err=5),
        dict(M=2 ** 31 - 1, ldo=2 ** 31), dict(N=2 ** 31 - 1), dict(K=2 ** 25 + 32))],
    *[("tsd_op_fp4_gemv", V, k) for k in (
        dict(W=None), dict(Ws=None), dict(x=None), dict(y=None), dict(M=0), dict(N=9), dict(N=-1), dict(K=33), dict(fmt=7), dict(act=-1),
        dict(Wa=4096), dict(ldx=63), dict(ldy=63), dict(y_type=1), dict(W=4100), dict(Ws=8196), dict(x=12289), dict(y=16386), dict(bias=2),
        dict(M=2 ** 31 - 1, ldy=2 ** 31), dict(K=2 ** 27, ldx=2 ** 27))],
    *[("tsd_op_fp4_quantize", Q, k) for k in (
        dict(x=None), dict(codes=None), dict(scales=None), dict(type=8), dict(rows=-1), dict(K=16), dict(K=65), dict(ldx=63), dict(fmt=3),
        dict(fmt=0), dict(x=4097), dict(codes=12296), dict(scales=16385), dict(amax=8193),
        dict(rows=2 ** 31 - 1), dict(K=2 ** 31 - 32, ldx=2 ** 31))],
    *[("tsd_op_fp4_dequantize", D, k) for k in (
        dict(y=None), dict(codes=None), dict(scales=None), dict(type=2), dict(rows=-1), dict(K=31), dict(ldy=63), dict(fmt=-1),
        dict(fmt=0, amax=4096), dict(y=12290), dict(codes=4104), dict(scales=8193), dict(amax=3),
        dict(rows=2 ** 31 - 1), dict(K=2 ** 31 - 32, ldy=2 ** 31))],
    *[("tsd_op_fp4_absmax", A, k) for k in (
        dict(x=None), dict(amax=None), dict(type=9), dict(rows=-1), dict(K=0), dict(ldx=63), dict(x=4098), dict(amax=8194))],
])
def test_refusals(fn, base, kw):
    """Refused before anything is touched: the addresses are nobody's."""
    assert getattr(tsd.lib(), fn)(*dict(base, **kw).values()) == -1


def test_empty_calls_need_no_device():
    assert tsd.lib().tsd_op_fp4_gemm(*dict(P, N=0).values()) == 0
    assert tsd.lib().tsd_op_fp4_gemv(*dict(V, N=0).values()) == 0
    assert tsd.lib().tsd_op_fp4_quantize(*dict(Q, rows=0).values()) == 0
    assert tsd.lib().tsd_op_fp4_dequantize(*dict(D, rows=0).values()) == 0


def test_wrappers_refuse_shapes_and_types():
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype)   # noqa: E731
    f = lambda *s: torch.zeros(*s)                                   # noqa: E731
    W, Ws = z(8, 32), z(tsd.fp4_scale_bytes(8, 64, MX))
    X, Xs = z(3, 32), z(tsd.fp4_scale_bytes(3, 64, MX))
    for call in (lambda: tsd.op_fp4_gemm(W, Ws[1:], X, Xs, MX, f(3, 8)), lambda: tsd.op_fp4_gemm(W, Ws, X, Xs, MX, f(3, 7)),
                 lambda: tsd.op_fp4_gemm(W, Ws, z(3, 48), z(512), MX, f(3, 8)), lambda: tsd.op_fp4_gemm(W, Ws, X, Xs, MX, f(8, 3).t()),
                 lambda: tsd.op_fp4_gemm(W, Ws, X, Xs, MX, f(3, 8), mode=tsd.EPI_SWIGLU), lambda: tsd.op_fp4_gemm(W[:, ::2], Ws, X, Xs, MX, f(3, 8)),
                 lambda: tsd.op_fp4_gemm(W, Ws, X, Xs, MX, f(3, 8), bias=f(7)), lambda: tsd.op_fp4_gemm(W.float(), Ws, X, Xs, MX, f(3, 8)),
                 lambda: tsd.op_fp4_gemm(W, Ws, X, Xs, NV, f(3, 8), w_amax=f(2)), lambda: tsd.op_fp4_gemv(W, Ws, MX, f(2, 60), f(2, 8)),
                 lambda: tsd.op_fp4_gemv(W, Ws, MX, f(2, 64).half(), f(2, 8)), lambda: tsd.op_fp4_quantize(f(3, 96), MX, X, Xs),
                 lambda: tsd.op_fp4_quantize(f(64, 3).t(), MX, X, Xs), lambda: tsd.op_fp4_dequantize(X, Xs, MX, f(3, 63)),
                 lambda: tsd.op_fp4_absmax(f(4), f(1)), lambda: tsd.op_fp4_absmax(f(4, 4), f(1).half()), lambda: tsd.fp4_scale_bytes(3, 40, MX)):
        with pytest.raises(ValueError):
            call()


def test_wrappers_name_the_argument_that_is_wrong():
    """Numbered from 1 in the order of the call; None counts."""
    x = torch.zeros(4, 8)
    for call, number in ((lambda: tsd.op_gate_norm(None, None, None, x), "1 is missing"),
                         (lambda: tsd.op_gate_norm(x, None, None, 3), "4 is not a tensor"),
                         (lambda: tsd.op_gate_norm(x, None, None, x, gate=3), "8 is not a tensor"),
                         (lambda: tsd.op_gate_norm(x, None, None, x, mod_div=2 ** 31), "17 is out of range"),
                         (lambda: tsd.op_fp4_absmax(x, None), "2 is missing"),
                         (lambda: tsd.op_fp4_gemm(x, x, x, x, MX, x, x_amax=3), "11 is not a tensor")):
        with pytest.raises(ValueError, match=f"argument {number}"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_tensor_factor_is_torch_s(seed):
    """The factor of a tensor's absolute maximum as torch computes it: values next to a border between two codes go the same way."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = 0.05 * torch.randn(2048, 1536, device=DEV, generator=g)
    amax = torch.empty(1, device=DEV)
    tsd.op_fp4_absmax(x, amax)
    assert amax.item() == x.abs().max().item()
    c, t = dev_quantize(x, NV, amax)
    z = x * (2688.0 / amax)
    c1, t1 = dev_quantize(z, NV)                                # without a factor: the same blocks
    assert torch.equal(c, c1) and torch.equal(t, t1)
