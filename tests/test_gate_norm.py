"""tsd_op_gate_norm (norm after a block, gate and residual scales, norm and modulation before the next
block) against the formula in 64 bits, and its refusals.

Tolerances. u = 2^-24 is half an f32 step. The kernel sums H terms in chains of at most 16 terms per
thread, 5 shuffle steps and 32 warp sums: a sum is off by at most c u sum|terms| with c = 16 + 5 + 32,
the mean by c u mean|v|, and 1 / sqrt(mean square + eps) by (c + 4) u relative plus what the errors of
the centred values bring. The rest is a handful of single roundings. The bounds below add these up
element by element; a 16-bit output adds half its step."""
import ctypes

import pytest
import torch

from tsd_b200 import tsd

DEV = "cuda:0"
U = 2.0 ** -24
C = 16 + 5 + 32
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ref_norm(v, kind, eps, err):
    """(norm, bound on its error) of rows v (f64) that are themselves known to within err."""
    if kind == tsd.NORM_NONE:
        return v, err
    if kind == tsd.NORM_LAYER:
        # the mean's error, then one subtraction
        merr = C * U * v.abs().mean(-1, keepdim=True) + err.mean(-1, keepdim=True)
        d = v - v.mean(-1, keepdim=True)
        err = err + merr + U * d.abs()
    else:
        d = v
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    n = d * r
    # d(1/r^2) = 2 mean(|d| err) + mean(err^2): relative error of r is half of that times r^2
    rrel = (C + 4) * U + 0.5 * r * r * (2 * (d.abs() * err).mean(-1, keepdim=True) + (err * err).mean(-1, keepdim=True))
    return n, r * err + n.abs() * (rrel + 2 * U) + r * err * rrel


def reference(x, y, a):
    """x', its bound, h, its bound in f64 for the keyword arguments `a` of op_gate_norm."""
    rows, H = x.shape
    f = lambda t: None if t is None else t.double()   # noqa: E731

    def per_row(t, div):
        return t[None, :] if t.dim() == 1 else t[torch.arange(rows, device=t.device) // div]

    xv = a["x_scale"] * x.double()
    xerr = U * xv.abs()
    if y is not None:
        yv = y.double()
        b, be = ref_norm(yv, a["post_norm"], a["post_eps"], torch.zeros_like(yv))
        for t in (f(a["post_gain"]), None if a["gate"] is None else per_row(f(a["gate"]), a["gate_div"])):
            if t is not None:
                b, be = b * t, be * t.abs() + 2 * U * (b * t).abs()
        xv = xv + a["y_scale"] * b
        xerr = xerr + abs(a["y_scale"]) * be + 2 * U * ((a["y_scale"] * b).abs() + xv.abs())
    h, he = ref_norm(xv, a["pre_norm"], a["pre_eps"], xerr)
    if a["pre_gain"] is not None:
        t = f(a["pre_gain"])
        h, he = h * t, he * t.abs() + 2 * U * (h * t).abs()
    if a["scale"] is not None:
        t = 1 + per_row(f(a["scale"]), a["mod_div"])
        h, he = h * t, he * t.abs() + 3 * U * (h * t).abs()
        he = he + U * h.abs() / t.abs().clamp(min=1e-3)       # the rounding of 1 + scale itself
    if a["shift"] is not None:
        t = per_row(f(a["shift"]), a["mod_div"])
        he = he + U * ((h + t).abs() + h.abs())
        h = h + t
    return xv, xerr, h, he


def args(**kw):
    d = dict(post_norm=tsd.NORM_NONE, post_gain=None, post_eps=1e-5, gate=None, gate_div=1, x_scale=1.0, y_scale=1.0,
             pre_norm=tsd.NORM_NONE, pre_gain=None, pre_eps=1e-6, shift=None, scale=None, mod_div=1)
    d.update(kw)
    return d


def check(x, y, x_out, h, a):
    xv, xe, hv, he = reference(x, y, a)
    if x_out is not None:
        bad = (x_out.double() - xv).abs() > xe
        assert not bad.any(), ("x_out", int(bad.sum()), float(((x_out.double() - xv).abs() / xe.clamp(min=1e-300)).max()))
    if h is not None:
        he = he + (0 if h.dtype == torch.float32 else (hv.abs() + he) * torch.finfo(h.dtype).eps / 2)
        if h.dtype == torch.float16:
            he = he + 2.0 ** -25                              # half a step of its subnormals
        bad = (h.double() - hv).abs() > he
        assert not bad.any(), ("h", int(bad.sum()), float(((h.double() - hv).abs() / he.clamp(min=1e-300)).max()))


def run(x, y, x_out, h, a, stream=0):
    tsd.op_gate_norm(x, y, x_out, h, stream=stream, **a)


def make(rows, H, seed, post, pre, gate, mod, div=3, gains=True, x_scale=0.75, y_scale=-1.25):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    shape = {"vector": (H,), "item": (-(-rows // div), H), "token": (rows, H)}
    a = args(post_norm=post, pre_norm=pre, x_scale=x_scale, y_scale=y_scale,
             post_gain=1 + 0.2 * n(H) if gains else None, pre_gain=1 + 0.2 * n(H) if gains else None)
    if gate:
        a.update(gate=n(*shape[gate]), gate_div=div if gate == "item" else 1)
    if mod:
        a.update(shift=n(*shape[mod]), scale=n(*shape[mod]), mod_div=div if mod == "item" else 1)
    return 3 * n(rows, H) + 1, n(rows, H), a


NORMS = [tsd.NORM_NONE, tsd.NORM_LAYER, tsd.NORM_RMS]
SHAPES = [(1, 1), (2, 2), (3, 5), (7, 33), (4, 64), (5, 1023), (1, 1536), (388, 1536), (2, 1024), (3, 4095), (3, 4100),
          (9, 8192), (2, 16383), (2, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,H", SHAPES)
@pytest.mark.parametrize("post,pre", [(0, 1), (1, 2), (2, 1), (2, 0)])
def test_shapes_and_norms(rows, H, post, pre):
    x, y, a = make(rows, H, 1, NORMS[post], NORMS[pre], "token", "token")
    x_out, h = torch.empty_like(x), torch.empty(rows, H, device=DEV)
    run(x, y, x_out, h, a)
    check(x, y, x_out, h, a)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,H", [(1024, 1536), (1100, 4), (1500, 2052), (1024, 6144), (1027, 6148), (3, 2052), (3, 4096), (5, 6148),
                                    (1025, 384), (1031, 388), (1026, 7), (1024, 256), (1029, 257), (4, 8190), (3, 8192), (2, 8196), (5, 4097), (2, 9001)])
def test_elements_per_thread(rows, H):
    """As above for the numbers of rows and widths at which a thread takes another number of elements."""
    x, y, a = make(rows, H, rows + H, tsd.NORM_RMS, tsd.NORM_LAYER, "token", "item")
    x_out, h = torch.full_like(x, float("nan")), torch.full((rows, H), float("nan"), device=DEV, dtype=torch.bfloat16)
    y = y.half()
    run(x, y, x_out, h, a)
    check(x, y, x_out, h, a)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [1536, 51])
def test_offsets_past_32_bits(H):
    """Row strides of 2^31 elements: offsets in elements and in bytes leave 32 bits."""
    ld = 2 ** 31
    far = lambda dt: torch.empty(ld + H, device=DEV, dtype=dt).as_strided((2, H), (ld, 1))   # noqa: E731
    x, y, a = make(2, H, H, tsd.NORM_LAYER, tsd.NORM_RMS, "token", "token")
    fx, fy, fh = far(torch.float32), far(torch.bfloat16), far(torch.float16)
    fx.copy_(x), fy.copy_(y), fh.fill_(float("nan"))
    run(fx, fy, fx, fh, a)
    check(x, y.bfloat16(), fx, fh, a)


@pytest.mark.gpu
@pytest.mark.parametrize("yt", list(DT))
@pytest.mark.parametrize("ht", list(DT))
@pytest.mark.parametrize("gate,mod", [(None, None), ("vector", "vector"), ("item", "token"), ("token", "item")])
@pytest.mark.parametrize("H", [48, 51, 1536])
def test_types_gates_and_modulations(yt, ht, gate, mod, H):
    x, y, a = make(10, H, 2, tsd.NORM_RMS, tsd.NORM_LAYER, gate, mod, gains=gate is None)
    y = y.to(DT[yt])
    x_out, h = torch.empty_like(x), torch.empty(10, H, device=DEV, dtype=DT[ht])
    run(x, y, x_out, h, a)
    check(x, y, x_out, h, a)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [96, 97, 5000])
def test_optional_outputs_and_inputs(H):
    x, y, a = make(6, H, 3, tsd.NORM_LAYER, tsd.NORM_RMS, "token", "token")
    full_x, full_h = torch.empty_like(x), torch.empty(6, H, device=DEV)
    run(x, y, full_x, full_h, a)
    h = torch.empty_like(full_h)
    run(x, y, None, h, a)                                      # h alone: the same bits
    assert torch.equal(h, full_h)
    only = dict(a, pre_norm=tsd.NORM_NONE, pre_gain=None, shift=None, scale=None)
    x_out = torch.empty_like(x)
    run(x, y, x_out, None, only)                               # the update alone
    assert torch.equal(x_out, full_x)
    first = args(x_scale=1.0, pre_norm=tsd.NORM_LAYER, pre_eps=1e-5, shift=a["shift"], scale=a["scale"])
    run(x, None, None, h, first)                               # no block before: norm and modulation of x
    check(x, None, None, h, first)
    one = dict(first, shift=None)
    run(x, None, x_out, h, one)
    check(x, None, x_out, h, one)
    assert torch.equal(x_out, x)
    x2 = x.clone()
    run(x2, y, x2, h, a)                                       # in place
    assert torch.equal(x2, full_x) and torch.equal(h, full_h)


@pytest.mark.gpu
def test_norm_and_modulation_equal_the_framework_s_ln_modulate():
    x, _, a = make(20, 1536, 4, tsd.NORM_NONE, tsd.NORM_LAYER, None, "item", div=5, gains=False)
    ref = torch.empty(20, 1536, device=DEV, dtype=torch.bfloat16)
    tsd.op_ln_modulate(x, 20, 1536, a["shift"], a["scale"], 1536, 0, 5, ref)
    h = torch.empty_like(ref)
    run(x, None, None, h, dict(a, x_scale=1.0, pre_eps=1e-5))
    # two f32 computations of one value, each rounded once: at most one bf16 step apart
    assert ((h.float() - ref.float()).abs() <= ref.float().abs() * torch.finfo(torch.bfloat16).eps).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,pad,off", [(64, 32, 0), (64, 5, 0), (64, 32, 1), (67, 13, 3), (1536, 4, 4), (1536, 4, 2)])
def test_strides_alignment_and_what_lies_around(H, pad, off):
    """Operands in the middle of wider buffers; nothing outside the outputs is written."""
    rows = 9
    x, y, a = make(rows, H, 5, tsd.NORM_RMS, tsd.NORM_LAYER, "token", "token")

    def wide(t, dtype):
        buf = torch.full((rows + 2, H + pad), 7.0, device=DEV, dtype=dtype)
        flat = buf.view(-1)
        v = flat[off:off + (rows + 1) * (H + pad)].view(rows + 1, H + pad)[:rows, :H]
        if t is not None:
            v.copy_(t)
        return buf, v

    for ht in (torch.float32, torch.bfloat16):
        _, xs = wide(x, torch.float32)
        _, ys = wide(y, torch.bfloat16)
        _, gs = wide(a["gate"], torch.float32)
        _, ss = wide(a["shift"], torch.float32)
        _, cs = wide(a["scale"], torch.float32)
        ob, xo = wide(None, torch.float32)
        hb, h = wide(None, ht)
        b = dict(a, gate=gs, shift=ss, scale=cs)
        run(xs, ys, xo, h, b)
        check(xs, ys, xo, h, b)
        for buf, v in ((ob, xo), (hb, h)):
            got = v.clone()
            v.fill_(7.0)
            assert (buf == 7.0).all()
            v.copy_(got)


@pytest.mark.gpu
def test_constant_rows_large_means_and_zero_rows():
    H = 1000
    x = torch.zeros(5, H, device=DEV)
    x[1] = 5.0                                                 # no variance
    x[2] = 1e4 + torch.randn(H, device=DEV)                    # a mean far above the deviations
    x[3] = 1e-20                                               # far below eps
    x[4] = torch.randn(H, device=DEV) * 1e15
    for kind in (tsd.NORM_LAYER, tsd.NORM_RMS):
        a = args(pre_norm=kind, pre_eps=1e-5)
        h = torch.empty_like(x)
        run(x, None, None, h, a)
        check(x, None, None, h, a)
        if kind == tsd.NORM_LAYER:
            assert (h[0] == 0).all() and (h[1] == 0).all()


@pytest.mark.gpu
def test_rows_that_are_not_finite_stay_alone():
    x, y, a = make(6, 300, 6, tsd.NORM_LAYER, tsd.NORM_RMS, "token", None)
    clean_x, clean_h = torch.empty_like(x), torch.empty_like(x)
    run(x, y, clean_x, clean_h, a)
    x[1, 7], y[3, 200], a["gate"][4, 0] = float("nan"), float("inf"), float("nan")
    x_out, h = torch.empty_like(x), torch.empty_like(x)
    run(x, y, x_out, h, a)
    for r in (0, 2, 5):
        assert torch.equal(x_out[r], clean_x[r]) and torch.equal(h[r], clean_h[r])
    for r in (1, 3, 4):
        assert torch.isnan(h[r]).any()


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    x, y, a = make(64, 1536, 7, tsd.NORM_RMS, tsd.NORM_LAYER, "token", "token")
    x_out, h = torch.empty_like(x), torch.empty(64, 1536, device=DEV, dtype=torch.bfloat16)
    run(x, y, x_out, h, a)
    want = x_out.clone(), h.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x_out.zero_(), h.zero_()
        run(x, y, x_out, h, a, s.cuda_stream)
    s.synchronize()
    assert torch.equal(x_out, want[0]) and torch.equal(h, want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(x, y, x_out, h, a, torch.cuda.current_stream().cuda_stream)
        run(x_out, y, x_out, h, a, torch.cuda.current_stream().cuda_stream)
    x.mul_(0.5)                                                # the graph reads what is there when it runs
    g.replay()
    ref_x, ref_h = torch.empty_like(x), torch.empty_like(h)
    run(x, y, ref_x, ref_h, a)
    run(ref_x, y, ref_x, ref_h, a)
    torch.cuda.synchronize()
    assert torch.equal(x_out, ref_x) and torch.equal(h, ref_h)


@pytest.mark.gpu
def test_no_rows_and_host_memory():
    x = torch.zeros(0, 64, device=DEV)
    tsd.op_gate_norm(x, None, None, torch.zeros(0, 64, device=DEV), pre_norm=tsd.NORM_RMS)
    x = torch.zeros(2, 64, device=DEV)
    with pytest.raises(tsd.TsdError, match="TSD_ERR_ARG"):
        tsd.op_gate_norm(x, torch.zeros(2, 64), x, None)       # y in pageable host memory


# ------------------------------------------------------------------------------------ without a GPU
def raw(**kw):
    """tsd_op_gate_norm on addresses that nothing may touch; a valid call except for `kw`."""
    d = dict(x=4096, ldx=64, y=8192, y_type=30, ldy=64, rows=4, H=64, post_norm=2, post_gain=None, post_eps=1e-6,
             gate=12288, ldg=64, gate_div=1, x_scale=1.0, y_scale=1.0, x_out=4096, ldxo=64, pre_norm=1, pre_gain=None,
             pre_eps=1e-6, shift=16384, scale=20480, ld_mod=64, mod_div=1, h=24576, h_type=30, ldh=64, stream=None)
    d.update(kw)
    return tsd.lib().tsd_op_gate_norm(*d.values())


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(x_out=None, h=None), dict(rows=-1), dict(H=0), dict(H=16385, ldx=20000, ldy=20000, ldxo=20000, ldh=20000),
    dict(ldx=63, ldxo=63), dict(ldy=63), dict(ldxo=65), dict(x_out=40960, ldxo=10), dict(ldh=1), dict(ldg=63), dict(ldg=-64),
    dict(ld_mod=5), dict(gate_div=0), dict(mod_div=0), dict(post_norm=3), dict(pre_norm=-1), dict(post_eps=-1e-6),
    dict(pre_eps=float("nan")), dict(y_type=8), dict(h_type=2), dict(h=4096), dict(h=8192), dict(x_out=8192),
    dict(y=None), dict(y=None, post_norm=0), dict(h=None), dict(h=None, pre_norm=0), dict(x=4098), dict(y=8193),
    dict(gate=12290), dict(shift=16385), dict(h=24577),
])
def test_refusals(kw):
    assert raw(**kw) == -1


def test_no_rows_needs_no_device():
    assert raw(rows=0) == 0


def test_wrapper_refuses_shapes_and_types():
    x, v = torch.zeros(4, 8), torch.zeros(8)
    h = torch.zeros(4, 8)
    for a, kw in [((x.half(), None, None, h), {}), ((x, x[:3], x, h), {}), ((x, None, x.half(), h), {}),
                  ((x, None, None, h[:, :4]), {}), ((x.t(), None, None, h.t()), {}), ((x, x, None, h), dict(post_gain=v[:7])),
                  ((x, x, None, h), dict(gate=torch.zeros(3, 8))), ((x, x, None, h), dict(gate=torch.zeros(1, 8), gate_div=3)),
                  ((x, x, None, h), dict(gate=v.double())), ((x, None, None, h), dict(shift=v, scale=x)),
                  ((x, None, None, h), dict(shift=v[::2]))]:
        with pytest.raises(ValueError):
            tsd.op_gate_norm(*a, **kw)
    with pytest.raises(tsd.TsdError):                          # a type that no operator takes
        tsd.op_gate_norm(x, None, None, torch.zeros(4, 8, dtype=torch.float64))


def test_the_bound_notices_a_wrong_result():
    """The oracle's own check: a value moved by a few f32 steps, a norm without its eps, a gate of the next row."""
    torch.manual_seed(0)
    x, y = torch.randn(4, 50), torch.randn(4, 50)
    a = args(post_norm=tsd.NORM_RMS, pre_norm=tsd.NORM_LAYER, gate=torch.randn(4, 50), x_scale=0.5)
    xv, xe, hv, he = reference(x, y, a)
    check(x, y, xv.float(), hv.float(), a)
    moved = hv.clone()
    moved[2, 3] += 2e-3
    for bad in (dict(x_out=xv.float(), h=moved.float()), dict(x_out=reference(x, y, dict(a, gate=a["gate"].roll(1, 0)))[0].float(), h=None),
                dict(x_out=None, h=reference(x, y, dict(a, pre_eps=1e-2))[2].float())):
        with pytest.raises(AssertionError):
            check(x, y, bad["x_out"], bad["h"], a)


def test_ctypes_signature_has_every_argument():
    assert len(tsd.lib().tsd_op_gate_norm.argtypes) == 28
    assert tsd.lib().tsd_op_gate_norm.restype is ctypes.c_int
