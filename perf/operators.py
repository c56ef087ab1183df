"""The block-boundary norm and the 4-bit floating-point operators: cases, plain forms, exact values.

Five operators of include/tsd_ops.h are measured, by the names of their Python wrappers in
thinksound.cpp_b200/tsd.py:

  gn  op_gate_norm                       norm after a block, gate and residual scales, norm and
                                         modulation before the next block
  q   op_fp4_absmax, op_fp4_quantize,    a tensor put into 4 bits and read back
      op_fp4_dequantize
  mm  op_fp4_gemm                        product of two 4-bit operands (projections, FFN)
  mv  op_fp4_gemv                        4-bit weights times a few f32 vectors (single tokens)

A 4-bit tensor [rows][K] is held as codes e2m1 (two to a byte, the even element in the low half)
and one scale to a block of K: "mx" has blocks of 32 and scales 2^(b - 127), "nv" blocks of 16 and
e4m3 scales, with the tensor's absolute maximum as a further f32 scale. Scale bytes lie in tiles of
128 rows x 4 blocks of 512 bytes, row-tile by row-tile: byte (r % 32) * 16 + (r % 128) / 32 * 4 + j % 4.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = {"mx": 32, "nv": 16}
TINY = 2.0 ** -100          # an absolute maximum below this counts as none


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one vector of one request: what a norm costs where only latency counts
        _gn("gn_one_vector", 1, 1536, "bf16", "rms", True, "vector", "rms", True, "none", "bf16"),
        # latent stream of one CFG pair between two blocks: adaLN gate and modulation of every token
        _gn("gn_pair_adaln", 388, 1536, "bf16", "none", False, "token", "layer", False, "token", "bf16"),
        # one item's text tokens at an odd width, both norms with gains, gate and modulation of the item
        _gn("gn_text_odd", 77, 1023, "f16", "layer", True, "item", "rms", True, "item", "f32"),
        # latent stream of 64 prompts as CFG pairs: both norms, everything per token
        _gn("gn_batch", 24832, 1536, "bf16", "rms", True, "token", "layer", False, "token", "bf16"),
        # a projection's weights as they are loaded: maximum, 4 bits, and back to f32 to look at the loss
        dict(name="q_weights", op="q", rows=4608, K=1536, src="f32", fmt="nv", amax=True, dst="f32"),
        # activations of 64 prompts on their way into a projection
        dict(name="q_batch", op="q", rows=24832, K=1536, src="bf16", fmt="mx", amax=False, dst="bf16"),
        # FFN entry of one CFG pair
        dict(name="mm_pair_swiglu", op="mm", N=388, M=8192, K=1536, fmt="mx", mode="swiglu", bias=False, amax=False, dst="bf16"),
        # FFN exit of one CFG pair: few tokens, long K
        dict(name="mm_pair_down", op="mm", N=388, M=1536, K=4096, fmt="nv", mode="store", bias=True, amax=True, dst="f32"),
        # one item's text tokens, sizes that end inside every tile
        dict(name="mm_text_ragged", op="mm", N=77, M=1000, K=2080, fmt="nv", mode="silu", bias=True, amax=True, dst="f32"),
        # QKV-sized and wider projection of 64 prompts
        dict(name="mm_batch", op="mm", N=24832, M=8192, K=1536, fmt="nv", mode="store", bias=True, amax=True, dst="bf16"),
        # all joint blocks' clip and text adaLN rows from one conditioning vector
        dict(name="mv_adaln", op="mv", N=1, M=129024, K=1536, fmt="nv", mode="store", bias=True, amax=True, dst="f32"),
        # a conditioning projection for a few vectors
        dict(name="mv_three", op="mv", N=3, M=1000, K=2080, fmt="mx", mode="silu", bias=True, amax=False, dst="bf16"),
    ]


def _gn(name, rows, H, y, post, post_gain, gate, pre, pre_gain, mod, dst):
    """gate / mod: "none", "vector" (one [H]), "item" (a row for each 97 rows) or "token" (a row for each row)."""
    return dict(name=name, op="gn", rows=rows, H=H, y=y, post=post, post_gain=post_gain, gate=gate, pre=pre,
                pre_gain=pre_gain, mod=mod, dst=dst)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gn", "q", "mm", "mv"])
    if op == "gn":
        H = _log(rng, 8, 8192)
        if rng.random() < 0.6:
            H = -(-H // 8) * 8
        c = _gn("", _log(rng, 1, min(24832, 24832 * 1536 // H)), H, rng.choice(["f32", "bf16", "f16"]),
                rng.choice(["none", "layer", "rms"]), rng.random() < 0.5, rng.choice(["none", "vector", "item", "token"]),
                rng.choice(["layer", "rms"]), rng.random() < 0.5, rng.choice(["none", "vector", "item", "token"]),
                rng.choice(["f32", "bf16", "f16"]))
        del c["name"]
        return c
    K = 32 * _log(rng, 1, 384)
    fmt = rng.choice(["mx", "nv"])
    if op == "q":
        return dict(op="q", rows=_log(rng, 1, min(24832, 24832 * 1536 // K)), K=K, src=rng.choice(["f32", "bf16", "f16"]),
                    fmt=fmt, amax=fmt == "nv" and rng.random() < 0.5, dst=rng.choice(["f32", "bf16"]))
    if op == "mm":
        M = _log(rng, 1, 12288)
        N = _log(rng, 1, min(24832, 24832 * 8192 * 1536 // (M * K)))
        mode = rng.choice(["store", "silu", "swiglu"])
        return dict(op="mm", N=N, M=M + M % 2 if mode == "swiglu" else M, K=K, fmt=fmt, mode=mode,
                    bias=mode != "swiglu" and rng.random() < 0.5, amax=fmt == "nv" and rng.random() < 0.5,
                    dst="bf16" if mode == "swiglu" else rng.choice(["f32", "bf16"]))
    return dict(op="mv", N=rng.randint(1, 8), M=_log(rng, 1, min(129024, 129024 * 1536 // K)), K=K, fmt=fmt,
                mode=rng.choice(["store", "silu"]), bias=rng.random() < 0.5, amax=fmt == "nv" and rng.random() < 0.5,
                dst=rng.choice(["f32", "bf16"]))


# ------------------------------------------------------------------------------------ the 4-bit format
def _scale_places(rows, K, fmt, dev):
    """Where the scale byte of row r, block j lies: [rows][K / block]."""
    nb = K // BLOCK[fmt]
    r = torch.arange(rows, device=dev, dtype=torch.int64)[:, None]
    j = torch.arange(nb, device=dev, dtype=torch.int64)[None, :]
    return (r // 128 * (-(-nb // 4)) + j // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + j % 4


def _scale_bytes(rows, K, fmt):
    return -(-rows // 128) * -(-(K // BLOCK[fmt]) // 4) * 512


def _scale_values(b, fmt):
    """Scale bytes as f32."""
    b = b.to(torch.int32)
    one = torch.ones((), device=b.device, dtype=torch.float64)
    if fmt == "mx":
        return torch.ldexp(one, b - 127).float()
    e, m = b >> 3, b & 7
    return torch.where(e > 0, torch.ldexp(1 + m.double() / 8, e - 7), m.double() / 512).float()


def _enc(amax):
    """The factor that brings a tensor of this absolute maximum to 448 * 6, in f32 (1 for none)."""
    return torch.where(amax >= TINY, 2688.0 / amax, torch.ones_like(amax))


def _dec(amax):
    return torch.where(amax >= TINY, amax / 2688.0, torch.ones_like(amax))


def _blocks(x, fmt, amax):
    """x as f32 blocks [rows][nb][block], scaled by the tensor's factor, and the blocks' scales (f32)."""
    z = x.float()
    if amax is not None:
        z = z * _enc(amax)
    z = z.reshape(x.shape[0], -1, BLOCK[fmt])
    top = z.abs().amax(-1)
    if fmt == "mx":   # 2^(floor(log2 top) - 2), at least 2^-127
        _, e = torch.frexp(top)
        s = torch.ldexp(torch.ones_like(top, dtype=torch.float64), torch.where(top > 0, (e - 3).clamp(min=-127), -127))
    else:             # top / 6 rounded to e4m3: in 64 bits, so that nothing next to a border moves over it
        t = top.double() / 6
        _, e = torch.frexp(t)
        step = torch.ldexp(torch.ones_like(t), (e - 1).clamp(min=-6) - 3)
        s = (torch.round(t / step) * step).clamp(max=448.0)
    return z, s.float()


def _round4(z, s):
    """z / s rounded to e2m1 (ties to the even code), in 64 bits for the borders."""
    s = s.double()[..., None]
    y = torch.where(s > 0, z.double() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(s))
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, y).float()


def _pack(v, s, fmt):
    """Values on the e2m1 grid [rows][nb][block] and scales [rows][nb] as the bytes of a 4-bit tensor."""
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.reshape(v.shape[0], -1)
    q = code[:, 0::2] | (code[:, 1::2] << 4)
    _, e = torch.frexp(s)
    e = e - 1
    if fmt == "mx":
        b = (e + 127).to(torch.uint8)
    else:
        b = torch.where(s < 2.0 ** -6, s * 512, (e + 7).float() * 8 + torch.ldexp(s, 3 - e) - 8).to(torch.uint8)
    K = code.shape[1]
    tiles = torch.zeros(_scale_bytes(v.shape[0], K, fmt), dtype=torch.uint8, device=v.device)
    tiles[_scale_places(v.shape[0], K, fmt, v.device).reshape(-1)] = b.reshape(-1)
    return q.contiguous(), tiles


def _unpack(q, tiles, fmt):
    """A 4-bit tensor without its tensor scale, as f32 [rows][K]."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=q.device)
    codes = torch.stack([q & 15, q >> 4], dim=-1).reshape(q.shape[0], -1)
    s = _scale_values(tiles[_scale_places(codes.shape[0], codes.shape[1], fmt, q.device)], fmt)
    return (grid[codes.to(torch.int32)].reshape(q.shape[0], -1, BLOCK[fmt]) * s[..., None]).reshape(codes.shape)


def _make4(x, fmt, amax):
    z, s = _blocks(x, fmt, amax)
    return _pack(_round4(z, s), s, fmt)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    c, st = case, dict(case=case)
    if c["op"] == "gn":
        R, H = c["rows"], c["H"]
        st["x"] = 3.0 * normal(R, H) + normal(1, H)
        st["y"] = normal(R, H).to(TYPES[c["y"]])
        for k in ("post", "pre"):
            st[k + "_gain"] = 1.0 + 0.1 * normal(H) if c[k + "_gain"] and c[k] != "none" else None
        items = -(-R // 97)
        shape = {"vector": (H,), "item": (items, H), "token": (R, H)}
        st["gate"] = None if c["gate"] == "none" else 0.5 * normal(*shape[c["gate"]])
        st["shift"], st["scale"] = (None, None) if c["mod"] == "none" else (0.2 * normal(*shape[c["mod"]]), 0.2 * normal(*shape[c["mod"]]))
        st["x_out"] = torch.empty(R, H, device="cuda")
        st["h"] = torch.empty(R, H, device="cuda", dtype=TYPES[c["dst"]])
        return st
    K, fmt = c["K"], c["fmt"]
    if c["op"] == "q":
        R = c["rows"]
        x = normal(R, K) * torch.exp(0.5 * normal(1, K))      # channels of unlike size, as activations have them
        st["x"] = (0.02 * x if c["src"] == "f32" else x).to(TYPES[c["src"]])
        st["amax"] = torch.empty(1, device="cuda") if c["amax"] else None
        st["q"] = torch.empty(R, K // 2, device="cuda", dtype=torch.uint8)
        st["tiles"] = torch.empty(_scale_bytes(R, K, fmt), device="cuda", dtype=torch.uint8)
        st["out"] = torch.empty(R, K, device="cuda", dtype=TYPES[c["dst"]])
        return st
    N, M = c["N"], c["M"]
    w = 0.02 * normal(M, K)
    st["w_amax"] = w.abs().max().reshape(1) if c["amax"] else None
    st["w"], st["w_tiles"] = _make4(w, fmt, st["w_amax"])
    del w
    st["bias"] = 0.1 * normal(M) if c["bias"] else None
    x = normal(N, K) * torch.exp(0.5 * normal(1, K))
    st["x"] = x
    if c["op"] == "mm":
        st["x_amax"] = x.abs().max().reshape(1) if c["amax"] else None
        st["x"], st["x_tiles"] = _make4(x.to(torch.bfloat16), fmt, st["x_amax"])
    st["out"] = torch.empty(N, M // 2 if c["mode"] == "swiglu" else M, device="cuda", dtype=TYPES[c["dst"]])
    return st


# ------------------------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _run_own(st)
    c = st["case"]
    if c["op"] == "gn":
        x, h = _gate_norm(st, torch.float32)
        return {"x": x, "h": h.to(TYPES[c["dst"]])}
    if c["op"] == "q":
        amax = st["x"].float().abs().max().reshape(1) if c["amax"] else None
        z, s = _blocks(st["x"], c["fmt"], amax)
        v = (_round4(z, s) * s[..., None]).reshape(st["x"].shape)
        return (v if amax is None else v * _dec(amax)).to(TYPES[c["dst"]])
    w = _unpack(st["w"], st["w_tiles"], c["fmt"])
    x = _unpack(st["x"], st["x_tiles"], c["fmt"]) if c["op"] == "mm" else st["x"]
    y = x @ w.t()
    if st["w_amax"] is not None:
        y = y * (_dec(st["w_amax"]) * _dec(st["x_amax"]) if c["op"] == "mm" else _dec(st["w_amax"]))
    if st["bias"] is not None:
        y = y + st["bias"]
    return _activate(y, c["mode"]).to(TYPES[c["dst"]])


def _activate(y, mode):
    if mode == "silu":
        return y / (1 + torch.exp(-y))
    if mode == "swiglu":      # rows of w1 and w3 alternate
        a, b = y[:, 0::2], y[:, 1::2]
        return a / (1 + torch.exp(-a)) * b
    return y


def _norm(v, kind, gain):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    if kind != "none":
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + (1e-5 if kind == "layer" else 1e-6))
    return v if gain is None else v * gain


def _rows_of(t, kind, rows):
    """A gate or modulation [H], [items][H] or [rows][H] for every row."""
    return t.repeat_interleave(97, dim=0)[:rows] if kind == "item" else t


def _gate_norm(st, dtype):
    c = st["case"]
    a = {k: st[k].to(dtype) if st[k] is not None else None for k in ("x", "y", "post_gain", "gate", "pre_gain", "shift", "scale")}
    b = _norm(a["y"], c["post"], a["post_gain"])
    if a["gate"] is not None:
        b = b * _rows_of(a["gate"], c["gate"], c["rows"])
    x = 0.75 * a["x"] + 0.5 * b
    h = _norm(x, c["pre"], a["pre_gain"])
    if a["shift"] is not None:
        h = h * (1 + _rows_of(a["scale"], c["mod"], c["rows"])) + _rows_of(a["shift"], c["mod"], c["rows"])
    return x, h


def _run_own(st):
    tsd = _tsd()
    c, stream = st["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "gn":
        div = {"none": 1, "vector": 1, "token": 1, "item": 97}
        kinds = {"none": tsd.NORM_NONE, "layer": tsd.NORM_LAYER, "rms": tsd.NORM_RMS}
        eps = {"none": 0.0, "layer": 1e-5, "rms": 1e-6}
        tsd.op_gate_norm(st["x"], st["y"], st["x_out"], st["h"], post_norm=kinds[c["post"]], post_gain=st["post_gain"],
                         post_eps=eps[c["post"]], gate=st["gate"], gate_div=div[c["gate"]], x_scale=0.75, y_scale=0.5,
                         pre_norm=kinds[c["pre"]], pre_gain=st["pre_gain"], pre_eps=eps[c["pre"]], shift=st["shift"],
                         scale=st["scale"], mod_div=div[c["mod"]], stream=stream)
        return {"x": st["x_out"], "h": st["h"]}
    fmt = tsd.FP4_MX if c["fmt"] == "mx" else tsd.FP4_NV
    if c["op"] == "q":
        if st["amax"] is not None:
            tsd.op_fp4_absmax(st["x"], st["amax"], stream=stream)
        tsd.op_fp4_quantize(st["x"], fmt, st["q"], st["tiles"], amax=st["amax"], stream=stream)
        tsd.op_fp4_dequantize(st["q"], st["tiles"], fmt, st["out"], amax=st["amax"], stream=stream)
        return st["out"]
    act = tsd.ACT_SILU if c["mode"] == "silu" else tsd.ACT_NONE
    if c["op"] == "mm":
        tsd.op_fp4_gemm(st["w"], st["w_tiles"], st["x"], st["x_tiles"], fmt, st["out"],
                        mode=tsd.EPI_SWIGLU if c["mode"] == "swiglu" else tsd.EPI_STORE, act=act, bias=st["bias"],
                        w_amax=st["w_amax"], x_amax=st["x_amax"], stream=stream)
    else:
        tsd.op_fp4_gemv(st["w"], st["w_tiles"], fmt, st["x"], st["out"], bias=st["bias"], act=act, w_amax=st["w_amax"],
                        stream=stream)
    return st["out"]


_loaded = []


def _tsd():
    if not _loaded:
        import __graft_entry__
        __graft_entry__.load_package()
        from tsd_b200 import tsd
        _loaded.append(tsd)
    return _loaded[0]


# ------------------------------------------------------------------------------------ work
def work(case):
    c = case
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if c["op"] == "gn":
        n, H = c["rows"] * c["H"], c["H"]
        rows = {"none": 0, "vector": 1, "item": -(-c["rows"] // 97), "token": c["rows"]}
        par = rows[c["gate"]] + 2 * rows[c["mod"]] + (c["post_gain"] and c["post"] != "none") + c["pre_gain"]
        return {"bytes": n * (8 + size[c["y"]] + size[c["dst"]]) + 4 * H * par, "flops": 16 * n}
    if c["op"] == "q":
        n = c["rows"] * c["K"]
        return {"bytes": n * (size[c["src"]] + size[c["dst"]]), "flops": 6 * n}
    packed = 0.5 + 1 / BLOCK[c["fmt"]]
    outs = c["N"] * (c["M"] // 2 if c["mode"] == "swiglu" else c["M"])
    x = packed if c["op"] == "mm" else 4
    return {"bytes": c["M"] * c["K"] * packed + c["N"] * c["K"] * x + outs * size[c["dst"]] + 4 * c["M"] * c["bias"],
            "flops": 2 * c["N"] * c["M"] * c["K"]}


# ------------------------------------------------------------------------------------ the definitions in 64 bits
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(a, table):
    """Place in an ascending table of the entry nearest to a >= 0, the even place on a tie, the last beyond the end."""
    t = torch.tensor(table, dtype=torch.float64, device=a.device)
    mid = (t[1:] + t[:-1]) / 2
    low = torch.bucketize(a, mid)                       # the number of borders below a
    tie = (low < len(mid)) & (a == mid[low.clamp(max=len(mid) - 1)])
    return torch.where(tie & (low % 2 == 1), low + 1, low), t


E4M3 = [m / 512.0 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]


def _exact_decode(q, tiles, fmt):
    """Codes times block scales in f64, from the bytes."""
    rows, K = q.shape[0], 2 * q.shape[1]
    t = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=q.device)
    v = torch.empty(rows, K, dtype=torch.float64, device=q.device)
    v[:, 0::2], v[:, 1::2] = t[(q & 15).long()], t[(q >> 4).long()]
    nb = K // BLOCK[fmt]
    kt = -(-nb // 4)
    # tiles as [row tile][block tile][32 rows][4 groups of 32 rows][4 blocks]
    b = tiles.reshape(-1, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, kt * 4)[:rows, :nb].long()
    if fmt == "mx":
        s = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=q.device), (b - 127).double())
    else:
        s = torch.tensor(E4M3 + [float("nan")], dtype=torch.float64, device=q.device)[b]
    return v * s.repeat_interleave(BLOCK[fmt], dim=1)


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["op"] == "gn":
        x, h = [], []
        y64, x64 = st["y"].double(), st["x"].double()
        f = lambda k: None if st[k] is None else st[k].double()  # noqa: E731
        item = torch.arange(c["rows"], device="cuda") // 97
        at = lambda t, kind: t[item] if kind == "item" else t    # noqa: E731

        def normed(v, kind, gain):
            if kind == "layer":
                var, mean = torch.var_mean(v, dim=-1, correction=0, keepdim=True)
                v = (v - mean) / (var + 1e-5).sqrt()
            elif kind == "rms":
                v = v * (v.square().sum(-1, keepdim=True) / v.shape[-1] + 1e-6).rsqrt()
            return v if gain is None else v * gain

        b = normed(y64, c["post"], f("post_gain"))
        b = b if st["gate"] is None else b * at(f("gate"), c["gate"])
        x = x64 * 3 / 4 + b / 2
        h = normed(x, c["pre"], f("pre_gain"))
        if st["shift"] is not None:
            h = h + h * at(f("scale"), c["mod"]) + at(f("shift"), c["mod"])
        return {"x": x, "h": h}
    if c["op"] == "q":
        # the tensor's factor and the scaled tensor are f32 by definition; the rest is decided exactly
        x, dec = st["x"].float(), 1.0
        if c["amax"]:
            m = x.abs().max()
            if float(m) >= TINY:
                x, dec = x * (2688.0 / m), (m / 2688.0).double()
        z = x.double().reshape(c["rows"], -1, BLOCK[c["fmt"]])
        top = z.abs().amax(-1, keepdim=True)
        if c["fmt"] == "mx":
            one = torch.ones_like(top)
            e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149))).int()     # off by one next to a power of two
            e = torch.where(torch.ldexp(one, e) > top, e - 1, e)
            e = torch.where(torch.ldexp(one, e + 1) <= top, e + 1, e)
            s = torch.ldexp(one, (e - 2).clamp(min=-127))
        else:
            k, t = _nearest(top / 6, E4M3)
            s = t[k]
        k, t = _nearest(z.abs() / s.clamp(min=2.0 ** -140), GRID)
        return (torch.sign(z) * t[k] * s * dec).reshape(c["rows"], c["K"])
    w = _exact_decode(st["w"], st["w_tiles"], c["fmt"])
    if st["w_amax"] is not None:
        w *= _dec(st["w_amax"].double())
    if c["op"] == "mm":
        x = _exact_decode(st["x"], st["x_tiles"], c["fmt"])
        if st["x_amax"] is not None:
            x *= _dec(st["x_amax"].double())
    else:
        x = st["x"].double()
    y = x @ w.t()
    if st["bias"] is not None:
        y += st["bias"].double()
    if c["mode"] == "swiglu":
        return y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
    return y * torch.sigmoid(y) if c["mode"] == "silu" else y
