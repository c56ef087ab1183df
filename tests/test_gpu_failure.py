"""Failure detection on the GPU without a GPU fault.

Every device-side wait in the library is bounded (tsd_set_wait_limit, 2 s by default): a wait that
runs out records an error code in a device error word and its kernel returns, so the context
stays usable and the host reports TSD_ERR_DEVICE. Here the head-parallel arrival wait is made to
run out on purpose (its counters are a buffer nothing writes), with a short limit, and a normal
forward runs afterwards on the same GPU and gives the same result as before.
"""
import time

import numpy as np
import pytest
import torch

from tsd_b200 import synth, tsd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALL = dict(hidden=128, n_head=2, depth=3, fused_depth=1, ffn=256)
SHAPE = dict(T=20, clip_S=8, sync_S=24, text_S=77, t5_S=9)


@pytest.fixture
def short_wait_limit():
    tsd.set_wait_limit(0, 100_000_000)          # 100 ms
    yield 0.1
    tsd.set_wait_limit(0, 2_000_000_000)        # back to the default


def test_peer_wait_runs_out_and_reports(short_wait_limit):
    hp = synth.DitHParams(**SMALL)
    W = synth.make_weights(hp, seed=5, wtype="bf16")
    items = synth.make_inputs(hp, seed=6, batch=2, **SHAPE)
    m = tsd.DitModel.from_weights(hp, W)
    before = m.forward(items)

    counters = torch.zeros(8, dtype=torch.int32, device=DEV)   # rank 1's arrivals: never written
    epoch = torch.ones(1, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tsd.op_peer_wait(counters, epoch, rank=0, world=2, ctas=1, err=err)
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    assert int(err.item()) != 0                       # the wait gave up and said so
    assert short_wait_limit * 0.9 <= dt < 1.5, dt     # after the short limit, not the 2 s default

    # arrivals that did happen satisfy the same wait at once
    counters[1] = 1
    err.zero_()
    tsd.op_peer_wait(counters, epoch, rank=0, world=2, ctas=1, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0

    # the GPU and the model are unaffected
    after = m.forward(items)
    assert np.array_equal(before, after)
    m.close()


def test_wait_limit_is_restored(short_wait_limit):
    tsd.set_wait_limit(0, 2_000_000_000)
    counters = torch.zeros(8, dtype=torch.int32, device=DEV)
    counters[1] = 3
    epoch = torch.full((1,), 3, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    tsd.op_peer_wait(counters, epoch, rank=0, world=2, ctas=1, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0


def ones4(rows, K):
    """A 4-bit tensor of ones on the device: codes, scales (rows 1 or a multiple of 128, K a multiple of 128)."""
    codes = torch.full((rows, K // 2), 0x22, device=DEV, dtype=torch.uint8)
    scales = torch.full((tsd.fp4_scale_bytes(rows, K, tsd.FP4_MX),), 127, device=DEV, dtype=torch.uint8)
    if rows == 1:
        scales.view(-1, 512)[:, 4:] = 0
    return codes, scales


# One tile whose sums take longer than the limit: a CTA's of 128 x 64, 65536 stages of 512 elements; those of 38 pairs of CTAs, 8192
# stages of 256 that have to bring 10 GB from memory (1.5 ms at 7 TB/s) and need 8192 x 512 cycles of the tensor cores; those
# of 128 CTAs of 128 x 128, 17 GB.
LONG_PRODUCTS = [(1, 1, 2 ** 25), (256, 9728, 2 ** 21), (128, 16384, 2 ** 21)]


@pytest.mark.parametrize("N,M,K", LONG_PRODUCTS)
def test_fp4_gemm_wait_that_runs_out_reports_and_leaves_the_gpu_usable(N, M, K):
    """The epilogue's wait for the sums is longer than the limit of 1 ms: the roles stop, what they have in flight lands, the
    kernel returns and the same call with the usual limit is right, as are others after it."""
    X, W = ones4(N, K), ones4(M, K)
    out, err = torch.zeros(N, M, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    small = ones4(128, 512)
    ref = torch.zeros(128, 128, device=DEV)
    torch.cuda.synchronize()
    tsd.set_wait_limit(0, 1_000_000)
    try:
        t0 = time.perf_counter()
        tsd.op_fp4_gemm(*W, *X, tsd.FP4_MX, out, err=err)
        tsd.op_fp4_gemm(*small, *small, tsd.FP4_MX, ref)      # right behind it, on the same SMs
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
    finally:
        tsd.set_wait_limit(0, 2_000_000_000)
    assert int(err.item()) != 0
    assert dt < 1.0, dt
    assert (ref == 512).all()
    err.zero_()
    tsd.op_fp4_gemm(*W, *X, tsd.FP4_MX, out, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0 and (out == K).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", [tsd.EPI_STORE, tsd.EPI_SWIGLU])
@pytest.mark.parametrize("N,M,K", [(1, 2, 2 ** 25), (250, 9728, 2 ** 21), (250, 19456, 2 ** 21)])
def test_fp4_gemm_wait_that_runs_out_leaves_nan(N, M, K, mode, dtype):
    """With and without an error word: an output is what it would be or NaN, never what lay there before; nothing around the
    outputs is written. One tile, one tile for each pair of CTAs, and two for some."""
    codes, scales = ones4(128 if M == 2 else M, K)
    W = codes[:M], scales
    if M == 2:
        scales.view(-1, 32, 16)[:, 2:] = 0                     # two of the tile's 128 rows
        scales.view(-1, 32, 16)[:, :, 4:] = 0
    xc, xs = ones4(1 if N == 1 else 256, K)
    if N == 250:                                               # rows past the end of the last row tile: no scales
        t = xs.view(2, -1, 32, 4, 4)
        for r in range(250 - 128, 128):
            t[1, :, r % 32, r // 32] = 0
    X = xc[:N], xs
    cols = M if mode == tsd.EPI_STORE else M // 2
    want = float(K) if mode == tsd.EPI_STORE else float(K) ** 2
    buf = torch.full((N, cols + 32), 5.0, device=DEV, dtype=dtype)
    out = buf[:, :cols]
    torch.cuda.synchronize()
    tsd.set_wait_limit(0, 1_000_000)
    try:
        tsd.op_fp4_gemm(*W, *X, tsd.FP4_MX, out, mode=mode)
        torch.cuda.synchronize()
    finally:
        tsd.set_wait_limit(0, 2_000_000_000)
    lost = torch.isnan(out)
    assert lost.any() and (out[~lost] == want).all()
    assert (buf[:, cols:] == 5.0).all()
    tsd.op_fp4_gemm(*W, *X, tsd.FP4_MX, out, mode=mode)
    assert (out == want).all()
