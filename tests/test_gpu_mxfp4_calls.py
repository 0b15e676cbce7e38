"""Calls of MXFP4 layers and products beside those of test_gpu_mxfp4.py.  Tolerances as there."""
import numpy as np
import pytest

import mimoe as M
from test_gpu_mxfp4 import LAYERS, Layer, rows

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = M.Context(0)
    c.reserve(160, 704, 448, 16, 8)
    yield c
    c.close()


def forward(ctx, lay, x, res=None, routing=None):
    T = len(x)
    out = M.DeviceBuffer(4 * T * lay.D)
    M.check("forward", ctx.forward(lay.L, M.to_device(x), T, None if res is None else M.to_device(res), out, routing))
    M.synchronize()
    return out.download(np.float32, (T, lay.D))


# ------------------------------------------------------------------ relu^2 of what is no number
@gpu
@pytest.mark.parametrize("threshold", [0, 1, 1 << 40])
@pytest.mark.parametrize("T", [1, 4, 20, 70])
@pytest.mark.parametrize("where", ["token", "routed", "shared"])
def test_relu_sqr_keeps_nan(ctx, where, T, threshold):
    """a token past the range of an fp16 scale, or a NaN block in a routed or the shared expert's first table: NaN in the
    rows that meet it on the few-row path and the GEMM alike, the other rows to the bit"""
    lay, bad = (Layer(seed=81, **LAYERS["nemotron_like"]) for _ in range(2))
    x = rows(np.random.default_rng(82), T, lay.D)
    hit = np.zeros(T, bool)
    xb = x
    if where == "token":
        hit[T // 2] = True
        xb = x.copy()
        xb[T // 2, 100] = 1e9
    elif where == "routed":
        e = lay.route(x)[0][0, 0]
        hit = (lay.route(x)[0] == e).any(1)
        raw = lay.host["gate"].copy()
        raw[e, 37, 17 * 3] = 255
        bad.keep["gate"].upload(raw)
    else:
        hit[:] = True
        raw = lay.shared["gate"].copy()
        raw[0, 200, 0] = 255
        bad.keep["sh_gate"].upload(raw)
    ctx.set_gemm_threshold(threshold)
    try:
        want, got = forward(ctx, lay, x), forward(ctx, bad, xb)
    finally:
        ctx.set_gemm_threshold(0)
    assert np.isfinite(want).all()
    assert np.array_equal(np.isnan(got), np.repeat(hit[:, None], lay.D, 1)), (np.isnan(got).any(1) != hit).nonzero()
    assert np.array_equal(got[~hit].view(np.uint32), want[~hit].view(np.uint32))
