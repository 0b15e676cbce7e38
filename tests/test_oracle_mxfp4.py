"""The CPU oracle's MXFP4 (quantizer, values, dot with Q8_0) against plain numpy forms, and the host-side checks of
the library's MXFP4 entry points that need no GPU."""
import numpy as np
import pytest

import _mxfp4 as X
import mimoe as M
import pyoracle as O


def rows_of_all_kinds(n=96, seed=5):
    rng = np.random.default_rng(seed)
    tie = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)      # midpoints between the steps, top 6
    r = [(rng.standard_normal((40, n)) * 0.02), rng.standard_normal((30, n)) * 10.0 ** rng.uniform(-44, 37, (30, 1)),
         np.zeros((2, n)), np.tile(tie, (3, n // 8)) * np.array([[1.0], [-1.0], [2.0 ** -20]]),
         np.tile(np.array([1.0, -1.0, 0.5, -0.5]), (2, n // 4)),
         np.full((1, n), 2.0 ** 127), np.full((1, n), np.finfo(np.float32).max), np.full((1, n), 1e-45),
         np.full((1, n), np.nextafter(np.float32(4), np.float32(0))), np.full((1, n), 2.0 ** -125), np.full((1, n), 2.0 ** -126)]
    r = np.concatenate(r).astype(np.float32)
    bad = np.tile(r[:4], 1).copy()
    bad[0, 3], bad[1, 40], bad[2, 95], bad[3, 0] = np.nan, np.inf, -np.inf, -np.nan
    return np.concatenate([r, bad])


def test_quantizer_and_values():
    x = rows_of_all_kinds()
    raw = O.quantize(O.TYPE_MXFP4, x)
    assert np.array_equal(raw, X.quantize(x))
    v = O.dequantize(O.TYPE_MXFP4, raw, x.shape[1])
    # the largest scale (2^127 times 3 and more) has values past float32's range: infinity there
    with np.errstate(over="ignore"):
        assert np.array_equal(v, X.values(raw).astype(np.float32), equal_nan=True)


def test_nearest_step_is_at_most_half_a_gap_off():
    x = np.random.default_rng(7).standard_normal((64, 64)).astype(np.float32)
    v = X.values(O.quantize(O.TYPE_MXFP4, x)).reshape(-1, 32)
    amax = np.abs(x.reshape(-1, 32)).max(1, keepdims=True)
    unit = 2.0 ** (np.floor(np.log2(amax)) - 2)
    # the widest gap is 2 units, half of it 1; above 6 units the error is at most 8 - 6
    off = np.abs(x.reshape(-1, 32) - v) / unit
    assert off.max() < 2.0 and off[np.abs(x.reshape(-1, 32)) <= 6 * unit].max() <= 1.0


@pytest.mark.parametrize("n", [32, 96, 704, 2048])
def test_dot(n):
    rng = np.random.default_rng(n)
    w = O.quantize(O.TYPE_MXFP4, (rng.standard_normal((5, n)) * 0.02).astype(np.float32))
    x = rng.standard_normal((3, n)).astype(np.float32)
    ref = X.q8_0(x) @ X.values(w).T
    for i in range(3):
        q = O.quantize(O.TYPE_Q8_0, x[i])
        for j in range(5):
            # the exact sum rounded once: half a step of float32, 2^-24
            assert abs(O.vec_dot(O.TYPE_MXFP4, w[j], q, n) - ref[i, j]) <= 2.0 ** -24 * abs(ref[i, j]) + 1e-13


def test_row_size_and_descriptor():
    assert M.TYPE_MXFP4 == 39 and M.row_size(M.TYPE_MXFP4, 64) == 34 and M.row_size(M.TYPE_MXFP4, 33) == 0
    t = M.tensor(4096, M.TYPE_MXFP4, [96, 5, 3])
    assert list(t.nb) == [17, 51, 255, 765]
