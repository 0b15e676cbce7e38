"""The operators around the experts through the C ABI (mi_moe_route, mi_moe_forward_router, mi_add_norm, mi_mul_mat)
against plain forms (_around.py).

Tolerances.  Routing: ids equal; a weight takes the score's rounding, the sum's, the addition of eps, the quotient, the
scaling and the expert's factor, half a step each: 6 half steps, 8 * 2^-24 of the value.  add_norm: the same float32 steps
in the same order with the row sums in 64 bits, so equal (sums that differ in their last bits, 2^-52, move a float32
rounding once in some 10^8 rows); codes equal byte for byte.  mul_mat: _around.mul_mat's bound of a float32 sum of
exact block parts.  Replays, other streams and repeated calls: equal bits."""
import numpy as np
import pytest

import _around as A
import mimoe as M
import pyoracle as O

pytestmark = pytest.mark.gpu
F32 = np.float32
EIGHT = {M.TYPE_Q4_0: M.TYPE_Q8_0, M.TYPE_Q4_K: M.TYPE_Q8_K}


@pytest.fixture(scope="module")
def ctx():
    c = M.Context(0)
    c.reserve(320, 8192, 64, 8, 2)
    yield c
    c.close()


# ------------------------------------------------------------------ helpers
class Rows:
    """a [T, n] array on the device with rows `pad` bytes longer than needed, `off` bytes into a buffer of guard bytes"""

    def __init__(self, T, n, type_=M.TYPE_F32, pad=0, off=0, data=None):
        self.T, self.n, self.type = T, n, type_
        self.rs = M.row_size(type_, n)
        self.nb, self.off = self.rs + pad, off
        self.host = np.full(off + self.nb * T + 64, 0xA5, np.uint8)
        if data is not None:
            self.view()[:] = np.ascontiguousarray(data).view(np.uint8).reshape(T, -1)
        self.buf = M.to_device(self.host)
        nb0 = M.BLOCK_BYTES.get(type_, 4)
        self.desc = M.tensor(self.buf.addr + off, type_, [n, T], [nb0, self.nb, self.nb * T, self.nb * T])
        self.desc._keep = self.buf

    def view(self):
        return np.lib.stride_tricks.as_strided(self.host[self.off:], (self.T, self.rs), (self.nb, 1))

    def get(self):
        """the rows; everything beside them is as it was"""
        now = self.buf.download(np.uint8, self.host.shape)
        rows = np.lib.stride_tricks.as_strided(now[self.off:], (self.T, self.rs), (self.nb, 1)).copy()
        rest = now.copy()
        np.lib.stride_tricks.as_strided(rest[self.off:], (self.T, self.rs), (self.nb, 1))[:] = self.view()
        assert np.array_equal(rest, self.host), "bytes outside the rows were written"
        return rows.view(F32) if self.type == M.TYPE_F32 else rows


def stream_rows(rng, T, n):
    x = rng.standard_normal((T, n)).astype(F32) * np.exp(0.5 * rng.standard_normal(n)).astype(F32)
    x[:, rng.integers(0, n, 2)] *= 8
    return x


# ------------------------------------------------------------------ routing
def run_route(ctx, logits, K, sigmoid, groups=1, kept=1, top=1, renorm=True, eps=0.0, scaling=1.0, bias=None, scale=None, pad=0, off=0,
              stream=None):
    T, E = logits.shape
    l = Rows(T, E, pad=pad, off=off, data=logits.astype(F32))
    sel, w = Rows(T, K), Rows(T, K)
    r = M.make_router(E, K, M.SCORE_SIGMOID if sigmoid else M.SCORE_SOFTMAX, groups, kept, top, renorm, eps, scaling,
                      M.to_device(np.asarray(bias, F32)) if bias is not None else None,
                      M.to_device(np.asarray(scale, F32)) if scale is not None else None)
    M.check("route", ctx.route(r, l.desc, sel.buf, w.buf, stream))
    M.synchronize()
    return sel.get().view(np.int32), w.get()


def check_route(ctx, logits, K, sigmoid, pad=0, off=0, **k):
    ids, w = run_route(ctx, logits, K, sigmoid, pad=pad, off=off, **k)
    want, ww = A.route(logits, K, sigmoid, **k)
    assert np.array_equal(ids, want)
    assert np.array_equal(np.isnan(w), np.isnan(ww))
    np.testing.assert_allclose(w, ww, rtol=8 * 2.0 ** -24, atol=2.0 ** -148)
    return ids, w


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,K,groups,kept,top", [
    (1, 256, 8, 8, 4, 2), (37, 256, 8, 8, 4, 2), (5, 128, 8, 4, 2, 1), (3, 64, 6, 1, 1, 1), (9, 51, 7, 3, 2, 2),
    (2, 1, 1, 1, 1, 1), (4, 2, 2, 2, 2, 1), (4, 2, 1, 2, 1, 1), (6, 130, 5, 10, 1, 2), (3, 1024, 64, 64, 17, 2), (7, 333, 12, 9, 5, 2),
    (3, 600, 9, 60, 3, 1), (2, 64, 64, 1, 1, 1), (2, 100, 50, 4, 2, 2), (5, 66, 3, 33, 2, 2), (301, 72, 4, 8, 3, 1), (3, 64, 1, 64, 1, 1)])
def test_route(ctx, T, E, K, groups, kept, top, sigmoid):
    rng = np.random.default_rng(T * 7 + E + K)
    logits = (2 * rng.standard_normal((T, E))).astype(F32)
    base = dict(groups=groups, kept=kept, top=top)
    check_route(ctx, logits, K, sigmoid, **base)
    check_route(ctx, logits, K, sigmoid, **base, bias=0.2 * rng.standard_normal(E), renorm=False, scaling=2.5, pad=20, off=4)
    check_route(ctx, logits, K, sigmoid, **base, bias=0.2 * rng.standard_normal(E), eps=1e-20, scale=rng.random(E) + 0.5)


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "softmax"])
def test_route_ties(ctx, sigmoid):
    """equal values: lower ids and lower groups; scores that round to the same float32 are equal"""
    rng = np.random.default_rng(5)
    logits = rng.integers(-2, 3, (64, 96)).astype(F32)
    for groups, kept, top in ((1, 1, 1), (8, 3, 2), (6, 2, 1)):
        check_route(ctx, logits, 7, sigmoid, groups=groups, kept=kept, top=top)
    same = np.zeros((3, 256), F32)
    assert (check_route(ctx, same, 8, sigmoid, groups=8, kept=2, top=2)[0] == np.arange(8)).all()
    high = (40 + rng.random((5, 64))).astype(F32)      # sigmoids of 1
    check_route(ctx, high, 6, sigmoid, groups=4, kept=2, top=2)


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "softmax"])
def test_route_masks(ctx, sigmoid):
    """masked experts (-inf, the type's lowest value), rows that the mask leaves nothing, infinities and NaN"""
    rng = np.random.default_rng(6)
    l = rng.standard_normal((12, 40)).astype(F32)
    l[0, 5:] = -np.inf
    l[1, :] = -np.inf
    l[2, :] = np.finfo(F32).min
    l[3, 1:] = np.finfo(F32).min
    l[4, 7] = np.nan
    l[5, :] = np.nan
    l[6, 3] = np.inf
    l[7, 8:] = np.nan
    l[8, :8] = -np.inf
    l[9, ::2] = np.finfo(F32).max
    l[10, 9] = -np.inf
    for k in (dict(), dict(groups=5, kept=2, top=2), dict(groups=8, kept=3, top=1)):
        check_route(ctx, l, 6, sigmoid, **k)
        check_route(ctx, l, 6, sigmoid, eps=1e-20, **k)
    bias = np.zeros(40, F32)
    bias[::3] = -np.inf
    bias[1] = np.nan
    for k in (dict(), dict(groups=5, kept=4, top=2), dict(groups=20, kept=6, top=2), dict(groups=20, kept=3, top=1)):
        check_route(ctx, l, 6, sigmoid, bias=bias, renorm=False, **k)


def test_route_as_the_gatings(ctx):
    """without groups: the choice of the layer's gatings (MI_GATING_SIGMOID_BIAS, MI_GATING_SOFTMAX_ALL)"""
    rng = np.random.default_rng(8)
    l = rng.standard_normal((50, 128)).astype(F32)
    bias = (0.1 * rng.standard_normal(128)).astype(F32)
    scale = (rng.random(128) + 0.5).astype(F32)
    ids, w = run_route(ctx, l, 8, True, eps=1e-20, scaling=2.5, bias=bias)
    oi, ow = O.route_gated(l, 8, 1, bias, None, 2.5, 1e-20)
    assert np.array_equal(ids, oi) and np.array_equal(w, ow)
    ids, w = run_route(ctx, l, 8, False, scale=scale)
    oi, ow = O.route_gated(l, 8, 2, None, scale, 1.0, 0.0)
    assert np.array_equal(ids, oi) and np.allclose(w, ow, rtol=2.0 ** -21, atol=0)


def test_route_many(ctx):
    rng = np.random.default_rng(9)
    l = rng.standard_normal((5000, 160)).astype(F32)
    check_route(ctx, l, 8, True, groups=8, kept=4, top=2, bias=0.1 * rng.standard_normal(160))


# ------------------------------------------------------------------ add_norm
@pytest.mark.parametrize("T,D,pad,off", [(1, 2048, 0, 0), (3, 2048, 0, 0), (5, 2816, 12, 4), (2, 1, 0, 0), (4, 7, 4, 8), (33, 256, 0, 0),
                                         (2, 4096, 32, 16), (3, 5120, 0, 0), (2, 8192, 4, 0), (2, 16384, 0, 0), (2, 12301, 0, 0),
                                         (700, 512, 0, 0), (300, 2688, 0, 0), (260, 4352, 16, 0)])
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
def test_add_norm(ctx, T, D, pad, off, layer):
    rng = np.random.default_rng(T + D)
    x, add = stream_rows(rng, T, D), stream_rows(rng, T, D)
    w, b = (1 + 0.1 * rng.standard_normal(D)).astype(F32), (0.1 * rng.standard_normal(D)).astype(F32)
    for use_add, use_w, kind in ((True, True, 0), (False, False, 0), (True, True, M.TYPE_Q8_0), (False, True, M.TYPE_Q8_K)):
        if kind and D % (32 if kind == M.TYPE_Q8_0 else 256):
            continue
        h, y = A.add_norm(x, add if use_add else None, layer, 1e-6, w if use_w else None, b if use_w else None)
        norm = M.make_norm(M.NORM_LAYER if layer else M.NORM_RMS, 1e-6, M.to_device(w) if use_w else None,
                           M.to_device(b) if use_w else None)
        dx, da = Rows(T, D, pad=pad, off=off, data=x), Rows(T, D, pad=2 * pad, off=off, data=add)
        ds, dy = Rows(T, D, pad=pad, off=off), Rows(T, D, pad=3 * pad)
        dq = Rows(T, D, kind, pad=pad, off=off) if kind else None
        M.check("add_norm", ctx.add_norm(norm, dx.desc, da.desc if use_add else None, ds.desc, dy.desc, dq.desc if dq else None))
        M.synchronize()
        assert np.array_equal(ds.get(), h)
        assert np.array_equal(dy.get(), y)
        dx.get(), da.get()
        if dq:
            assert np.array_equal(dq.get(), A.q8_bytes(y, kind))
            # the codes alone, and the sum alone beside them
            d2, s2 = Rows(T, D, kind, off=4), Rows(T, D)
            M.check("add_norm", ctx.add_norm(norm, dx.desc, da.desc if use_add else None, None, None, d2.desc))
            assert np.array_equal(d2.get(), A.q8_bytes(y, kind))
            M.check("add_norm", ctx.add_norm(norm, dx.desc, da.desc if use_add else None, s2.desc, None, d2.desc))
            assert np.array_equal(s2.get(), h)


@pytest.mark.parametrize("sum_on,y_on", [("x", None), ("add", "x"), ("x", "add"), (None, "x"), (None, "add")])
def test_add_norm_in_place(ctx, sum_on, y_on):
    rng = np.random.default_rng(4)
    for T, D in ((3, 2080), (400, 1024)):
        x, add = stream_rows(rng, T, D), stream_rows(rng, T, D)
        h, y = A.add_norm(x, add, False, 1e-5)
        d = {"x": Rows(T, D, pad=16, data=x), "add": Rows(T, D, data=add)}
        s = d[sum_on].desc if sum_on else None
        out = d[y_on] if y_on else Rows(T, D)
        M.check("add_norm", ctx.add_norm(M.make_norm(M.NORM_RMS, 1e-5), d["x"].desc, d["add"].desc, s, out.desc))
        assert np.array_equal(out.get(), y)
        if s is not None:
            assert np.array_equal(d[sum_on].get(), h)


@pytest.mark.parametrize("kind", [M.TYPE_Q8_0, M.TYPE_Q8_K])
@pytest.mark.parametrize("T", [12, 600])
def test_add_norm_blocks(ctx, kind, T):
    """blocks of zeros, of tiny and of huge values, of equal magnitudes of both signs, with a NaN or an infinity; a
    NaN in one row leaves the others alone"""
    rng = np.random.default_rng(11)
    D = 768
    x = rng.standard_normal((T, D)).astype(F32)
    x[0, :256] = 0
    x[1] = 0
    x[2, 256:] *= F32(1e-30)
    x[3, :256] = np.where(rng.random(256) < 0.5, 2, -2)
    x[4, 300] = np.nan
    x[5, 10] = np.inf
    x[6, :] = -np.inf
    x[7] *= F32(1e19)          # squares past the type's range
    w = np.ones(D, F32)
    w[64:96] = 3e7             # Q8_0 scales past the fp16 range
    w[512] = np.nan
    h, y = A.add_norm(x, None, False, 0.0, w)
    dy, dq = Rows(T, D), Rows(T, D, kind)
    M.check("add_norm", ctx.add_norm(M.make_norm(M.NORM_RMS, 0.0, M.to_device(w)), Rows(T, D, data=x).desc, None, None, dy.desc, dq.desc))
    got, q = dy.get(), dq.get()
    assert np.array_equal(got, y, equal_nan=True)
    bytes_ = 34 if kind == M.TYPE_Q8_0 else 292
    want = A.q8_bytes(y, kind).reshape(T, -1, bytes_)
    q = q.reshape(T, -1, bytes_)
    nan = ~np.isfinite(y.reshape(T, q.shape[1], -1)).all(2)
    assert np.array_equal(q[~nan], want[~nan])
    assert (q[nan][:, (2 if kind == M.TYPE_Q8_0 else 4):] == 0).all()
    d = np.ascontiguousarray(q[nan][:, :2]).view(np.float16) if kind == M.TYPE_Q8_0 else np.ascontiguousarray(q[nan][:, :4]).view(F32)
    assert np.isnan(d).all()


def test_dequantize_q8_K(ctx):
    rng = np.random.default_rng(12)
    raw = O.quantize(O.TYPE_Q8_K, stream_rows(rng, 67, 1024))
    dst = Rows(67, 1024)
    M.check("dequantize", ctx.dequantize(M.TYPE_Q8_K, M.to_device(raw), dst.buf, 67, 1024))
    assert np.array_equal(dst.get(), O.dequantize(O.TYPE_Q8_K, raw, 1024).reshape(67, 1024))
    b = M.DeviceBuffer(2048)
    assert ctx.dequantize(M.TYPE_Q8_K, b, b, 1, 128) == M.ERR_SHAPE and ctx.dequantize(M.TYPE_Q8_K, b.addr + 2, b, 1, 256) == M.ERR_UNSUPPORTED


# ------------------------------------------------------------------ mul_mat
def check_mul_mat(ctx, type_, T, N, n, x=None, raw=None, pad=0, off=0, apad=0, aoff=0, seed=0):
    rng = np.random.default_rng(T * 31 + N + n + seed)
    x = stream_rows(rng, T, n) if x is None else x
    raw = O.quantize(type_, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1) if raw is None else raw
    a = Rows(N, n, type_, pad=apad, off=aoff, data=raw)
    rows8 = A.q8_bytes(x, EIGHT[type_])
    want, tol = A.mul_mat(raw, type_, rows8, n)
    outs = []
    for b in (Rows(T, n, pad=pad, off=off, data=x), Rows(T, n, EIGHT[type_], pad=pad, off=off, data=rows8)):
        d = Rows(T, N, pad=pad, off=off)
        M.check("mul_mat", ctx.mul_mat(a.desc, b.desc, d.desc))
        M.synchronize()
        outs.append(d.get())
        b.get()
    assert np.array_equal(outs[0], outs[1], equal_nan=True)      # given in 8 bits: the same bits
    good = np.isfinite(want)
    assert (np.abs(outs[0].astype(np.float64) - want)[good] <= tol[good]).all()
    assert np.isnan(outs[0][~good]).all()
    return outs[0]


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T", [1, 2, 3, 5, 16, 17, 33, 64, 70])
@pytest.mark.parametrize("N,n", [(1, 256), (17, 512), (64, 1024), (100, 2048), (48, 2816), (33, 8192)])
def test_mul_mat(ctx, type_, T, N, n):
    check_mul_mat(ctx, type_, T, N, n)


@pytest.mark.parametrize("T", [1, 4, 19])
@pytest.mark.parametrize("n", [32, 64, 96, 160, 416, 1056, 2688, 4000])
def test_mul_mat_odd_blocks(ctx, n, T):
    check_mul_mat(ctx, M.TYPE_Q4_0, T, 50, n)


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T,N,n", [(1, 20000, 512), (6, 3712, 2560), (200, 300, 1024), (300, 130, 512), (640, 70, 256), (1, 2048, 7680), (9, 1000, 7168)])
def test_mul_mat_large(ctx, type_, T, N, n):
    check_mul_mat(ctx, type_, T, N, n)


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T", [1, 7, 40])
@pytest.mark.parametrize("pad,off,apad,aoff", [(4, 4, 16, 16), (8, 12, 32, 0), (16, 16, 48, 32), (64, 0, 0, 16)])
def test_mul_mat_strides(ctx, type_, T, pad, off, apad, aoff):
    check_mul_mat(ctx, type_, T, 37, 768, pad=pad, off=off, apad=apad, aoff=aoff)
    if type_ == M.TYPE_Q4_0:
        check_mul_mat(ctx, type_, T, 37, 736, pad=pad, off=off, apad=apad + 2, aoff=aoff + 2)
        check_mul_mat(ctx, type_, T, 21, 2048, pad=pad, off=off, apad=2, aoff=6)


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T", [1, 6, 21])
def test_mul_mat_extremes(ctx, type_, T):
    """every code and scale byte, largest codes throughout (the longest exact sums), rows of zeros, of tiny and of large
    values; rows that are no numbers are NaN and leave the others alone"""
    rng = np.random.default_rng(T)
    n, N = 1024, 40
    raw = rng.integers(0, 256, (N, M.row_size(type_, n)), dtype=np.uint8)
    blk = raw.reshape(N, -1, M.BLOCK_BYTES[type_])
    small = (0.01 * rng.standard_normal((*blk.shape[:2], 2))).astype(np.float16).view(np.uint8).reshape(*blk.shape[:2], 4)
    blk[..., :2 if type_ == M.TYPE_Q4_0 else 4] = small[..., :2 if type_ == M.TYPE_Q4_0 else 4]
    blk[0, :, 2 if type_ == M.TYPE_Q4_0 else 4:] = 0xFF
    blk[1, :, 2 if type_ == M.TYPE_Q4_0 else 4:] = 0
    x = stream_rows(rng, T, n)
    check_mul_mat(ctx, type_, T, N, n, x, raw)
    for k, v in enumerate((F32(3), F32(-3), F32(0), F32(1e-30), F32(8e6))):
        x[k % T] = v
        check_mul_mat(ctx, type_, T, N, n, x, raw)
    x = stream_rows(rng, T, n)
    good = check_mul_mat(ctx, type_, T, N, n, x, raw)
    for v in (np.nan, np.inf, F32(1e38) if type_ == M.TYPE_Q4_0 else -np.inf):
        y = x.copy()
        y[T // 2, 77] = v
        got = check_mul_mat(ctx, type_, T, N, n, y, raw)
        assert np.isnan(got[T // 2]).all()
        keep = np.arange(T) != T // 2
        assert np.array_equal(got[keep], good[keep])


def test_mul_mat_row_bits_do_not_depend_on_the_batch(ctx):
    """a row's result is the same bits alone and among others of the same path (each row's sums are its own)"""
    rng = np.random.default_rng(2)
    for type_ in EIGHT:
        x = stream_rows(rng, 16, 2048)
        raw = O.quantize(type_, (0.05 * rng.standard_normal((200, 2048))).astype(F32)).reshape(200, -1)
        all_ = check_mul_mat(ctx, type_, 16, 200, 2048, x, raw)
        again = check_mul_mat(ctx, type_, 16, 200, 2048, x, raw)
        assert np.array_equal(all_, again)


# ------------------------------------------------------------------ as they are used
def test_dense_block_of_a_decode_step(ctx):
    """residual + norm -> 8-bit rows -> two matrices, on a stream of its own, captured and replayed with new inputs"""
    rng = np.random.default_rng(21)
    for type_, kind in ((M.TYPE_Q4_0, M.NORM_RMS), (M.TYPE_Q4_K, M.NORM_LAYER)):
        T, n, N = 3, 1536, 500
        w, b = (1 + 0.1 * rng.standard_normal(n)).astype(F32), (0.1 * rng.standard_normal(n)).astype(F32)
        raw = [O.quantize(type_, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1) for _ in range(2)]
        mats = [Rows(N, n, type_, data=r) for r in raw]
        x, add, s, q = Rows(T, n), Rows(T, n), Rows(T, n), Rows(T, n, EIGHT[type_])
        outs = [Rows(T, N) for _ in mats]
        norm = M.make_norm(kind, 1e-5, M.to_device(w), M.to_device(b))

        def step(st):
            M.check("add_norm", ctx.add_norm(norm, x.desc, add.desc, s.desc, None, q.desc, st.h))
            for m, o in zip(mats, outs):
                M.check("mul_mat", ctx.mul_mat(m.desc, q.desc, o.desc, st.h))
                M.check("mul_mat", ctx.mul_mat(m.desc, s.desc, o.desc, st.h))      # (float32 rows: the workspace)
                M.check("mul_mat", ctx.mul_mat(m.desc, q.desc, o.desc, st.h))

        st = M.Stream()
        graph = M.Graph(st, step)
        for i in range(4):
            hx, ha = stream_rows(rng, T, n), stream_rows(rng, T, n)
            x.buf.upload(hx), add.buf.upload(ha)
            step(st)
            st.synchronize()
            eager = [o.get() for o in outs]
            h, y = A.add_norm(hx, ha, kind == M.NORM_LAYER, 1e-5, w, b)
            assert np.array_equal(s.get(), h)
            for got, r in zip(eager, raw):
                want, tol = A.mul_mat(r, type_, A.q8_bytes(y, EIGHT[type_]), n)
                assert (np.abs(got - want) <= tol).all()
            for o in outs:
                o.buf.zero()
            M.synchronize()
            graph.launch(st)
            st.synchronize()
            for o, e in zip(outs, eager):
                assert np.array_equal(o.buf.download(F32, (T, N)), e)
                o.host[:] = o.buf.download(np.uint8, o.host.shape)
        graph.destroy()
        st.destroy()


def _layer(rng, type_, D, E, K, I, keep):
    def tab(*shape):
        keep.append(M.to_device(O.quantize(type_, (0.08 * rng.standard_normal(shape)).astype(F32))))
        return M.tensor(keep[-1], type_, list(shape[::-1]))

    wr = (0.1 * rng.standard_normal((E, D))).astype(F32)
    keep.append(M.to_device(wr))
    return M.make_layer(D, E, K, I, keep[-1], None, tab(E, I, D), tab(E, I, D), tab(E, D, I), False, M.ACT_SILU)


@pytest.mark.parametrize("type_", [M.TYPE_Q4_K, M.TYPE_Q8_0, M.TYPE_MXFP4], ids=["q4_K", "q8_0", "mxfp4"])
@pytest.mark.parametrize("T", [1, 5, 150])
def test_forward_router(type_, T):
    """the block with a router is the block's parts: its logits, mi_moe_route on them, mi_moe_expert_ffn; with a norm and
    with the router's own rows too"""
    rng = np.random.default_rng(T)
    D, E, K, I = 512, 64, 6, 256
    ctx = M.Context(0)
    ctx.reserve(T, D, I, E, K)
    ctx.set_fused_decode(False)
    keep = []
    L = _layer(rng, type_, D, E, K, I, keep)
    bias, scale = M.to_device((0.1 * rng.standard_normal(E)).astype(F32)), M.to_device((rng.random(E) + 0.5).astype(F32))
    r = M.make_router(E, K, M.SCORE_SIGMOID, 8, 3, 2, True, 1e-20, 2.5, bias, scale)
    norm = M.make_norm(M.NORM_RMS, 1e-6, M.to_device((1 + 0.1 * rng.standard_normal(D)).astype(F32)))
    h, xr = Rows(T, D, data=stream_rows(rng, T, D)), Rows(T, D, data=stream_rows(rng, T, D))
    y = Rows(T, D)
    M.check("norm", ctx.norm(norm, h.buf, T, D, y.buf))
    M.synchronize()
    for n, x, router_rows in ((None, y, None), (norm, h, None), (None, y, xr)):
        out, logits, sel, w, counts, ref = Rows(T, D), Rows(T, E), Rows(T, K), Rows(T, K), Rows(1, E), Rows(T, D)
        routing = M.Routing(logits.buf.addr, sel.buf.addr, w.buf.addr, counts.buf.addr, None, None)
        M.check("forward", ctx.forward_router(L, r, n, x.buf, router_rows.buf if router_rows else None, T, h.buf, out.buf, routing))
        M.synchronize()
        l = logits.get()
        ids, ww = A.route(l, K, True, 8, 3, 2, True, 1e-20, 2.5, bias.download(F32, (E,)), scale.download(F32, (E,)))
        s2, w2 = Rows(T, K), Rows(T, K)
        M.check("route", ctx.route(r, logits.desc, s2.buf, w2.buf))
        M.synchronize()
        got = sel.get().view(np.int32)
        assert np.array_equal(got, ids) and np.array_equal(s2.get().view(np.int32), ids) and np.array_equal(w.get(), w2.get())
        np.testing.assert_allclose(w.get(), ww, rtol=8 * 2.0 ** -24)
        assert np.array_equal(counts.get().view(np.int32)[0], np.bincount(ids.ravel(), minlength=E))
        M.check("expert_ffn", ctx.expert_ffn(L, y.buf, T, h.buf, sel.buf, sel.buf, w.buf, ref.buf))
        M.synchronize()
        assert np.array_equal(out.get(), ref.get())
    # the layer's own gating is as it was
    out1, out2 = Rows(T, D), Rows(T, D)
    M.check("forward", ctx.forward(L, y.buf, T, h.buf, out1.buf))
    plain = M.make_router(E, K, M.SCORE_SOFTMAX)
    M.check("forward", ctx.forward_router(L, plain, None, y.buf, None, T, h.buf, out2.buf))
    M.synchronize()
    assert np.allclose(out1.get(), out2.get(), rtol=0, atol=1e-3 * np.abs(out1.get()).max())   # (weights: another rounding)
    ctx.close()


@pytest.mark.parametrize("type_", [M.TYPE_Q4_K, M.TYPE_Q8_0], ids=["q4_K", "q8_0"])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_forward_router_as_the_gating(type_, T):
    """a router without groups and the layer's own gating of the same kind: the same bits, shared expert and all"""
    rng = np.random.default_rng(T + 50)
    D, E, K, I = 512, 32, 4, 256
    ctx = M.Context(0)
    ctx.reserve(T, D, I, E, K)
    keep = []
    L = _layer(rng, type_, D, E, K, I, keep)

    def tab(n, k):
        keep.append(M.to_device(O.quantize(type_, (0.08 * rng.standard_normal((n, k))).astype(F32))))
        return M.tensor(keep[-1], type_, [k, n])

    L.sh_n_ff, L.sh_act, L.sh_gate, L.sh_up, L.sh_down = I, M.ACT_SILU, tab(I, D), tab(I, D), tab(D, I)
    bias = M.to_device((0.1 * rng.standard_normal(E)).astype(F32))
    L.gating, L.sel_bias, L.routed_scaling, L.gate_eps = M.GATING_SIGMOID_BIAS, bias.addr, 2.5, 1e-20
    r = M.make_router(E, K, M.SCORE_SIGMOID, renorm=True, eps=1e-20, scaling=2.5, sel_bias=bias)
    x, res = Rows(T, D, data=stream_rows(rng, T, D)), Rows(T, D, data=stream_rows(rng, T, D))
    a, b = Rows(T, D), Rows(T, D)
    M.check("forward", ctx.forward(L, x.buf, T, res.buf, a.buf))
    L.gating = 77      # (not read)
    M.check("forward", ctx.forward_router(L, r, None, x.buf, None, T, res.buf, b.buf))
    M.synchronize()
    assert np.array_equal(a.get(), b.get())
    # captured and replayed on another input
    st = M.Stream()
    g = M.Graph(st, lambda s: M.check("forward", ctx.forward_router(L, r, None, x.buf, None, T, res.buf, b.buf, None, s.h)))
    for i in range(3):
        x.buf.upload(stream_rows(rng, T, D))
        M.check("forward", ctx.forward_router(L, r, None, x.buf, None, T, res.buf, a.buf))
        M.synchronize()
        b.buf.zero()
        M.synchronize()
        g.launch(st)
        st.synchronize()
        assert np.array_equal(a.buf.download(F32, (T, D)), b.buf.download(F32, (T, D)))
    g.destroy()
    st.destroy()
    ctx.close()


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
def test_mul_mat_many_rows(type_):
    """more rows than one pass takes"""
    ctx = M.Context(0)
    T, N, n = 33000, 19, 256
    ctx.reserve(T, n, 32, 1, 1)
    rng = np.random.default_rng(1)
    check_mul_mat(ctx, type_, T, N, n, x=(rng.standard_normal((T, n))).astype(F32))
    ctx.close()


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T,n", [(1, 65536), (4, 40960), (8, 20480), (17, 12288), (70, 5120), (1, 1 << 17)])
def test_mul_mat_long_rows(type_, T, n):
    """rows whose operands do not fit LDS at once, or only for few tokens"""
    ctx = M.Context(0)
    ctx.reserve(T, n, 32, 1, 1)
    check_mul_mat(ctx, type_, T, 37, n)
    ctx.close()


@pytest.mark.parametrize("T", [2, 20])
def test_mul_mat_subnormal_scales(ctx, T):
    """Q8_0 scales in fp16's subnormal range, and below it: the codes of the oracle, scales rounded as its"""
    rng = np.random.default_rng(3)
    x = stream_rows(rng, T, 256)
    x[:, :64] *= F32(1e-5)
    x[:, 64:128] *= F32(3e-7)
    x[:, 128:160] *= F32(1e-9)
    raw = O.quantize(M.TYPE_Q4_0, (0.05 * rng.standard_normal((40, 256))).astype(F32)).reshape(40, -1)
    check_mul_mat(ctx, M.TYPE_Q4_0, T, 40, 256, x, raw)
    dq, dy = Rows(T, 256, M.TYPE_Q8_0), Rows(T, 256)
    w = np.exp(-20 * rng.random(256)).astype(F32)
    M.check("add_norm", ctx.add_norm(M.make_norm(M.NORM_RMS, 0.0, M.to_device(w)), Rows(T, 256, data=x).desc, None, None, dy.desc, dq.desc))
    assert np.array_equal(dq.get(), A.q8_bytes(dy.get(), M.TYPE_Q8_0))


def test_halves(ctx):
    """values on the border between two codes: away from zero in Q8_0, to even in Q8_K"""
    q = np.tile(np.concatenate([np.arange(-126.5, 127, 1), [127, 126.5]]), 8)[:2048].astype(F32).reshape(2, 1024)
    q[:, ::32] = 127      # every block's largest: the scale is 1
    for kind in (M.TYPE_Q8_0, M.TYPE_Q8_K):
        w = M.to_device(q[0])
        ones = np.ones((1, 1024), F32)      # norm: 1 / sqrt(1 + eps), eps = 0
        dq, dy = Rows(1, 1024, kind), Rows(1, 1024)
        M.check("add_norm", ctx.add_norm(M.make_norm(M.NORM_RMS, 0.0, w), Rows(1, 1024, data=ones).desc, None, None, dy.desc, dq.desc))
        assert np.array_equal(dy.get(), q[:1])
        assert np.array_equal(dq.get(), A.q8_bytes(q[:1], kind))
    raw = O.quantize(M.TYPE_Q4_0, (0.05 * np.random.default_rng(0).standard_normal((33, 1024))).astype(F32)).reshape(33, -1)
    rawk = O.quantize(M.TYPE_Q4_K, (0.05 * np.random.default_rng(0).standard_normal((33, 1024))).astype(F32)).reshape(33, -1)
    for T in (1, 2, 18):
        x = np.tile(q, (9, 1))[:T]
        check_mul_mat(ctx, M.TYPE_Q4_0, T, 33, 1024, x, raw)
        check_mul_mat(ctx, M.TYPE_Q4_K, T, 33, 1024, x, rawk)


def test_capacity(ctx):
    small = M.Context(0)
    small.reserve(4, 512, 256, 4, 2)
    a = Rows(8, 512, M.TYPE_Q4_0)
    for T, n, rc in ((8, 512, M.OK), (9, 512, M.ERR_CAPACITY)):
        assert small.mul_mat(a.desc, Rows(T, n, data=np.zeros((T, n), F32)).desc, Rows(T, 8).desc) == rc
    M.synchronize()
    assert small.mul_mat(Rows(8, 1024, M.TYPE_Q4_0).desc, Rows(1, 1024, data=np.zeros((1, 1024), F32)).desc, Rows(1, 8).desc) == M.ERR_CAPACITY
    M.check("mul_mat", small.mul_mat(a.desc, Rows(30, 512, M.TYPE_Q8_0, data=np.zeros((30, 544), np.uint8)).desc, Rows(30, 8).desc))
    M.synchronize()
    small.close()


# ------------------------------------------------------------------ where launches and plans change over
@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T", [7, 8, 9])
def test_mul_mat_bits_where_the_operands_are_made_elsewhere(type_, T):
    """long rows, whose sums' order follows the operands' place in LDS: float32 rows and 8-bit rows give the same bits
    on both sides of the batch from which the operands are made in a launch of their own"""
    ctx = M.Context(0)
    ctx.reserve(T, 8448, 32, 1, 1)
    check_mul_mat(ctx, type_, T, 4096, 8448)
    ctx.close()


def _spots(T, n):
    """rows around the ends of what 2^32 threads cover, for any count of threads a row"""
    s = {0, T - n} | {(1 << k) - n // 2 for k in range(20, 33) if (1 << k) + n // 2 <= T}
    return sorted(s)


def test_route_more_rows_than_a_launch_has_threads(ctx):
    T, E, n = (1 << 26) + 29, 4, 8
    rng = np.random.default_rng(11)
    lg = M.DeviceBuffer(4 * T * E).zero()
    sel, w = M.DeviceBuffer(4 * T), M.DeviceBuffer(4 * T)
    M.call("mi_memset_d", sel.ptr, 0xFF, 4 * T)
    rows = {s: rng.standard_normal((n, E)).astype(F32) for s in _spots(T, n)}
    for s, l in rows.items():
        lg.upload(l, 16 * s)
    M.check("route", ctx.route(M.make_router(E, 1, M.SCORE_SIGMOID, renorm=False), M.tensor(lg, M.TYPE_F32, [E, T]), sel, w))
    M.synchronize()
    for s, l in rows.items():
        assert np.array_equal(sel.download(np.int32, (n,), 4 * s), l.argmax(1))
    for b in (lg, sel, w):
        b.free()


def test_add_norm_more_rows_than_a_launch_has_threads(ctx):
    T, D, n = (1 << 25) + 29, 4, 8
    rng = np.random.default_rng(12)
    x, y = M.DeviceBuffer(4 * T * D).zero(), M.DeviceBuffer(4 * T * D)
    M.call("mi_memset_d", y.ptr, 0xFF, 4 * T * D)
    rows = {s: rng.standard_normal((n, D)).astype(F32) for s in _spots(T, n)}
    for s, v in rows.items():
        x.upload(v, 16 * s)
    M.check("add_norm", ctx.add_norm(M.make_norm(M.NORM_RMS, 1e-6), M.tensor(x, M.TYPE_F32, [D, T]), None, None,
                                     M.tensor(y, M.TYPE_F32, [D, T])))
    M.synchronize()
    for s, v in rows.items():
        assert np.array_equal(y.download(F32, (n, D), 16 * s), A.add_norm(v, None, False, 1e-6)[1])
    for b in (x, y):
        b.free()


def test_dequantize_q8_K_more_blocks_than_a_launch_has_threads(ctx):
    n, T = 8, (1 << 26) + 29
    try:
        q, y = M.DeviceBuffer(292 * T).zero(), M.DeviceBuffer(1024 * T)
    except M.MimoeError:
        pytest.skip("88 GB of device memory")
    rng = np.random.default_rng(13)
    rows = {s: A.q8_bytes(rng.standard_normal((n, 256)).astype(F32), M.TYPE_Q8_K) for s in _spots(T, n)}
    for s, v in rows.items():
        q.upload(v, 292 * s)
    M.check("dequantize", ctx.dequantize(M.TYPE_Q8_K, q, y, T, 256))
    M.synchronize()
    for s, v in rows.items():
        d, c = v[:, :4].copy().view(F32), v[:, 4:260].view(np.int8)
        assert np.array_equal(y.download(F32, (n, 256), 1024 * s), d * c.astype(F32))
    for b in (q, y):
        b.free()


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T,N,n", [(17, 2100, 512), (33, 2200, 512), (33, 2200, 5120), (100, 1000, 1024), (65, 12300, 512),
                                   (70, 12297, 2816), (200, 6200, 768), (17, 40, 7936), (200, 52, 7168)])
def test_mul_mat_tiles_of_rows(ctx, type_, T, N, n):
    """16, 32 and 64 rows of b a work-group, their operands in LDS at once and in parts"""
    check_mul_mat(ctx, type_, T, N, n)


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
@pytest.mark.parametrize("T,N,n", [(8, 4096, 8448), (9, 70, 512), (24, 100, 2048), (33, 2200, 5120), (70, 12297, 768), (16, 33, 8192)])
def test_mul_mat_rows_in_8_bits_without_workspace(type_, T, N, n):
    """the work-groups make the operands then: the same bits"""
    rng = np.random.default_rng(T + N)
    rows8 = A.q8_bytes(stream_rows(rng, T, n), EIGHT[type_])
    a = Rows(N, n, type_, data=O.quantize(type_, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1))
    b = Rows(T, n, EIGHT[type_], data=rows8)
    outs = []
    for reserved in (False, True):
        c = M.Context(0)
        if reserved:
            c.reserve(T, n, 32, 1, 1)
        d = Rows(T, N)
        M.check("mul_mat", c.mul_mat(a.desc, b.desc, d.desc))
        M.synchronize()
        outs.append(d.get())
        c.close()
    assert np.array_equal(*outs)


@pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])
def test_dense_block_of_a_batch(ctx, type_):
    """norm -> 8-bit rows -> matrix and float32 rows -> matrix, captured; other products of the same context, which
    use the same workspace, between the replays"""
    T, n, N = 45, 1024, 4300      # the operands in a launch of their own, 32 rows a work-group
    rng = np.random.default_rng(8)
    a = Rows(N, n, type_, data=O.quantize(type_, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1))
    x, y, q = Rows(T, n), Rows(T, n), Rows(T, n, EIGHT[type_])
    d8, d32, other = Rows(T, N), Rows(T, N), Rows(T, N)
    noise = Rows(T, n, data=stream_rows(rng, T, n))
    norm = M.make_norm(M.NORM_RMS, 1e-6)

    def step(st):
        M.check("add_norm", ctx.add_norm(norm, x.desc, None, None, y.desc, q.desc, st.h))
        M.check("mul_mat", ctx.mul_mat(a.desc, q.desc, d8.desc, st.h))
        M.check("mul_mat", ctx.mul_mat(a.desc, y.desc, d32.desc, st.h))

    st = M.Stream()
    graph = M.Graph(st, step)
    for i in range(4):
        x.buf.upload(stream_rows(rng, T, n))
        step(st)
        st.synchronize()
        want = d8.buf.download(F32, (T, N))
        assert np.isfinite(want).all() and np.array_equal(want, d32.buf.download(F32, (T, N)))
        M.check("mul_mat", ctx.mul_mat(a.desc, noise.desc, other.desc, st.h))
        d8.buf.zero(), d32.buf.zero()
        M.synchronize()
        graph.launch(st)
        M.check("mul_mat", ctx.mul_mat(a.desc, noise.desc, other.desc, st.h))
        graph.launch(st)
        st.synchronize()
        assert np.array_equal(want, d8.buf.download(F32, (T, N))) and np.array_equal(want, d32.buf.download(F32, (T, N)))
    graph.destroy()
    st.destroy()
