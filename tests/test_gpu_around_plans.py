"""Products of 4-bit matrices (mi_mul_mat) where their plans differ: a row's bits among other rows of the same plan, the
kernels of few rows past what the dot products take, float32 rows in a captured step.

Tolerances: _around.mul_mat's bound of a float32 sum of exact block parts; within a plan, and between eager and
replayed calls, equal bits."""
import numpy as np
import pytest

import _around as A
import mimoe as M
import pyoracle as O
from test_gpu_around import EIGHT, F32, Rows, check_mul_mat, stream_rows

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("type_", [M.TYPE_Q4_0, M.TYPE_Q4_K], ids=["q4_0", "q4_K"])


def products(ctx, a, type_, x, eight):
    """rows of x through a, given in float32 or in 8 bits"""
    T, n = x.shape
    b = Rows(T, n, EIGHT[type_], data=A.q8_bytes(x, EIGHT[type_])) if eight else Rows(T, n, data=x)
    d = Rows(T, a.T)
    M.check("mul_mat", ctx.mul_mat(a.desc, b.desc, d.desc))
    M.synchronize()
    return d.get()


@TYPES
@pytest.mark.parametrize("eight", [False, True], ids=["f32", "8bit"])
@pytest.mark.parametrize("lo,hi,N,n", [(9, 16, 200, 2048),       # 16 rows a work-group, waves share a tile of the matrix
                                       (17, 32, 2100, 512),      # 32 rows
                                       (33, 64, 24600, 256),     # 64 rows, a wave a tile
                                       (65, 128, 12300, 512)])   # the same, two work-groups of rows
def test_a_rows_bits_among_others(type_, eight, lo, hi, N, n):
    """a row's result is the same bits in any batch of the plan: fewer rows, other rows around it, another place"""
    ctx = M.Context(0)
    ctx.reserve(hi, n, 32, 1, 1)
    rng = np.random.default_rng(lo)
    a = Rows(N, n, type_, data=O.quantize(type_, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1))
    x = stream_rows(rng, hi, n)
    whole = products(ctx, a, type_, x, eight)
    want, tol = A.mul_mat(a.view().copy(), type_, A.q8_bytes(x, EIGHT[type_]), n)
    assert (np.abs(whole - want) <= tol).all()
    for pick in (np.arange(lo), np.arange(hi - lo, hi), rng.permutation(hi), rng.permutation(hi)[:(lo + hi) // 2],
                 np.repeat(rng.integers(0, hi), lo)):
        assert np.array_equal(products(ctx, a, type_, x[pick], eight), whole[pick])
    ctx.close()


# rows of the matrix-unit kernel's forms of up to 4 and of up to 7 tokens: their operands are more than the dot
# products' LDS holds (40 bytes a token and 32 values, 160 KB), or T N n is past 9 * 2^24 (Q4_0; Q4_K 9 * 2^23).  Q4_0
# rows whose last set of 128 values holds 1, 2 or 3 blocks.
@pytest.mark.parametrize("T,N,n,type_", [(1, 21, 131104, M.TYPE_Q4_0), (2, 37, 65600, M.TYPE_Q4_0), (3, 20, 43744, M.TYPE_Q4_0),
                                         (4, 50, 40992, M.TYPE_Q4_0), (5, 9800, 3104, M.TYPE_Q4_0), (6, 8200, 3136, M.TYPE_Q4_0),
                                         (7, 6900, 3168, M.TYPE_Q4_0), (5, 33, 32800, M.TYPE_Q4_0), (7, 50, 24032, M.TYPE_Q4_0),
                                         (3, 10000, 2560, M.TYPE_Q4_K), (4, 9000, 2304, M.TYPE_Q4_K), (7, 5000, 2304, M.TYPE_Q4_K),
                                         (6, 50, 28160, M.TYPE_Q4_K)])
def test_few_rows_on_the_matrix_units(T, N, n, type_):
    assert T * 40 * (n // 32) > 160 * 1024 or T * N * n > 9 << (24 if type_ == M.TYPE_Q4_0 else 23)
    ctx = M.Context(0)
    ctx.reserve(T, n, 32, 1, 1)
    check_mul_mat(ctx, type_, T, N, n)
    ctx.close()


@TYPES
def test_float32_rows_in_a_captured_step(type_):
    """residual + norm, then float32 rows of three tokens through two matrices (made into operands by the work-groups
    themselves), each product kept: eager, replayed and from the same rows in 8 bits"""
    rng = np.random.default_rng(23)
    T, n, N = 3, 1536, 500
    ctx = M.Context(0)
    ctx.reserve(T, n, 32, 1, 1)
    raw = [O.quantize(type_, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1) for _ in range(2)]
    mats = [Rows(N, n, type_, data=r) for r in raw]
    x, add, s, y, q = Rows(T, n), Rows(T, n), Rows(T, n), Rows(T, n), Rows(T, n, EIGHT[type_])
    rows = [(m, b) for m in mats for b in (s, y, q)]
    outs = [Rows(T, N) for _ in rows]
    norm = M.make_norm(M.NORM_RMS, 1e-5)

    def step(st):
        M.check("add_norm", ctx.add_norm(norm, x.desc, add.desc, s.desc, y.desc, q.desc, st.h))
        for (m, b), o in zip(rows, outs):
            M.check("mul_mat", ctx.mul_mat(m.desc, b.desc, o.desc, st.h))

    st = M.Stream()
    graph = M.Graph(st, step)
    for i in range(4):
        hx, ha = stream_rows(rng, T, n), stream_rows(rng, T, n)
        x.buf.upload(hx), add.buf.upload(ha)
        step(st)
        st.synchronize()
        eager = [o.buf.download(F32, (T, N)) for o in outs]
        h, yh = A.add_norm(hx, ha, False, 1e-5)
        for k, r in enumerate(raw):
            for got, v in ((eager[3 * k], h), (eager[3 * k + 1], yh)):
                want, tol = A.mul_mat(r, type_, A.q8_bytes(v, EIGHT[type_]), n)
                assert (np.abs(got - want) <= tol).all()
            assert np.array_equal(eager[3 * k + 1], eager[3 * k + 2])
        for o in outs:
            o.buf.zero()
        M.synchronize()
        graph.launch(st)
        st.synchronize()
        for o, e in zip(outs, eager):
            assert np.array_equal(o.buf.download(F32, (T, N)), e)
    graph.destroy()
    st.destroy()
    ctx.close()


@pytest.mark.parametrize("T", [1, 3, 7, 20, 70])
def test_rows_that_mi_quantize_wrote(T):
    """Q8_0 rows of mi_quantize: the bytes of mi_add_norm's blocks and the bits of the float32 rows' product, with blocks
    of zeros, scales below fp16's and codes between two"""
    rng = np.random.default_rng(T)
    n, N = 736, 300
    ctx = M.Context(0)
    ctx.reserve(T, n, 32, 1, 1)
    x = stream_rows(rng, T, n)
    x[:, 32:64] = 0
    x[:, 64:96] *= F32(1e-7)
    x[:, 96:128] *= F32(1e-12)
    x[:, 128:160] = np.arange(-15.5, 16.5)
    x[:, 128] = 127
    a = Rows(N, n, M.TYPE_Q4_0, data=O.quantize(M.TYPE_Q4_0, (0.05 * rng.standard_normal((N, n))).astype(F32)).reshape(N, -1))
    b, q = Rows(T, n, data=x), Rows(T, n, M.TYPE_Q8_0)
    M.check("quantize", ctx.quantize(M.TYPE_Q8_0, b.buf, q.buf, T, n))
    outs = [Rows(T, N), Rows(T, N)]
    for r, d in zip((b, q), outs):
        M.check("mul_mat", ctx.mul_mat(a.desc, r.desc, d.desc))
    M.synchronize()
    assert np.array_equal(q.get(), A.q8_bytes(x, M.TYPE_Q8_0))
    assert np.array_equal(outs[0].get(), outs[1].get())
    ctx.close()
