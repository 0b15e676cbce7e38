"""MXFP4 expert tables through the C ABI against float64 forms (_mxfp4.py) and the CPU oracle.

Tolerances.  mi_quantize and mi_dequantize: exact.  Products of few rows per expert: exact block sums added in fp64
(error 2^-53 times the number of blocks), rounded to float32 once: 2^-24 of the value, and 2^-50 of the sum of the
terms' sizes where they cancel.  The GEMM adds a block pair's digit sum to a float32 accumulator, four per 64 values:
n / 16 additions, each off by at most a step (2^-23, whether the matrix unit rounds or cuts) of the largest partial
sum, so a value is off by at most n / 16 * 2^-23 of its terms' sizes (|x| . |w|); the digits' partial sums are at most
2 |x| . |w| together (a balanced digit's part overshoots what it stands for by at most a half), so twice that.
Layers of few rows: the products as above, the GLU in fp64 rounded to float32, Q8_0 codes equal; z, z w and the
result rounded to float32: (K + 3) 2^-24 of the terms' sizes; the weights (softmax in float32: exp and sum within 4
steps) add 2^-21.
Layers on the GEMM: an error of the gate/up products can move a code of the activation rows by a step (1 / 127 of its
block's largest) and an fp16 scale by a step (2^-10): held to 1e-2 as the other 32-value types are, and 1e-3 measured
by the root of the mean square."""
import numpy as np
import pytest

import _mxfp4 as X
import mimoe as M
import pyoracle as O
from test_oracle_mxfp4 import rows_of_all_kinds

pytestmark = pytest.mark.gpu
MX = M.TYPE_MXFP4


@pytest.fixture(scope="module")
def ctx():
    c = M.Context(0)
    c.reserve(640, 2816, 1856, 64, 8)
    yield c
    c.close()


def table(rng, E, N, n, std=0.02):
    return O.quantize(O.TYPE_MXFP4, (rng.standard_normal((E, N, n)) * std).astype(np.float32))


def rows(rng, *shape):
    x = rng.standard_normal(shape).astype(np.float32) * np.exp(rng.standard_normal(shape[-1])).astype(np.float32)
    return x


# ------------------------------------------------------------------ quantize, dequantize
@pytest.mark.parametrize("offset", [0, 4, 1, 3])
def test_quantize_exact(ctx, offset):
    x = rows_of_all_kinds()
    for nrows in (1, 3, len(x)):
        src = M.DeviceBuffer(x.nbytes + 16).upload(x[:nrows], 4 if offset else 0)
        n = nrows * M.row_size(MX, x.shape[1])
        dst = M.to_device(np.full(n + 64, 0xA5, np.uint8))
        M.check("quantize", ctx.quantize(MX, src.addr + (4 if offset else 0), dst.addr + offset, nrows, x.shape[1]))
        got = dst.download(np.uint8, (n + 64,))
        assert np.array_equal(got[offset:offset + n].reshape(nrows, -1), X.quantize(x[:nrows]))
        assert (got[:offset] == 0xA5).all() and (got[offset + n:] == 0xA5).all()


def test_quantize_many_blocks(ctx):
    x = rows(np.random.default_rng(3), 700, 1056)
    dst = M.DeviceBuffer(700 * M.row_size(MX, 1056))
    M.check("quantize", ctx.quantize(MX, M.to_device(x), dst, 700, 1056))
    assert np.array_equal(dst.download(np.uint8, (700, 561)), O.quantize(O.TYPE_MXFP4, x))


@pytest.mark.parametrize("type_", [MX, M.TYPE_Q4_0, M.TYPE_Q5_0, M.TYPE_Q8_0, M.TYPE_F16])
@pytest.mark.parametrize("nrows,n", [(1, 32), (5, 96), (129, 32), (67, 2816)])
def test_dequantize_exact(ctx, type_, nrows, n):
    rng = np.random.default_rng(nrows + n)
    raw = O.quantize(type_, rows(rng, nrows, n))
    if type_ == MX:
        raw = rng.integers(0, 256, raw.shape, dtype=np.uint8)      # every scale byte and code
    ref = O.dequantize(type_, raw, n)
    for so, do in ((0, 0), (1 if type_ == MX else 2, 4)):
        src = M.DeviceBuffer(raw.nbytes + 8).upload(raw, so)
        dst = M.to_device(np.full(nrows * n + 8, 7.0, np.float32))
        M.check("dequantize", ctx.dequantize(type_, src.addr + so, dst.addr + do, nrows, n))
        got = dst.download(np.float32, (nrows * n + 8,))
        assert np.array_equal(got[do // 4:do // 4 + nrows * n].reshape(nrows, n), ref, equal_nan=True)
        assert (got[:do // 4] == 7.0).all() and (got[do // 4 + nrows * n:] == 7.0).all()


def test_refusals(ctx):
    b = M.DeviceBuffer(1 << 16)
    assert ctx.quantize(MX, b, b, 1, 48) == M.ERR_SHAPE and ctx.quantize(MX, b, b, -1, 32) == M.ERR_SHAPE
    assert ctx.quantize(MX, b.addr + 2, b, 1, 32) == M.ERR_UNSUPPORTED and ctx.quantize(MX, None, b, 1, 32) == M.ERR_NULL
    assert ctx.quantize(MX, b, b, 0, 32) == 0 and ctx.dequantize(MX, b, b, 0, 32) == 0
    assert ctx.dequantize(M.TYPE_Q4_K, b, b, 1, 256) == M.ERR_TYPE and ctx.dequantize(M.TYPE_F32, b, b, 1, 32) == M.ERR_TYPE
    assert ctx.dequantize(MX, b, b, 1, 33) == M.ERR_SHAPE and ctx.dequantize(MX, b, b.addr + 2, 1, 32) == M.ERR_UNSUPPORTED
    assert ctx.dequantize(MX, b, None, 1, 32) == M.ERR_NULL
    t = lambda ty, ne, nb=None: M.tensor(b, ty, ne, nb)
    f, i = M.TYPE_F32, M.TYPE_I32
    ok = (t(MX, [64, 8, 2]), t(f, [64, 1, 1]), t(i, [2, 1]), t(f, [8, 2, 1]))
    assert ctx.mul_mat_id(t(MX, [48, 8, 2]), t(f, [48, 1, 1]), ok[2], ok[3]) == M.ERR_UNSUPPORTED
    assert ctx.mul_mat_id(ok[0], t(f, [96, 1, 1]), ok[2], ok[3]) == M.ERR_SHAPE
    assert ctx.mul_mat_id(t(MX, [64, 8, 2], [17, 33, 272, 544]), ok[1], ok[2], ok[3]) == M.ERR_SHAPE
    assert ctx.mul_mat_id(ok[0], ok[1], ok[2], t(M.TYPE_F16, [8, 2, 1])) == M.ERR_TYPE
    # one family per layer; no tiled copies of MXFP4
    lay = M.make_layer(64, 2, 1, 32, b, None, t(MX, [64, 64, 2]), None, t(M.TYPE_Q8_0, [32, 64, 2]), True, M.ACT_SILU)
    assert ctx.forward(lay, b, 1, None, b) == M.ERR_UNSUPPORTED
    lay = M.make_layer(64, 2, 1, 32, b, None, t(MX, [64, 64, 2]), None, t(MX, [32, 64, 2]), True, M.ACT_SILU)
    lay.gate_tiled = lay.gate
    assert ctx.forward(lay, b, 1, None, b) == M.ERR_TYPE and M.tiled_bytes(lay.gate) == M.ERR_TYPE


# ------------------------------------------------------------------ products
def run_product(ctx, raw, b, ids, pad=0, offset=0, stream=None):
    """raw [E, N, row]; rows pad bytes apart, the table at a byte offset; dst starts as 9s"""
    E, N, rb = raw.shape
    T, K = ids.shape
    n = b.shape[-1]
    wide = np.full((E, N, rb + pad), 0xFF, np.uint8)
    wide[..., :rb] = raw
    w = M.DeviceBuffer(wide.nbytes + 16).upload(wide, offset)
    nb1 = rb + pad
    dst = M.to_device(np.full((T, K, N), 9.0, np.float32))
    bd, idd = M.to_device(b.astype(np.float32)), M.to_device(ids.astype(np.int32))
    rc = ctx.mul_mat_id(M.tensor(w, MX, [n, N, E], [17, nb1, nb1 * N, nb1 * N * E], offset=offset), M.tensor(bd, M.TYPE_F32, [n, b.shape[1], T]),
                        M.tensor(idd, M.TYPE_I32, [K, T]), M.tensor(dst, M.TYPE_F32, [N, K, T]), stream)
    M.check("mul_mat_id", rc)
    M.synchronize()
    return dst.download(np.float32, (T, K, N))


def check_product(got, raw, b, ids, few):
    ref = X.product(raw, b, ids)
    size = X.product_sizes(raw, b, ids)
    n = b.shape[-1]
    tol = 2.0 ** -24 * np.abs(ref) + 2.0 ** -50 * size if few else 2.0 ** -24 * np.abs(ref) + n / 16 * 2.0 ** -23 * 2 * size
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    off = np.abs(got - ref)
    assert not (off > tol)[~np.isnan(ref)].any(), (np.nanmax(off / np.maximum(tol, 1e-300)), np.argwhere(off > tol)[:4])


SHAPES = [(32, 1), (32, 16), (64, 33), (96, 64), (704, 70), (2048, 160), (2112, 48), (2816, 257), (1056, 129)]


@pytest.mark.parametrize("path", ["few", "gemm"])
@pytest.mark.parametrize("n,N", SHAPES)
@pytest.mark.parametrize("own_rows", [False, True])
def test_product_shapes(ctx, path, n, N, own_rows):
    rng = np.random.default_rng(n * 1000 + N)
    E, K = 6, 3
    raw = table(rng, E, N, n)
    ctx.set_gemm_threshold(1 if path == "gemm" else 1 << 40)
    try:
        for T in (1, 2, 5, 47, 150):
            b = rows(rng, T, K if own_rows else 1, n)
            ids = np.stack([rng.permutation(E)[:K] for _ in range(T)])
            check_product(run_product(ctx, raw, b, ids), raw, b, ids, path == "few")
    finally:
        ctx.set_gemm_threshold(0)


@pytest.mark.parametrize("kind", [1, 2, 5])
@pytest.mark.parametrize("n,N", SHAPES)
def test_product_row_tiles(ctx, kind, n, N):
    """every row tile of the GEMM, at row counts below, at and past it"""
    rng = np.random.default_rng(n + N + kind)
    raw = table(rng, 3, N, n)
    ctx.set_gemm_threshold(1)
    ctx.set_gemm_tiles(kind)
    try:
        for counts in ((1, 0, 31), (32, 33, 64), (65, 128, 129), (127, 260, 2)):
            ids = rng.permutation(np.repeat(np.arange(3), counts))[:, None]
            b = rows(rng, len(ids), 1, n)
            check_product(run_product(ctx, raw, b, ids), raw, b, ids, False)
    finally:
        ctx.set_gemm_threshold(0)
        ctx.set_gemm_tiles(0)


@pytest.mark.parametrize("path", ["few", "gemm"])
@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (2, 3), (7, 2), (15, 5)])
def test_product_any_alignment(ctx, path, pad, offset):
    rng = np.random.default_rng(pad + 16 * offset)
    raw = table(rng, 4, 50, 352)
    b, ids = rows(rng, 9, 1, 352), rng.integers(0, 4, (9, 2))
    ctx.set_gemm_threshold(1 if path == "gemm" else 1 << 40)
    try:
        check_product(run_product(ctx, raw, b, ids, pad, offset), raw, b, ids, path == "few")
    finally:
        ctx.set_gemm_threshold(0)


@pytest.mark.parametrize("path", ["few", "gemm"])
def test_product_hot_expert_and_bad_ids(ctx, path):
    """every slot on one expert, the same expert twice in a token, ids outside: zero rows, counted"""
    rng = np.random.default_rng(11)
    raw = table(rng, 5, 96, 320)
    b = rows(rng, 300, 2, 320)
    ids = np.full((300, 2), 3)
    ctx.set_gemm_threshold(1 if path == "gemm" else 1 << 40)
    try:
        check_product(run_product(ctx, raw, b, ids), raw, b, ids, path == "few")
        ids = rng.integers(-2, 7, (300, 2))
        ctx.take_errors()
        check_product(run_product(ctx, raw, b, ids), raw, b, ids, path == "few")
        assert ctx.take_errors()[0] == int(((ids < 0) | (ids >= 5)).sum())
        ids[:] = 99
        assert not run_product(ctx, raw, b, ids).any()
    finally:
        ctx.take_errors()
        ctx.set_gemm_threshold(0)


@pytest.mark.parametrize("path", ["few", "gemm"])
def test_product_values_at_the_edges(ctx, path):
    """NaN blocks, the smallest and largest scales, rows with NaN, infinities, zeros, 1e30 and 1e-30"""
    rng = np.random.default_rng(12)
    raw = table(rng, 3, 40, 160)
    raw[0, 3, 17] = 255                    # row 3, block 1: NaN
    raw[1, :, 0] = 0                       # 2^-127
    raw[1, 5, 34] = 200                    # 2^73 in one block of a row
    raw[2, :, 51] = 230
    b = rows(rng, 12, 1, 160)
    b[0] = 0.0
    b[1, 0, 70], b[2, 0, 0], b[3, 0, 159] = np.nan, np.inf, -np.inf
    b[4, 0, :32], b[5, 0] = 1e30, b[5, 0] * 1e-30
    b[6, 0, 32:64], b[7, 0, 5] = 0.0, 8.0e6
    ids = np.tile(np.array([[0, 1, 2]]), (12, 1))
    ctx.set_gemm_threshold(1 if path == "gemm" else 1 << 40)
    try:
        got = run_product(ctx, raw, b, ids)
        ref = X.product(raw, b, ids)
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        size = X.product_sizes(raw, b, ids)
        # (products of the smallest scales may flush below the smallest normal number)
        tol = 2.0 ** -24 * np.abs(ref) + (2.0 ** -50 if path == "few" else 2 * 160 / 16 * 2.0 ** -23) * size + 160 * 2.0 ** -126
        assert (np.abs(got - ref) <= tol)[~np.isnan(ref)].all()
    finally:
        ctx.set_gemm_threshold(0)


def test_product_of_no_tokens(ctx):
    raw = table(np.random.default_rng(1), 2, 16, 32)
    w = M.to_device(raw)
    rc = ctx.mul_mat_id(M.tensor(w, MX, [32, 16, 2]), M.tensor(w, M.TYPE_F32, [32, 1, 0]), M.tensor(w, M.TYPE_I32, [2, 0]),
                        M.tensor(w, M.TYPE_F32, [16, 2, 0]))
    assert rc == 0


# ------------------------------------------------------------------ layers
class Layer:
    def __init__(self, D, E, K, I, fused, act, seed, gating=0, shared=0, sh_gate_inp=False, bias=False):
        rng = np.random.default_rng(seed)
        self.D, self.E, self.K, self.I, self.gating = D, E, K, I, gating
        self.host = dict(D=D, E=E, K=K, I=I, fused=fused, act=act, gate_type=MX, down_type=MX,
                         router_w=(rng.standard_normal((E, D)) * 0.05).astype(np.float32), router_b=None)
        self.host["gate"] = table(rng, E, 2 * I if fused else I, D)
        self.host["up"] = None if fused or act == 4 else table(rng, E, I, D)
        self.host["down"] = table(rng, E, D, I)
        self.keep = keep = {k: M.to_device(v) for k, v in self.host.items() if isinstance(v, np.ndarray)}
        up = None if self.host["up"] is None else M.tensor(keep["up"], MX, [D, I, E])
        L = M.make_layer(D, E, K, I, keep["router_w"], None, M.tensor(keep["gate"], MX, [D, 2 * I if fused else I, E]), up,
                         M.tensor(keep["down"], MX, [I, D, E]), fused, act)
        L.gating = gating
        self.scale = self.sel_bias = None
        if gating == 1:
            self.sel_bias = (rng.standard_normal(E) * 0.05).astype(np.float32)
            keep["sel_bias"] = M.to_device(self.sel_bias)
            L.sel_bias, L.routed_scaling, L.gate_eps = keep["sel_bias"].addr, 2.5, 1e-20
        if gating == 2:
            self.scale = rng.uniform(0.5, 1.5, E).astype(np.float32)
            keep["scale"] = M.to_device(self.scale)
            L.expert_scale = keep["scale"].addr
        self.shared = None
        if shared:
            sh = self.shared = dict(I=shared, fused=False, act=act, gate=table(rng, 1, shared, D), up=None if act == 4 else table(rng, 1, shared, D),
                                    down=table(rng, 1, D, shared))
            for k in ("gate", "up", "down"):
                if sh[k] is not None:
                    keep["sh_" + k] = M.to_device(sh[k])
                    setattr(L, "sh_" + k, M.tensor(keep["sh_" + k], MX, [shared, D] if k == "down" else [D, shared]))
            L.sh_n_ff, L.sh_act = shared, act
            if sh_gate_inp:
                sh["inp"] = (rng.standard_normal((1, D)) * 0.05).astype(np.float32)
                keep["sh_inp"] = M.to_device(sh["inp"])
                L.sh_gate_inp = keep["sh_inp"].addr
        self.L = L

    def route(self, x):
        """the oracle's ids and weights (logits, ids: bit for bit the library's)"""
        return O.route_gated(O.router_logits(self.host["router_w"], None, x), self.K, self.gating, self.sel_bias, self.scale,
                             2.5 if self.gating == 1 else 1.0, 1e-20 if self.gating == 1 else 0.0)

    def reference(self, x, res, xr=None):
        sel, w = self.route(x if xr is None else xr)
        y = X.ffn(self.host, x, sel, sel, w)
        if self.shared:
            T = len(x)
            s = 1.0 / (1.0 + np.exp(-(x.astype(np.float64) @ self.shared["inp"][0].astype(np.float64)))) if "inp" in self.shared else np.ones(T)
            z = np.zeros((T, 1), np.int32)
            y = y + X.ffn(self.shared, x, z, z, s[:, None].astype(np.float32))
        return y + (0 if res is None else res)


def check_layer(got, ref, moe_size, few):
    e = float(np.linalg.norm(got - ref) / np.linalg.norm(ref))
    if few:
        assert (np.abs(got - ref) <= 2.0 ** -20 * moe_size + 2.0 ** -23 * np.abs(ref)).all(), e
    else:
        assert e <= 1e-3, e
    return e


def sizes(lay, x, xr=None):
    """a bound of the terms' sizes: the slots' weighted outputs by their absolute values"""
    sel, w = lay.route(x if xr is None else xr)
    with np.errstate(all="ignore"):
        y = X.ffn_slots(lay.host, x, sel, sel)
    s = (np.abs(y) * np.abs(w[..., None])).sum(1)
    if lay.shared:
        z = np.zeros((len(x), 1), np.int32)
        s = s + np.abs(X.ffn_slots(lay.shared, x, z, z))[:, 0]
    return s


LAYERS = {
    "moondream_like": dict(D=512, E=16, K=4, I=256, fused=True, act=1),
    "qwen_like": dict(D=512, E=16, K=8, I=96, fused=False, act=0),
    "gemma_like": dict(D=352, E=8, K=2, I=160, fused=False, act=2, gating=2),
    "nemotron_like": dict(D=672, E=12, K=6, I=224, fused=False, act=4, gating=1, shared=448),
    "talker_like": dict(D=512, E=8, K=3, I=128, fused=False, act=0, shared=256, sh_gate_inp=True),
    "erf": dict(D=64, E=4, K=1, I=32, fused=True, act=3),
    "wide": dict(D=2816, E=64, K=8, I=704, fused=False, act=2),
}


@pytest.mark.parametrize("name", LAYERS)
@pytest.mark.parametrize("path", ["default", "few", "gemm"])
def test_layer(ctx, name, path):
    lay = Layer(seed=len(name), **LAYERS[name])
    rng = np.random.default_rng(21)
    ctx.set_gemm_threshold({"default": 0, "few": 1 << 40, "gemm": 1}[path])
    try:
        for T in (1, 2, 3, 8, 16) + ((70,) if name != "wide" else ()):
            few = path == "few" or (path == "default" and T * lay.K <= 2 * lay.E)
            x, res = rows(rng, T, lay.D), rows(rng, T, lay.D)
            out = M.DeviceBuffer(4 * T * lay.D)
            sel = M.DeviceBuffer(4 * T * lay.K)
            r = M.Routing()
            r.sel = sel.addr
            M.check("forward", ctx.forward(lay.L, M.to_device(x), T, M.to_device(res), out, r))
            M.synchronize()
            assert np.array_equal(sel.download(np.int32, (T, lay.K)), lay.route(x)[0])
            e = check_layer(out.download(np.float32, (T, lay.D)), lay.reference(x, res), sizes(lay, x), few)
            print(f"{name} {path} T={T}: rel-L2 {e:.2e}", flush=True)
    finally:
        ctx.set_gemm_threshold(0)


@pytest.mark.parametrize("kind", [M.NORM_RMS, M.NORM_LAYER])
def test_layer_norm_equals_norm_then_forward(ctx, kind):
    lay = Layer(seed=3, **LAYERS["qwen_like"])
    rng = np.random.default_rng(kind)
    w, b = M.to_device(rows(rng, 512)), M.to_device(rows(rng, 512))
    norm = M.make_norm(kind, 1e-6, w, b if kind == M.NORM_LAYER else None)
    for T in (1, 5, 16, 90):
        h = M.to_device(rows(rng, T, 512))
        hn, a, c = (M.DeviceBuffer(4 * T * 512) for _ in range(3))
        M.check("norm", ctx.norm(norm, h, T, 512, hn))
        M.check("forward", ctx.forward(lay.L, hn, T, h, a))
        M.check("forward_norm", ctx.forward_norm(lay.L, norm, h, T, h, c))
        M.synchronize()
        assert np.array_equal(a.download(np.uint8, (4 * T * 512,)), c.download(np.uint8, (4 * T * 512,)))


def test_router_input_and_in_place(ctx):
    lay = Layer(seed=4, **LAYERS["gemma_like"])
    rng = np.random.default_rng(8)
    for T in (1, 7, 60):
        x, xr, res = rows(rng, T, 352), rows(rng, T, 352), rows(rng, T, 352)
        out = M.to_device(res)
        M.check("router_input", ctx.forward_router_input(lay.L, M.to_device(x), M.to_device(xr), T, out, out))
        M.synchronize()
        check_layer(out.download(np.float32, (T, 352)), lay.reference(x, res, xr), sizes(lay, x, xr), T * lay.K <= 2 * lay.E)


def test_expert_ffn_caller_ids(ctx):
    """two id sets, ids outside in each: their slots add nothing and are counted"""
    lay = Layer(seed=5, **LAYERS["moondream_like"])
    rng = np.random.default_rng(9)
    for T in (1, 2, 6, 40):
        x = rows(rng, T, 512)
        gu, dn = rng.integers(-1, 18, (T, 4)), rng.integers(-1, 18, (T, 4))
        w = rng.uniform(0, 1, (T, 4)).astype(np.float32)
        out = M.DeviceBuffer(4 * T * 512)
        ctx.take_errors()
        M.check("expert_ffn", ctx.expert_ffn(lay.L, M.to_device(x), T, None, M.to_device(gu.astype(np.int32)), M.to_device(dn.astype(np.int32)),
                                             M.to_device(w), out))
        assert ctx.take_errors()[0] == int(((gu < 0) | (gu >= 16)).sum() + ((dn < 0) | (dn >= 16)).sum())
        ref = X.ffn(lay.host, x, gu, dn, w)
        got = out.download(np.float32, (T, 512))
        assert np.linalg.norm(got - ref) <= 1e-3 * np.linalg.norm(ref) + 1e-20
        dead = ~(((gu >= 0) & (gu < 16)) & ((dn >= 0) & (dn < 16))).any(1)
        assert not got[dead].any()


def test_noalloc_equals_chain(ctx):
    lay = Layer(seed=6, **LAYERS["qwen_like"])
    rng = np.random.default_rng(10)
    c = M.Context(0)
    c.reserve(64, 512, 96, 16, 8)
    c.set_fused_decode(M.DECODE_CHAIN)
    for T in (1, 6, 64):
        x = M.to_device(rows(rng, T, 512))
        a, b = M.DeviceBuffer(4 * T * 512), M.DeviceBuffer(4 * T * 512)
        M.check("noalloc", M.forward_noalloc(lay.L, x, T, x, a))
        M.check("forward", c.forward(lay.L, x, T, x, b))
        M.synchronize()
        assert np.array_equal(a.download(np.uint8, (4 * T * 512,)), b.download(np.uint8, (4 * T * 512,)))
    c.close()


def test_graph_replays(ctx):
    """a decode step captured and replayed on rewritten inputs, eager work between the replays"""
    lay = Layer(seed=7, **LAYERS["qwen_like"])
    rng = np.random.default_rng(13)
    st = M.Stream()
    for T in (1, 9, 80):
        x, out, eager = (M.DeviceBuffer(4 * T * 512) for _ in range(3))
        x.upload(rows(rng, T, 512))
        g = M.Graph(st, lambda s: M.check("forward", ctx.forward(lay.L, x, T, x, out, None, s.addr)))
        for _ in range(4):
            x.upload(rows(rng, T, 512))
            M.synchronize()
            g.launch(st)
            st.synchronize()
            M.check("forward", ctx.forward(lay.L, x, T, x, eager))
            M.synchronize()
            assert np.array_equal(out.download(np.uint8, (4 * T * 512,)), eager.download(np.uint8, (4 * T * 512,)))
        g.destroy()
    st.destroy()


def test_quantize_then_layer_run_together(ctx):
    """as a program uses them: tables quantized on the GPU, a prefill and decode steps of the layer on a stream"""
    rng = np.random.default_rng(14)
    D, E, K, I = 512, 16, 4, 256
    wf = {"gate": (rng.standard_normal((E, 2 * I, D)) * 0.02).astype(np.float32), "down": (rng.standard_normal((E, D, I)) * 0.02).astype(np.float32)}
    dev, host = {}, dict(D=D, E=E, K=K, I=I, fused=True, act=1, up=None)
    st = M.Stream()
    for k, v in wf.items():
        n = v.shape[-1]
        dev[k] = M.DeviceBuffer(v.size // 32 * 17)
        M.check("quantize", ctx.quantize(MX, M.to_device(v), dev[k], v.size // n, n, st.addr))
        st.synchronize()
        host[k] = dev[k].download(np.uint8, (*v.shape[:-1], n // 32 * 17))
        back = M.DeviceBuffer(v.nbytes)
        M.check("dequantize", ctx.dequantize(MX, dev[k], back, v.size // n, n, st.addr))
        st.synchronize()
        assert np.array_equal(back.download(np.float32, v.shape), X.values(host[k]).astype(np.float32))
    rw = (rng.standard_normal((E, D)) * 0.05).astype(np.float32)
    rd = M.to_device(rw)
    L = M.make_layer(D, E, K, I, rd, None, M.tensor(dev["gate"], MX, [D, 2 * I, E]), None, M.tensor(dev["down"], MX, [I, D, E]), True, 1)
    for T in (200, 1, 1, 3):
        x = rows(rng, T, D)
        out = M.DeviceBuffer(4 * T * D)
        xd = M.to_device(x)
        M.check("forward", ctx.forward(L, xd, T, None, out, None, st.addr))
        st.synchronize()
        sel, w = O.route_gated(O.router_logits(rw, None, x), K, 0)
        ref = X.ffn(host, x, sel, sel, w)
        got = out.download(np.float32, (T, D))
        assert np.linalg.norm(got - ref) <= (1e-3 if T * K > 2 * E else 1e-6) * np.linalg.norm(ref)
    st.destroy()


# ------------------------------------------------------------------ a few tokens' launches
# (the launches take norm and router up to 4 tokens and rows of 64-value chunks up to 4096, the rest up to 32 tokens)
FEW = {
    "eleven_chunks": dict(D=704, E=5, K=2, I=32, fused=True, act=0),
    "no_chunks": dict(D=96, E=7, K=3, I=96, fused=False, act=1),
    "widest": dict(D=4096, E=6, K=2, I=64, fused=False, act=2, gating=2),
    "past_widest": dict(D=4160, E=6, K=2, I=64, fused=True, act=3),
    "many_experts": dict(D=64, E=256, K=10, I=32, fused=False, act=4, gating=1),
    "every_expert": dict(D=128, E=32, K=32, I=32, fused=False, act=0),
    "long_down": dict(D=128, E=16, K=6, I=2080, fused=False, act=4, gating=1, shared=4128),
    "gated_shared": dict(D=320, E=12, K=3, I=1056, fused=False, act=0, shared=96, sh_gate_inp=True),
}


def check_few(got, ref, size, K):
    """the tolerance of layers of few rows (above) for K slots and a shared expert"""
    assert (np.abs(got - ref) <= ((K + 4) * 2.0 ** -24 + 2.0 ** -21) * size + 2.0 ** -23 * np.abs(ref)).all()


@pytest.fixture(scope="module")
def few_ctx():
    c = M.Context(0)
    c.reserve(24, 4160, 2080, 256, 32)
    yield c
    c.set_fused_decode(M.DECODE_FUSED)
    c.close()


@pytest.mark.parametrize("name", FEW)
def test_few_tokens(few_ctx, name):
    """the few launches and the separate ones against the float64 form, at and past the sizes where they change"""
    lay = Layer(seed=40 + len(name), **FEW[name])
    rng = np.random.default_rng(len(name))
    few_ctx.set_gemm_threshold(1 << 40)
    for T in (1, 2, 3, 4, 5, 15, 16, 17):
        x, res = rows(rng, T, lay.D), rows(rng, T, lay.D)
        ref, size = lay.reference(x, res), sizes(lay, x)
        xd, rd = M.to_device(x), M.to_device(res)
        for mode in (M.DECODE_FUSED, M.DECODE_CHAIN):
            few_ctx.set_fused_decode(mode)
            out = M.to_device(np.full((T + 1, lay.D), 7.0, np.float32))
            M.check("forward", few_ctx.forward(lay.L, xd, T, rd, out))
            M.synchronize()
            got = out.download(np.float32, (T + 1, lay.D))
            assert (got[T] == 7.0).all()
            check_few(got[:T], ref, size, lay.K)


@pytest.mark.parametrize("kind", [M.NORM_RMS, M.NORM_LAYER])
@pytest.mark.parametrize("name", ["eleven_chunks", "no_chunks", "widest", "gated_shared"])
def test_few_tokens_norm(few_ctx, name, kind):
    """the norm inside equals the norm in front bit for bit; weights and bias at any 4 bytes, out over the rows"""
    lay = Layer(seed=50 + len(name), **FEW[name])
    rng = np.random.default_rng(len(name) + kind)
    few_ctx.set_gemm_threshold(1 << 40)
    few_ctx.set_fused_decode(M.DECODE_FUSED)
    w, b = M.to_device(rows(rng, lay.D + 1)), M.to_device(rows(rng, lay.D + 3))
    for norm in (M.make_norm(kind, 1e-5, w.addr + 4, b.addr + 12 if kind == M.NORM_LAYER else None), M.make_norm(kind, 1e-5, None, None)):
        for T in (1, 3, 4, 5):
            h = M.to_device(rows(rng, T, lay.D))
            hn, a = M.DeviceBuffer(4 * T * lay.D), M.DeviceBuffer(4 * T * lay.D)
            M.check("norm", few_ctx.norm(norm, h, T, lay.D, hn))
            M.check("forward", few_ctx.forward(lay.L, hn, T, h, a))
            M.check("forward_norm", few_ctx.forward_norm(lay.L, norm, h, T, h, h))
            M.synchronize()
            assert np.array_equal(a.download(np.uint8, (4 * T * lay.D,)), h.download(np.uint8, (4 * T * lay.D,)))


def test_few_tokens_not_a_number(few_ctx):
    """a token with a NaN, an infinity, or values past the range of an fp16 scale: itself alone"""
    lay = Layer(seed=60, **FEW["eleven_chunks"])
    rng = np.random.default_rng(61)
    few_ctx.set_gemm_threshold(1 << 40)
    x = rows(rng, 4, 704)
    clean = x.copy()
    x[0, 5], x[1, 700], x[2, 64] = np.nan, np.inf, 1e9
    for mode in (M.DECODE_FUSED, M.DECODE_CHAIN):
        few_ctx.set_fused_decode(mode)
        got = []
        for v in (x, clean):
            out = M.DeviceBuffer(4 * 4 * 704)
            M.check("forward", few_ctx.forward(lay.L, M.to_device(v), 4, None, out))
            M.synchronize()
            got.append(out.download(np.float32, (4, 704)))
        assert np.isnan(got[0][:3]).all()
        assert np.array_equal(got[0][3], got[1][3]) and np.isfinite(got[1]).all()


def test_few_tokens_norm_graph(few_ctx):
    lay = Layer(seed=62, **FEW["gated_shared"])
    rng = np.random.default_rng(63)
    few_ctx.set_gemm_threshold(0)
    few_ctx.set_fused_decode(M.DECODE_FUSED)
    norm = M.make_norm(M.NORM_RMS, 1e-6, M.to_device(rows(rng, 320)), None)
    st = M.Stream()
    for T in (1, 4, 7):
        x, out, eager = (M.DeviceBuffer(4 * T * 320) for _ in range(3))
        x.upload(rows(rng, T, 320))
        g = M.Graph(st, lambda s: M.check("forward_norm", few_ctx.forward_norm(lay.L, norm, x, T, x, out, None, s.addr)))
        for _ in range(3):
            x.upload(rows(rng, T, 320))
            M.synchronize()
            g.launch(st)
            st.synchronize()
            M.check("forward_norm", few_ctx.forward_norm(lay.L, norm, x, T, x, eager))
            M.synchronize()
            assert np.array_equal(out.download(np.uint8, (4 * T * 320,)), eager.download(np.uint8, (4 * T * 320,)))
        g.destroy()
    st.destroy()


@pytest.mark.parametrize("T,K,shift", [(1, 1, 0), (3, 4, 4), (8, 8, 0), (8, 8, 8), (70, 8, 0), (90, 6, 12)])
def test_product_of_few_rows_by_ids(ctx, T, K, shift):
    """rows that the work-groups make operands of themselves, and (rows off 16 bytes, more than 512 rows) that another
    launch does; ids outside, each expert's rows odd in number"""
    n, N, E = 2080, 96, 64
    rng = np.random.default_rng(T + K)
    raw = table(rng, E, N, n)
    ctx.set_gemm_threshold(1 << 40)
    try:
        for own in (False, True):
            b = rows(rng, T, K if own else 1, n)
            ids = rng.integers(-1, 6, (T, K)) if T > 1 else np.array([[E - 1]])
            bd = M.DeviceBuffer(b.nbytes + 16).upload(b, shift)
            out = M.to_device(np.full((T * K + 1, N), 7.0, np.float32))
            ctx.take_errors()
            wd, idd = M.to_device(raw), M.to_device(ids.astype(np.int32))
            M.check("mul_mat_id", ctx.mul_mat_id(M.tensor(wd, MX, [n, N, E]), M.tensor(bd.addr + shift, M.TYPE_F32, [n, b.shape[1], T]),
                                                 M.tensor(idd, M.TYPE_I32, [K, T]), M.tensor(out, M.TYPE_F32, [N, K, T])))
            M.synchronize()
            assert ctx.take_errors()[0] == (ids < 0).sum()
            got = out.download(np.float32, (T * K + 1, N))
            assert (got[-1] == 7.0).all() and not got[:-1].reshape(T, K, N)[ids < 0].any()
            check_product(got[:-1].reshape(T, K, N), raw, b, ids, True)
    finally:
        ctx.set_gemm_threshold(0)


def test_few_tokens_at_their_largest(ctx):
    """31, 32 (the last that the few launches take) and 33 tokens"""
    lay = Layer(seed=70, **FEW["gated_shared"])
    rng = np.random.default_rng(71)
    ctx.set_gemm_threshold(1 << 40)
    try:
        for T in (31, 32, 33):
            x, res = rows(rng, T, 320), rows(rng, T, 320)
            out = M.DeviceBuffer(4 * T * 320)
            xd, rd = M.to_device(x), M.to_device(res)
            M.check("forward", ctx.forward(lay.L, xd, T, rd, out))
            M.synchronize()
            check_few(out.download(np.float32, (T, 320)), lay.reference(x, res), sizes(lay, x), lay.K)
    finally:
        ctx.set_gemm_threshold(0)


def test_product_tiles_same_bits(ctx):
    """a row's sums do not depend on the tile that it is in"""
    rng = np.random.default_rng(72)
    raw, b = table(rng, 4, 300, 704), rows(rng, 333, 1, 704)
    ids = rng.integers(0, 4, (333, 2))
    ctx.set_gemm_threshold(1)
    try:
        got = []
        for kind in (1, 2):
            ctx.set_gemm_tiles(kind)
            got.append(run_product(ctx, raw, b, ids))
        assert np.array_equal(got[0], got[1])
    finally:
        ctx.set_gemm_threshold(0)
        ctx.set_gemm_tiles(0)


@pytest.mark.parametrize("T", [1, 3, 20, 80])
def test_layer_rows_off_16_bytes(ctx, T):
    lay = Layer(seed=73, **LAYERS["qwen_like"])
    rng = np.random.default_rng(74)
    x, res = rows(rng, T, 512), rows(rng, T, 512)
    got = []
    for off in (0, 4):
        xd, rd = M.DeviceBuffer(x.nbytes + 16).upload(x, off), M.DeviceBuffer(x.nbytes + 16).upload(res, off)
        out = M.DeviceBuffer(x.nbytes + 16)
        M.check("forward", ctx.forward(lay.L, xd.addr + off, T, rd.addr + off, out.addr + off))
        M.synchronize()
        got.append(out.download(np.float32, (T, 512), off))
        check_layer(got[-1], lay.reference(x, res), sizes(lay, x), T * lay.K <= 2 * lay.E)


def test_two_contexts_on_two_streams(ctx):
    """calls that run side by side, each context's workspace its own"""
    lay = Layer(seed=75, **LAYERS["nemotron_like"])
    rng = np.random.default_rng(76)
    other = M.Context(0)
    other.reserve(64, 672, 448, 12, 6)
    streams = (M.Stream(), M.Stream())
    try:
        for T in (1, 4, 12, 60):
            x = [M.to_device(rows(rng, T, 672)) for _ in range(2)]
            alone = []
            for c, v in zip((ctx, other), x):
                o = M.DeviceBuffer(4 * T * 672)
                M.check("forward", c.forward(lay.L, v, T, v, o))
                M.synchronize()
                alone.append(o.download(np.uint8, (4 * T * 672,)))
            outs = [M.DeviceBuffer(4 * T * 672) for _ in range(2)]
            for _ in range(8):
                for c, v, o, st in zip((ctx, other), x, outs, streams):
                    M.check("forward", c.forward(lay.L, v, T, v, o, None, st.addr))
            for st in streams:
                st.synchronize()
            for a, o in zip(alone, outs):
                assert np.array_equal(a, o.download(np.uint8, (4 * T * 672,)))
    finally:
        for st in streams:
            st.destroy()
        other.close()
