"""Calls of MXFP4 layers and products beside those of test_gpu_mxfp4.py.  Tolerances as there."""
import pathlib
import subprocess

import numpy as np
import pytest

import _mxfp4 as X
import mimoe as M
import pyoracle as O
from test_gpu_mxfp4 import LAYERS, Layer, check_layer, check_product, rows, run_product, sizes, table

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


# ------------------------------------------------------------------ operands past a pass
def digit_bytes(n):
    """of an operand row of n values: 96 a block, whole pairs of blocks"""
    return (n // 32 + 1) // 2 * 192


def layer_bytes(lay, tokens):
    return tokens * max(digit_bytes(lay.D), lay.K * digit_bytes(lay.I))


@pytest.fixture
def passes(ctx):
    ctx.set_gemm_threshold(1)
    ctx.take_errors()
    yield ctx
    ctx.set_mx_pass_bytes(0)
    ctx.set_gemm_threshold(0)
    ctx.take_errors()


def test_pass_bytes_refusals_without_device():
    assert M.load().mi_moe_ctx_set_mx_pass_bytes(None, 0) == M.ERR_NULL


@gpu
def test_pass_bytes_refusals(passes):
    lib = M.load()
    assert [lib.mi_moe_ctx_set_mx_pass_bytes(passes.h, n) for n in (-1, 0xF0000001, 0xF0000000, 1, 0)] == [M.ERR_ARG, M.ERR_ARG, 0, 0, 0]


@gpu
@pytest.mark.parametrize("tokens", [1, 16, 33])
@pytest.mark.parametrize("name", ["moondream_like", "nemotron_like", "talker_like"])
def test_layer_in_passes(passes, name, tokens):
    """outputs and dispatch lists of the undivided call to the bit; the last pass is a short one"""
    lay = Layer(seed=83, **LAYERS[name])
    T = 70
    rng = np.random.default_rng(84)
    x, res = rows(rng, T, lay.D), rows(rng, T, lay.D)
    got = []
    for nbytes in (0, layer_bytes(lay, tokens) + 100):
        passes.set_mx_pass_bytes(nbytes)
        lists = {"counts": lay.E, "offsets": lay.E + 1, "perm": T * lay.K, "sel": T * lay.K}
        bufs = {k: M.DeviceBuffer(4 * n) for k, n in lists.items()}
        r = M.Routing()
        for k, b in bufs.items():
            setattr(r, k, b.addr)
        got.append([forward(passes, lay, x, res, r).view(np.int32).ravel()] + [bufs[k].download(np.int32, (n,)) for k, n in lists.items()])
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    check_layer(got[1][0].view(np.float32).reshape(T, lay.D), lay.reference(x, res), sizes(lay, x), False)


@gpu
@pytest.mark.parametrize("two_ids", [False, True])
def test_expert_ffn_in_passes(passes, two_ids):
    """the caller's ids, one or two buffers of them, some outside: the same rows and the same count"""
    lay = Layer(seed=85, **LAYERS["qwen_like"])
    T, E, K = 61, lay.E, lay.K
    rng = np.random.default_rng(86)
    x, w = rows(rng, T, lay.D), rng.random((T, K)).astype(np.float32)
    gu = rng.integers(-1, E + 1, (T, K)).astype(np.int32)
    dn = rng.integers(-1, E + 1, (T, K)).astype(np.int32) if two_ids else gu
    xd, wd, gd = M.to_device(x), M.to_device(w), M.to_device(gu)
    dd = M.to_device(dn) if two_ids else gd
    got = []
    for nbytes in (0, layer_bytes(lay, 20)):
        passes.set_mx_pass_bytes(nbytes)
        out = M.DeviceBuffer(4 * T * lay.D)
        M.check("expert_ffn", passes.expert_ffn(lay.L, xd, T, xd, gd, dd, wd, out))
        M.synchronize()
        got.append((out.download(np.float32, (T, lay.D)), passes.take_errors()[0]))
    assert np.array_equal(got[0][0].view(np.uint32), got[1][0].view(np.uint32))
    outside = sum(int(((i < 0) | (i >= E)).sum()) for i in ((gu, dn) if two_ids else (gu,)))
    assert got[0][1] == got[1][1] == outside
    ref = X.ffn(lay.host, x, gu, dn, w)
    assert np.linalg.norm(got[1][0] - x - ref) <= 1e-3 * np.linalg.norm(ref)


@gpu
@pytest.mark.parametrize("own_rows", [False, True])
def test_product_in_passes(passes, own_rows):
    rng = np.random.default_rng(87)
    raw = table(rng, 6, 40, 96)
    b = rows(rng, 50, 3 if own_rows else 1, 96)
    ids = rng.integers(-1, 7, (50, 3))
    whole = run_product(passes, raw, b, ids)
    assert passes.take_errors()[0] == int(((ids < 0) | (ids >= 6)).sum())
    for tokens in (1, 7, 25):
        passes.set_mx_pass_bytes(tokens * b.shape[1] * digit_bytes(96) + 50)
        got = run_product(passes, raw, b, ids)
        assert np.array_equal(got.view(np.uint32), whole.view(np.uint32)), tokens
        assert passes.take_errors()[0] == int(((ids < 0) | (ids >= 6)).sum())
    check_product(whole, raw, b, ids, False)


@gpu
@pytest.mark.parametrize("name", ["qwen_like", "nemotron_like"])
def test_a_token_past_a_pass(passes, name):
    """takes the products of few rows, at any count of tokens"""
    lay = Layer(seed=88, **LAYERS[name])
    rng = np.random.default_rng(89)
    passes.set_mx_pass_bytes(layer_bytes(lay, 1) - 1)
    for T in (1, 5, 70):
        x = rows(rng, T, lay.D)
        got = forward(passes, lay, x, x)
        check_layer(got, lay.reference(x, x), sizes(lay, x), not lay.shared or T <= 32)
    raw, ids = table(rng, 6, 40, 96), rng.integers(0, 6, (50, 3))
    b = rows(rng, 50, 3, 96)
    passes.set_mx_pass_bytes(3 * digit_bytes(96) - 1)
    check_product(run_product(passes, raw, b, ids), raw, b, ids, True)


# ------------------------------------------------------------------ the exact workspace
EXACT = {
    "one_block": dict(D=32, E=3, K=2, I=32, fused=True, act=0),
    "odd_blocks": dict(D=96, E=5, K=3, I=288, fused=False, act=1),
    "wide_shared": dict(D=160, E=4, K=4, I=96, fused=False, act=4, gating=1, shared=384),   # n_ff * n_expert_used
    "whole": dict(D=256, E=4, K=1, I=256, fused=False, act=2, shared=256, sh_gate_inp=True),
}


@gpu
@pytest.mark.parametrize("name", EXACT)
@pytest.mark.parametrize("threshold", [1, 1 << 40])
def test_exact_workspace(ctx, name, threshold):
    """a context reserved for the call alone gives the bits of a roomy one"""
    lay = Layer(seed=90, **EXACT[name])
    rng = np.random.default_rng(91)
    for T in (1, 37):
        tight = M.Context(0)
        tight.reserve(T, lay.D, lay.I, lay.E, lay.K)
        x, res = rows(rng, T, lay.D), rows(rng, T, lay.D)
        raw, ids = table(rng, lay.E, 48, lay.D), rng.integers(0, lay.E, (T, lay.K))
        b = rows(rng, T, lay.K, lay.D)
        got = []
        try:
            for c in (ctx, tight):
                c.set_gemm_threshold(threshold)
                got.append((forward(c, lay, x, res), run_product(c, raw, b, ids)))
        finally:
            ctx.set_gemm_threshold(0)
            tight.close()
        assert all(np.array_equal(p.view(np.uint32), q.view(np.uint32)) for p, q in zip(*got))
        check_layer(got[0][0], lay.reference(x, res), sizes(lay, x), threshold > 1)
        check_product(got[0][1], raw, b, ids, threshold > 1)


# ------------------------------------------------------------------ the C++ host mirror
SELFTEST = pathlib.Path(M.__file__).parent / "host" / "vqa_moe_selftest"


@gpu
def test_host_tensor_strides():
    r = subprocess.run([str(SELFTEST)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "tensor strides of 9 types" in r.stderr, r.stderr


@gpu
@pytest.mark.parametrize("same", [True, False])
@pytest.mark.parametrize("threshold", [1 << 30, 1])
def test_host_table_form(tmp_path, same, threshold):
    """vqa::moe::build_expert_ffn_table_res on MXFP4 tables"""
    rng = np.random.default_rng(92)
    D, I, E, K, T = 160, 96, 6, 3, 12
    L = dict(E=E, I=I, act=0, fused=False, gate=table(rng, E, I, D), up=table(rng, E, I, D), down=table(rng, E, D, I))
    x, res, w = rows(rng, T, D), rows(rng, T, D), rng.random((T, K)).astype(np.float32)
    gu = rng.integers(0, E, (T, K)).astype(np.int32)
    dn = gu if same else rng.integers(0, E, (T, K)).astype(np.int32)
    (tmp_path / "meta.txt").write_text(f"{T} {D} {I} {E} {K} {M.TYPE_MXFP4} {M.TYPE_MXFP4} 0 {int(same)} {threshold}\n")
    for name, a in (("x", x), ("res", res), ("gate", L["gate"]), ("up", L["up"]), ("down", L["down"]), ("ids_gu", gu), ("ids_dn", dn), ("w", w)):
        (tmp_path / f"{name}.bin").write_bytes(np.ascontiguousarray(a).tobytes())
    r = subprocess.run([str(SELFTEST), "--table", str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    got = np.fromfile(tmp_path / "out.bin", np.float32).reshape(T, D)
    y = np.abs(X.ffn_slots(L, x, gu, dn) * w[..., None]).sum(1)
    check_layer(got, res + X.ffn(L, x, gu, dn, w), y, threshold > 1)


# ------------------------------------------------------------------ shared experts of another type or activation
MIXED = {   # routed type, its act, the shared expert's type and act
    "mx_q8_0": (O.TYPE_MXFP4, 0, O.TYPE_Q8_0, 0),
    "mx_q4_k": (O.TYPE_MXFP4, 1, O.TYPE_Q4_K, 1),
    "mx_f32": (O.TYPE_MXFP4, 4, O.TYPE_F32, 4),
    "mx_other_act": (O.TYPE_MXFP4, 0, O.TYPE_MXFP4, 4),
    "mx_ungated": (O.TYPE_MXFP4, 4, O.TYPE_MXFP4, 0),
    "q8_0_mx": (O.TYPE_Q8_0, 0, O.TYPE_MXFP4, 0),
    "q4_k_mx": (O.TYPE_Q4_K, 2, O.TYPE_MXFP4, 3),
    "f32_mx": (O.TYPE_F32, 0, O.TYPE_MXFP4, 4),
}


@gpu
@pytest.mark.parametrize("gated_row", [False, True])
@pytest.mark.parametrize("name", MIXED)
def test_mixed_shared_expert(ctx, name, gated_row):
    """MXFP4 experts beside a shared expert of another type or activation, and an MXFP4 shared expert beside other tables:
    against the oracle, the norm inside against the norm apart, with lists asked for against without"""
    rt, act, st, sh_act = MIXED[name]
    D, E, K, I, S = 512, 10, 3, 256, 256
    rng = np.random.default_rng(93)
    w = lambda t, *shape: (lambda a: a if t == O.TYPE_F32 else O.quantize(t, a))((rng.standard_normal(shape) * 0.05).astype(np.float32))
    host = dict(D=D, E=E, K=K, I=I, act=act, fused=False, gate_type=rt, down_type=rt, router_w=(rng.standard_normal((E, D)) * 0.05).astype(np.float32),
                router_b=None, gate=w(rt, E, I, D), up=None if act == 4 else w(rt, E, I, D), down=w(rt, E, D, I),
                sh_I=S, sh_act=sh_act, sh_type=st, sh_down_type=st, sh_gate=w(st, S, D), sh_up=None if sh_act == 4 else w(st, S, D),
                sh_down=w(st, D, S), sh_gate_inp=(rng.standard_normal(D) * 0.05).astype(np.float32) if gated_row else None)
    dev = {k: M.to_device(v) for k, v in host.items() if isinstance(v, np.ndarray)}
    L = M.make_layer(D, E, K, I, dev["router_w"], None, M.tensor(dev["gate"], rt, [D, I, E]), None if act == 4 else M.tensor(dev["up"], rt, [D, I, E]),
                     M.tensor(dev["down"], rt, [I, D, E]), False, act)
    L.sh_n_ff, L.sh_act = S, sh_act
    L.sh_gate, L.sh_down = M.tensor(dev["sh_gate"], st, [D, S]), M.tensor(dev["sh_down"], st, [S, D])
    if sh_act != 4:
        L.sh_up = M.tensor(dev["sh_up"], st, [D, S])
    if gated_row:
        L.sh_gate_inp = dev["sh_gate_inp"].addr
    norm = M.make_norm(M.NORM_RMS, 1e-6)
    for T in (1, 3, 8, 70):
        x, res = rows(rng, T, D), rows(rng, T, D)
        xd, rd = M.to_device(x), M.to_device(res)
        outs = [M.DeviceBuffer(4 * T * D) for _ in range(4)]
        M.check("forward", ctx.forward(L, xd, T, rd, outs[0]))
        counts = M.DeviceBuffer(4 * E)
        r = M.Routing()
        r.counts = counts.addr
        M.check("forward", ctx.forward(L, xd, T, rd, outs[1], r))
        xn = M.DeviceBuffer(4 * T * D)
        M.check("norm", ctx.norm(norm, xd, T, D, xn))
        M.check("forward", ctx.forward(L, xn, T, rd, outs[2]))
        M.check("forward_norm", ctx.forward_norm(L, norm, xd, T, rd, outs[3]))
        M.synchronize()
        got = [o.download(np.float32, (T, D)) for o in outs]
        ref, dbg = O.moe_forward(host, x, res)
        e = float(np.linalg.norm(got[0] - ref) / np.linalg.norm(ref - res))
        print(f"{name} gated row {gated_row} T={T}: rel-L2 {e:.2e}", flush=True)
        assert e <= 1e-2
        assert np.array_equal(counts.download(np.int32, (E,)), dbg["counts"])
        assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
        assert np.array_equal(got[2].view(np.uint32), got[3].view(np.uint32))


# ------------------------------------------------------------------ addresses, graphs
@gpu
@pytest.mark.parametrize("T", [1, 3, 20, 80])
def test_layer_rows_off_16_bytes_same_bits(ctx, T):
    """the loads of rows off 16 bytes give the bits of aligned ones (another first launch up to 4 tokens)"""
    lay = Layer(seed=94, **LAYERS["qwen_like"])
    rng = np.random.default_rng(95)
    x, res = rows(rng, T, 512), rows(rng, T, 512)
    got = []
    for off in (0, 4):
        xd, rd = M.DeviceBuffer(x.nbytes + 16).upload(x, off), M.DeviceBuffer(x.nbytes + 16).upload(res, off)
        out = M.DeviceBuffer(x.nbytes + 16)
        M.check("forward", ctx.forward(lay.L, xd.addr + off, T, rd.addr + off, out.addr + off))
        M.synchronize()
        got.append(out.download(np.uint32, (T, 512), off))
    assert np.array_equal(*got)


@gpu
@pytest.mark.parametrize("T", [1, 6, 70])
def test_expert_ffn_graph(ctx, T):
    """captured and replayed with other rows and ids in the same buffers, eager calls between the replays"""
    lay = Layer(seed=96, **LAYERS["moondream_like"])
    rng = np.random.default_rng(97)
    D, E, K = lay.D, lay.E, lay.K
    xd, idd, wd, out, eager = M.DeviceBuffer(4 * T * D), M.DeviceBuffer(4 * T * K), M.DeviceBuffer(4 * T * K), M.DeviceBuffer(4 * T * D), M.DeviceBuffer(4 * T * D)

    def fill():
        x, ids, w = rows(rng, T, D), rng.integers(0, E, (T, K)).astype(np.int32), rng.random((T, K)).astype(np.float32)
        for b, v in ((xd, x), (idd, ids), (wd, w)):
            b.upload(v)
        M.synchronize()
        return x, ids, w

    st = M.Stream()
    fill()
    g = M.Graph(st, lambda s: M.check("expert_ffn", ctx.expert_ffn(lay.L, xd, T, xd, idd, idd, wd, out, s.addr)))
    try:
        for _ in range(4):
            x, ids, w = fill()
            M.check("expert_ffn", ctx.expert_ffn(lay.L, xd, T, xd, idd, idd, wd, eager))
            M.synchronize()
            g.launch(st)
            st.synchronize()
            a, b = out.download(np.float32, (T, D)), eager.download(np.float32, (T, D))
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
            ref = X.ffn(lay.host, x, ids, ids, w)
            assert np.linalg.norm(a - x - ref) <= 1e-3 * np.linalg.norm(ref)
    finally:
        g.destroy()
        st.destroy()


# ------------------------------------------------------------------ sums at the end of float32's range
@gpu
@pytest.mark.parametrize("threshold", [1, 1 << 40])
def test_product_past_the_range(ctx, threshold):
    """sums of positive terms: within the products' tolerance where they stay below 2^126, no numbers above 2^129 (digits
    of both signs past 2^128: infinite or NaN), one row not disturbing the next"""
    rng = np.random.default_rng(99)
    raw = np.abs(X.values(table(rng, 2, 48, 96)))
    raw = O.quantize(O.TYPE_MXFP4, raw.astype(np.float32))
    raw[:, 0::3, 0::17] = 247    # 2^120
    raw[:, 1::3, 0::17] = 254    # 2^127
    b = np.abs(rows(rng, 40, 2, 96)) * np.float32(0.01)
    b[0::2] *= np.float32(1e4)
    ids = rng.integers(0, 2, (40, 2))
    ctx.set_gemm_threshold(threshold)
    try:
        got = run_product(ctx, raw, b, ids)
    finally:
        ctx.set_gemm_threshold(0)
    ref = X.product(raw, b, ids)
    small, large = ref <= 2.0 ** 126, ref >= 2.0 ** 129
    assert small.any() and large.any() and (small & (ref > 2.0 ** 118)).any()
    tol = 2.0 ** -24 * ref + (2.0 ** -50 if threshold > 1 else 2 * 96 / 16 * 2.0 ** -23) * ref
    assert (np.abs(got - ref) <= tol)[small].all()
    assert not np.isfinite(got[large]).any()
