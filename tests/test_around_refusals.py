"""What the operators around the experts refuse (mi_moe_route, mi_moe_forward_router, mi_add_norm, mi_mul_mat): every
check comes before the first device call, so a zeroed stand-in for a context (nothing reserved) is enough."""
import ctypes as C

import pytest

import mimoe as M

NULL, SHAPE, TYPE, CAPACITY, UNSUPPORTED, ARG = M.ERR_NULL, M.ERR_SHAPE, M.ERR_TYPE, M.ERR_CAPACITY, M.ERR_UNSUPPORTED, M.ERR_ARG
A = 1 << 20     # addresses that no call reads


@pytest.fixture(scope="module")
def ctx():
    class Standin(M.Context):
        def __init__(self):
            self.block = C.create_string_buffer(1 << 16)
            self.h = C.c_void_p(C.addressof(self.block))

        def close(self):
            pass

    return Standin()


def f32(ne, nb=None, at=A):
    return M.tensor(at, M.TYPE_F32, ne, nb)


def test_route(ctx):
    def rc(r, logits=None, sel=A * 4, w=A * 8):
        return ctx.route(r, logits if logits is not None else f32([r.n_expert, 5]), sel, w)

    ok = dict(E=64, K=4, score=M.SCORE_SIGMOID, n_group=8, n_group_used=2, group_top=2)
    R = lambda **k: M.make_router(**{**ok, **k})
    assert M.load().mi_moe_route(None, C.byref(R()), C.byref(f32([64, 5])), A, A, None) == NULL
    assert M.load().mi_moe_route(ctx.h, None, C.byref(f32([64, 5])), A, A, None) == NULL
    assert rc(R(), sel=None) == NULL and rc(R(), w=None) == NULL and rc(R(), f32([64, 5], at=0)) == NULL
    for bad in (dict(E=0), dict(E=-1), dict(K=0), dict(K=65, E=64), dict(K=17), dict(n_group=-1), dict(n_group=7),
                dict(n_group_used=0), dict(n_group_used=9), dict(E=8, n_group=8, K=2)):
        assert rc(R(**bad)) == SHAPE, bad
    for bad in (dict(score=2), dict(score=-1), dict(group_top=0), dict(group_top=3)):
        assert rc(R(**bad)) == ARG, bad
    for bad in (dict(E=1032), dict(E=512, K=65, n_group=1), dict(E=260, n_group=65, n_group_used=60)):
        assert rc(R(**bad)) == UNSUPPORTED, bad
    assert rc(R(), M.tensor(A, M.TYPE_F16, [64, 5])) == TYPE
    assert rc(R(), f32([63, 5])) == SHAPE and rc(R(), f32([64, -1])) == SHAPE and rc(R(), f32([64, 5, 2])) == SHAPE
    assert rc(R(), f32([64, 5], [4, 252, 0, 0])) == SHAPE and rc(R(), f32([64, 5], [8, 256, 0, 0])) == SHAPE
    assert rc(R(), f32([64, 5], [4, 258, 0, 0])) == UNSUPPORTED and rc(R(), f32([64, 5], at=A + 2)) == UNSUPPORTED
    assert rc(R(), sel=A) == ARG and rc(R(), w=A + 4 * 64 * 5 - 4) == ARG and rc(R(), sel=A * 8 + 4) == ARG
    assert rc(R(), f32([64, 0])) == M.OK


def test_forward_router(ctx):
    t = M.tensor(A, M.TYPE_Q4_K, [256, 256, 64])
    L = M.make_layer(256, 64, 4, 256, A, None, t, t, t, False, M.ACT_SILU)
    r = M.make_router(64, 4, M.SCORE_SOFTMAX)

    def rc(layer=L, router=r, norm=None, x=A, T=1, out=A * 2):
        return ctx.forward_router(layer, router, norm, x, None, T, None, out)

    assert M.load().mi_moe_forward_router(ctx.h, C.byref(L), None, None, A, None, 1, None, A, None, None) == NULL
    assert M.load().mi_moe_forward_router(ctx.h, None, C.byref(r), None, A, None, 1, None, A, None, None) == NULL
    assert rc(router=M.make_router(63, 4, M.SCORE_SOFTMAX)) == SHAPE and rc(router=M.make_router(64, 3, M.SCORE_SOFTMAX)) == SHAPE
    assert rc(router=M.make_router(64, 4, 5)) == ARG
    assert rc(norm=M.make_norm(3, 1e-6)) == ARG
    assert rc(T=-1) == SHAPE
    assert rc() == CAPACITY      # nothing reserved


def test_add_norm(ctx):
    n = M.make_norm(M.NORM_RMS, 1e-6)
    x, add, s, y = (f32([256, 3], at=A * k) for k in (1, 2, 3, 4))
    q = M.tensor(A * 5, M.TYPE_Q8_0, [256, 3])

    def rc(x=x, add=add, s=s, y=y, q=q, n=n):
        return ctx.add_norm(n, x, add, s, y, q)

    lib = M.load()
    assert lib.mi_add_norm(None, C.byref(n), C.byref(x), None, None, C.byref(y), None, None) == NULL
    assert lib.mi_add_norm(ctx.h, None, C.byref(x), None, None, C.byref(y), None, None) == NULL
    assert lib.mi_add_norm(ctx.h, C.byref(n), None, None, None, C.byref(y), None, None) == NULL
    assert rc(y=None, q=None) == NULL
    for k in ("x", "add", "s", "y"):
        assert rc(**{k: f32([256, 3], at=0)}) == NULL
        assert rc(**{k: M.tensor(A * 7, M.TYPE_F16, [256, 3])}) == TYPE
        assert rc(**{k: f32([256, 3], [4, 1026, 0, 0], A * 7)}) == UNSUPPORTED
        assert rc(**{k: f32([256, 3], [4, 1020, 0, 0], A * 7)}) == SHAPE
        if k != "x":
            assert rc(**{k: f32([255, 3], at=A * 7)}) == SHAPE and rc(**{k: f32([256, 2], at=A * 7)}) == SHAPE
    assert rc(n=M.make_norm(M.NORM_NONE, 0)) == ARG and rc(n=M.make_norm(9, 0)) == ARG
    assert rc(q=M.tensor(A * 7, M.TYPE_Q4_0, [256, 3])) == TYPE and rc(q=M.tensor(0, M.TYPE_Q8_0, [256, 3])) == NULL
    assert rc(q=M.tensor(A * 7 + 1, M.TYPE_Q8_0, [256, 3])) == UNSUPPORTED
    assert rc(q=M.tensor(A * 7 + 2, M.TYPE_Q8_K, [256, 3])) == UNSUPPORTED
    assert rc(q=M.tensor(A * 7, M.TYPE_Q8_K, [256, 3], [292, 294, 0, 0])) == UNSUPPORTED
    wide = [f32([48, 3], at=A * k) for k in (1, 2, 3, 4)]
    assert ctx.add_norm(n, *wide, M.tensor(A * 7, M.TYPE_Q8_0, [48, 3], [34, 68, 0, 0])) == SHAPE   # 48 values: no whole blocks
    # overlaps: an output on another, q on an input, an output on part of an input
    assert rc(y=s) == ARG and rc(q=M.tensor(A * 4, M.TYPE_Q8_0, [256, 3])) == ARG
    assert rc(q=M.tensor(A, M.TYPE_Q8_0, [256, 3])) == ARG
    assert rc(s=f32([256, 3], at=A + 1024)) == ARG and rc(y=f32([256, 3], [4, 2048, 0, 0], A)) == ARG
    big = [f32([16388, 1], at=A * k) for k in (1, 2, 3, 4)]
    assert ctx.add_norm(n, *big) == UNSUPPORTED
    assert ctx.add_norm(n, *(f32([256, 0], at=A * k) for k in (1, 2, 3, 4))) == M.OK


def test_mul_mat(ctx):
    a, b, d = M.tensor(A, M.TYPE_Q4_0, [256, 64]), M.tensor(A * 2, M.TYPE_Q8_0, [256, 3]), f32([64, 3], at=A * 3)

    def rc(a=a, b=b, d=d):
        return ctx.mul_mat(a, b, d)

    lib = M.load()
    for k in range(4):
        args = [ctx.h, C.byref(a), C.byref(b), C.byref(d)]
        args[k] = None
        assert lib.mi_mul_mat(*args, None) == NULL
    assert rc(M.tensor(0, M.TYPE_Q4_0, [256, 64])) == NULL and rc(d=f32([64, 3], at=0)) == NULL
    for t in (M.TYPE_Q5_0, M.TYPE_Q8_0, M.TYPE_Q6_K, M.TYPE_MXFP4):
        assert rc(M.tensor(A, t, [256, 64])) == TYPE
    assert rc(b=M.tensor(A * 2, M.TYPE_Q8_K, [256, 3])) == TYPE and rc(b=M.tensor(A * 2, M.TYPE_F16, [256, 3])) == TYPE
    assert rc(d=M.tensor(A * 3, M.TYPE_F16, [64, 3])) == TYPE
    assert ctx.mul_mat(M.tensor(A, M.TYPE_Q4_K, [256, 64]), b, d) == TYPE
    assert rc(M.tensor(A, M.TYPE_Q4_0, [256, 64, 2])) == SHAPE and rc(b=M.tensor(A * 2, M.TYPE_Q8_0, [288, 3])) == SHAPE
    assert rc(d=f32([63, 3], at=A * 3)) == SHAPE and rc(d=f32([64, 2], at=A * 3)) == SHAPE
    assert rc(M.tensor(A, M.TYPE_Q4_0, [256, 64], [18, 142, 0, 0])) == SHAPE
    assert rc(d=f32([64, 3], [4, 252, 0, 0], A * 3)) == SHAPE and rc(d=f32([64, 3], [4, 258, 0, 0], A * 3)) == UNSUPPORTED
    assert rc(M.tensor(A + 1, M.TYPE_Q4_0, [256, 64])) == UNSUPPORTED
    assert rc(b=M.tensor(A * 2 + 1, M.TYPE_Q8_0, [256, 3])) == UNSUPPORTED
    k8 = M.tensor(A * 2, M.TYPE_Q8_K, [256, 3])
    assert ctx.mul_mat(M.tensor(A + 8, M.TYPE_Q4_K, [256, 64]), k8, d) == UNSUPPORTED
    assert ctx.mul_mat(M.tensor(A, M.TYPE_Q4_K, [256, 64], [144, 152, 0, 0]), k8, d) == UNSUPPORTED
    assert rc(M.tensor(A, M.TYPE_Q4_0, [100, 64], [18, 72, 0, 0])) == SHAPE
    assert rc(b=f32([256, 3], at=A * 2)) == CAPACITY             # nothing reserved
    assert rc(d=f32([64, 3], at=A * 2)) == ARG and rc(d=f32([64, 3], at=A + 144 * 64 - 4)) == ARG
    assert rc(b=M.tensor(A * 2, M.TYPE_Q8_0, [256, 0]), d=f32([64, 0], at=A * 3)) == M.OK


def test_row_size():
    assert M.row_size(M.TYPE_Q8_K, 512) == 584 and M.row_size(M.TYPE_Q8_K, 300) == 0


def test_outputs_on_parameters(ctx):
    r = M.make_router(64, 4, M.SCORE_SIGMOID, sel_bias=A * 20, expert_scale=A * 30)
    lg = f32([64, 5])
    for at in (A * 20, A * 30):
        assert ctx.route(r, lg, at + 252, A * 8) == ARG and ctx.route(r, lg, A * 8, at - 76) == ARG
    n = M.make_norm(M.NORM_LAYER, 1e-6, weight=A * 20, bias=A * 30)
    x = f32([256, 3])
    for at in (A * 20, A * 30):
        on = f32([256, 3], at=at + 1020)
        assert ctx.add_norm(n, x, None, on, f32([256, 3], at=A * 4)) == ARG
        assert ctx.add_norm(n, x, None, None, on) == ARG
        assert ctx.add_norm(n, x, None, None, None, M.tensor(at, M.TYPE_Q8_0, [256, 3])) == ARG
