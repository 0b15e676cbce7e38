"""The operators around the routed experts: their plain forms, and the calls that a user makes.

  route    mi_moe_route: router logits to expert ids and weights, with softmax or sigmoid scores, a selection bias,
           groups of experts of which the best are kept, top-k, renormalized and scaled weights
  norm     mi_add_norm: h + r, its RMSNorm or LayerNorm, as float32 rows or in 8 bits with scales (ggml's Q8_0: 32
           values with a 16-bit scale; Q8_K: 256 values with a 32-bit scale)
  product  mi_mul_mat: a matrix in 4 bits with group scales (ggml's Q4_0, Q4_K) times a few rows, which go to the
           matrix type's 8-bit form first (Q8_0 for Q4_0, Q8_K for Q4_K)
  chain    mi_add_norm to 8 bits and mi_mul_mat on those rows: the input side of a dense block

The widths are the library's: rows of 2048 (moondream3, qwen3omni), 2816 (diffusiongemma) and 2688 (nemotronomni, with a
shared expert of 3712); 128 experts of which 8 (qwen3omni), and 256, the most that a layer takes.
"""
import math
import pathlib
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
Q4_0, Q8_0, Q4_K, Q8_K = 2, 8, 12, 15
EIGHT = {"q4_0": Q8_0, "q4_K": Q8_K}           # the 8-bit form that a matrix type's products take
EPS, GATE_EPS = 1e-6, 1e-20


def _route(name, T, E, K, score, groups=1, kept=1, top=1, bias=False, renorm=True, scaling=1.0, expert_scale=False):
    return {"name": name, "op": "route", "T": T, "E": E, "K": K, "score": score, "groups": groups, "kept": kept, "top": top,
            "bias": bias, "renorm": renorm, "scaling": scaling, "expert_scale": expert_scale}


def _norm(name, T, D, kind, out):
    return {"name": name, "op": "norm", "T": T, "D": D, "kind": kind, "out": out}


def _product(name, T, N, n, type_):
    return {"name": name, "op": "product", "T": T, "N": N, "n": n, "type": type_}


def _chain(name, T, N, n, type_, kind):
    return {"name": name, "op": "chain", "T": T, "N": N, "n": n, "type": type_, "kind": kind}


def listed():
    return [
        # text generation: one token, balanced by a bias, the best half of eight groups
        _route("route_1", 1, 256, 8, "sigmoid", 8, 4, 2, bias=True, scaling=2.5),
        # a few dozen sequences decoded together, groups by their best expert
        _route("route_29", 29, 128, 8, "softmax", 4, 2, 1, renorm=False, scaling=1.5, expert_scale=True),
        # a long prompt
        _route("route_8192", 8192, 256, 8, "sigmoid", 8, 4, 2, bias=True, scaling=2.5),
        # one token between attention and the router
        _norm("norm_1", 1, 2048, "rms", "f32"),
        # a decode batch whose rows feed 4-bit matrices
        _norm("norm_13_q8_0", 13, 2816, "rms", "q8_0"),
        # a prompt's rows for 4-bit matrices of 256-value blocks
        _norm("norm_4096_q8_K", 4096, 2048, "layer", "q8_K"),
        # one token through an attention block's output matrix
        _product("product_1", 1, 2048, 2048, "q4_0"),
        # one token's logits: the largest matrix of a model
        _product("product_1_head", 1, 65536, 2048, "q4_K"),
        # a decode batch through a shared expert's first matrix, rows of 84 blocks
        _product("product_13", 13, 3712, 2688, "q4_0"),
        # an image's or a prompt's tokens through a dense layer's first matrix
        _product("product_200", 200, 8192, 2048, "q4_K"),
        # one token into a dense layer: residual, norm, 8 bits, first matrix
        _chain("chain_1", 1, 8192, 2048, "q4_K", "layer"),
        # a small decode batch into a shared expert
        _chain("chain_6", 6, 3712, 2688, "q4_0", "rms"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["route", "norm", "product", "product", "chain"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 3, 4, 8])
        E = groups * rng.randint(max(2, 16 // groups), 256 // groups)
        kept = rng.randint(1, groups)
        K = rng.randint(1, min(12, kept * (E // groups)))
        c = _route("", _log_int(rng, 1, 8192), E, K, rng.choice(["softmax", "sigmoid"]), groups, kept, rng.choice([1, 2]),
                   rng.random() < 0.6, rng.random() < 0.7, rng.choice([1.0, 2.5]), rng.random() < 0.3)
    elif kind == "norm":
        out = rng.choice(["f32", "q8_0", "q8_K"])
        step = {"f32": 1, "q8_0": 32, "q8_K": 256}[out]
        D = step * _log_int(rng, max(1, 256 // step), 8192 // step)
        c = _norm("", _log_int(rng, 1, 4096 * 2048 // max(D, 2048)), D, rng.choice(["rms", "layer"]), out)
    else:
        type_ = rng.choice(["q4_0", "q4_K"])
        step = 32 if type_ == "q4_0" else 256
        n = step * _log_int(rng, max(1, 128 // step), 8192 // step)
        T = _log_int(rng, 1, 200) if kind == "product" else _log_int(rng, 1, 24)
        N = _log_int(rng, 16, min(65536, (65536 if T <= 8 else 8192) * 2048 // n))
        c = _product("", T, N, n, type_) if kind == "product" else _chain("", T, N, n, type_, rng.choice(["rms", "layer"]))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _gen(seed, *salt):
    v = seed
    for s in salt:
        v = (v * 1000003 + s + 1) % (1 << 62)
    return torch.Generator(device="cuda").manual_seed(v)


def _normal(shape, seed, *salt, std=1.0):
    return torch.randn(shape, generator=_gen(seed, *salt), device="cuda") * std


def _rows(T, n, seed, *salt):
    """Rows of a residual stream: channels of different sizes, a few of them large."""
    size = torch.exp(0.4 * _normal((n,), seed, *salt, 1))
    size[torch.randperm(n, generator=_gen(seed, *salt, 2), device="cuda")[:4]] *= 8.0
    return _normal((T, n), seed, *salt, 3) * size


def _bytes(h):
    """The two bytes of 16-bit values [..., 1], lowest first."""
    return h.to(torch.float16).view(torch.int16).view(torch.uint8)


def _pack_q4_0(x):
    """x [N, n] to rows of 18-byte blocks: d f16, 16 bytes of codes (value j low nibble of byte j, 16 + j high)."""
    b = x.unflatten(-1, (-1, 32))
    top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = top / -8.0
    q = torch.where(d != 0, b / d, 0.0).add_(8.5).floor_().clamp_(0, 15).to(torch.uint8)
    return torch.cat([_bytes(d), q[..., :16] | (q[..., 16:] << 4)], -1).flatten(-2)


def _pack_q4_K(x):
    """x [N, n] to rows of 144-byte blocks of 256: d f16, dmin f16, eight 6-bit scales and minima in 12 bytes, 128 bytes
    of codes; value = d * scale * code - dmin * minimum."""
    b = x.unflatten(-1, (-1, 8, 32))
    low = (-b.amin(-1)).clamp_min(0.0)
    step = ((b.amax(-1) + low) / 15.0).clamp_min(1e-12)
    d, dm = step.amax(-1, keepdim=True) / 63.0, low.amax(-1, keepdim=True) / 63.0
    sc = (step / d).round().clamp(1, 63).to(torch.uint8)
    mn = torch.where(dm > 0, low / dm, 0.0).round().clamp(0, 63).to(torch.uint8)
    q = ((b + (dm * mn)[..., None]) / (d * sc)[..., None]).round_().clamp_(0, 15).to(torch.uint8)
    lo = torch.cat([sc[..., :4] | ((sc[..., 4:] >> 4) << 6), mn[..., :4] | ((mn[..., 4:] >> 4) << 6)], -1)
    hi = (sc[..., 4:] & 15) | ((mn[..., 4:] & 15) << 4)
    codes = (q[..., 0::2, :] | (q[..., 1::2, :] << 4)).flatten(-2)
    return torch.cat([_bytes(d), _bytes(dm), lo, hi, codes], -1).flatten(-2)


def _matrix(type_, N, n, seed, *salt):
    """A matrix's bytes [N, row], made a part at a time."""
    step = max(1, (1 << 25) // n)
    pack = _pack_q4_0 if type_ == "q4_0" else _pack_q4_K
    return torch.cat([pack(_normal((min(step, N - r), n), seed, *salt, r, std=0.02)) for r in range(0, N, step)])


def _inputs(case, seed):
    """What prepare() and exact() both start from."""
    T = case["T"]
    if case["op"] == "route":
        E = case["E"]
        # a trained router's logits: experts of different popularity, tokens that prefer a few
        s = {"logits": 1.5 * _normal((T, E), seed, 1) + 0.7 * _normal((E,), seed, 2)}
        if case["bias"]:
            s["bias"] = -0.1 * torch.sigmoid(_normal((E,), seed, 3))
        if case["expert_scale"]:
            s["scale"] = 0.5 + torch.rand((E,), generator=_gen(seed, 4), device="cuda")
        return s
    n = case["D"] if case["op"] == "norm" else case["n"]
    s = {"x": _rows(T, n, seed, 5)}
    if case["op"] != "product":
        s["add"] = 0.3 * _rows(T, n, seed, 6)
        s["w"] = 1.0 + 0.1 * _normal((n,), seed, 7)
        if case["kind"] == "layer":
            s["b"] = 0.05 * _normal((n,), seed, 8)
    if case["op"] != "norm":
        s["matrix"] = _matrix(case["type"], case["N"], n, seed, 9)
    return s


# ---------------------------------------------------------------- the calls
def _library():
    at = str(pathlib.Path.cwd() / "skyvision.cpp_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mimoe
    return mimoe


def _describe(state):
    """The handle, the buffers and the descriptors that a user's program keeps."""
    M, case = _library(), state["case"]
    state["ctx"] = ctx = M.Context(0)
    T = case["T"]

    def f32(t):
        return M.tensor(t.data_ptr(), M.TYPE_F32, [t.shape[1], t.shape[0]])

    if case["op"] == "route":
        state["sel"] = torch.empty((T, case["K"]), dtype=torch.int32, device="cuda")
        state["weights"] = torch.empty((T, case["K"]), device="cuda")
        state["router"] = M.make_router(case["E"], case["K"], M.SCORE_SIGMOID if case["score"] == "sigmoid" else M.SCORE_SOFTMAX,
                                        n_group=case["groups"], n_group_used=case["kept"], group_top=case["top"],
                                        renorm=case["renorm"], eps=GATE_EPS, scaling=case["scaling"],
                                        sel_bias=state["bias"].data_ptr() if "bias" in state else None,
                                        expert_scale=state["scale"].data_ptr() if "scale" in state else None)
        state["logits_desc"] = f32(state["logits"])
        return
    n = state["x"].shape[1]
    if case["op"] != "norm":
        N = case["N"]
        ctx.reserve(T, n, 1, 1, 1)
        state["out"] = torch.empty((T, N), device="cuda")
        state["a"] = M.tensor(state["matrix"].data_ptr(), Q4_0 if case["type"] == "q4_0" else Q4_K, [n, N])
        state["dst"] = f32(state["out"])
    if case["op"] == "product":
        state["rows"] = f32(state["x"])
        return
    state["sum"] = torch.empty_like(state["x"])
    state["norm"] = M.make_norm(M.NORM_LAYER if case["kind"] == "layer" else M.NORM_RMS, EPS, state["w"].data_ptr(),
                                state["b"].data_ptr() if "b" in state else None)
    state["x_desc"], state["add_desc"], state["sum_desc"] = f32(state["x"]), f32(state["add"]), f32(state["sum"])
    type_ = EIGHT[case["type"]] if case["op"] == "chain" else {"f32": None, "q8_0": Q8_0, "q8_K": Q8_K}[case["out"]]
    if case["op"] == "norm":
        state["y"] = torch.empty_like(state["x"])
    if type_ is None:
        state["y_desc"] = f32(state["y"])
    else:
        state["codes"] = torch.empty(T * M.row_size(type_, n), dtype=torch.uint8, device="cuda")
        state["rows"] = M.tensor(state["codes"].data_ptr(), type_, [n, T])


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        _describe(state)
    torch.cuda.synchronize()
    return state


def _check(rc, what):
    if rc:
        raise RuntimeError("%s: status %d" % (what, rc))


def _call(state):
    case, ctx = state["case"], state["ctx"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "route":
        _check(ctx.route(state["router"], state["logits_desc"], state["sel"].data_ptr(), state["weights"].data_ptr(), stream), "route")
        return [state["sel"], state["weights"]]
    if case["op"] != "product":
        _check(ctx.add_norm(state["norm"], state["x_desc"], state["add_desc"], state["sum_desc"], state.get("y_desc"),
                            state.get("rows"), stream), "add_norm")
    if case["op"] == "norm":
        if "rows" in state:      # the values that the codes stand for
            _check(ctx.dequantize(state["rows"].type, state["codes"].data_ptr(), state["y"].data_ptr(), case["T"], case["D"], stream),
                   "dequantize")
        return [state["sum"], state["y"]]
    _check(ctx.mul_mat(state["a"], state["rows"], state["dst"], stream), "mul_mat")
    return state["out"] if case["op"] == "product" else [state["sum"], state["out"]]


def run(state):
    if own:
        return _call(state)
    case = state["case"]
    if case["op"] == "route":
        return _plain_route(case, state)
    if case["op"] == "product":
        return _rows8(state["x"], EIGHT[case["type"]]) @ _values(state["matrix"], case["type"]).T
    total, y = _plain_norm(case, state)
    if case["op"] == "norm":
        return [total, y if case["out"] == "f32" else _rows8(y, Q8_0 if case["out"] == "q8_0" else Q8_K)]
    return [total, _rows8(y, EIGHT[case["type"]]) @ _values(state["matrix"], case["type"]).T]


# ---------------------------------------------------------------- plain forms
def _scores(case, logits):
    """The experts' scores: numbers of 32 bits, each computed in 64 and rounded (a router ranks them, and two that round
    to the same number tie)."""
    if case["score"] == "sigmoid":
        return (1.0 / (1.0 + torch.exp(-logits.to(F64)))).to(F32)
    e = torch.exp((logits - logits.amax(-1, keepdim=True)).to(F64)).to(F32)
    return e * (1.0 / e.to(F64).sum(-1, keepdim=True)).to(F32)


def _plain_route(case, state):
    T, E, K, G = case["T"], case["E"], case["K"], case["groups"]
    s = _scores(case, state["logits"])
    choice = s + state["bias"] if "bias" in state else s
    if G > 1:
        group = choice.reshape(T, G, E // G)
        best = torch.sort(group, dim=-1, descending=True)[0][..., :case["top"]].sum(-1)
        keep = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :case["kept"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=s.device).scatter_(1, keep, True)
        choice = torch.where(kept[..., None], group, -math.inf).reshape(T, E)
    ids = torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :K]
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / (w.to(F64).sum(-1, keepdim=True).to(F32) + GATE_EPS)
    w = w * case["scaling"]
    if "scale" in state:
        w = w * state["scale"][ids]
    return [ids.to(torch.int32), w]


def _plain_norm(case, state):
    """The sum and its norm: the row's sums in 64 bits (every value's code depends on them), everything else in 32."""
    h = state["x"] + state["add"]
    d = h if case["kind"] == "rms" else h - h.to(F64).mean(-1, keepdim=True).to(F32)
    var = (d * d).to(F64).mean(-1, keepdim=True).to(F32) + EPS
    y = d * (1.0 / torch.sqrt(var.to(F64)).to(F32).to(F64)).to(F32) * state["w"]
    return h, y + state["b"] if "b" in state else y


def _rows8(x, type_):
    """x [T, n] in 8 bits, as the values that it stands for. Q8_0: 32 values, d = amax / 127 held in 16 bits, codes
    round(x / d), halves away from zero; Q8_K: 256 values, d in 32 bits, halves to even."""
    if type_ == Q8_0:
        b = x.unflatten(-1, (-1, 32))
        d = (b.abs().amax(-1, keepdim=True).to(F64) / 127.0).to(F32)
        inv = torch.where(d > 0, 1.0 / d.to(F64), 0.0).to(F32)
        q = (b * inv).to(F64)
        q = torch.sign(q) * torch.floor(q.abs() + 0.5)
        return (d.to(torch.float16).to(F64) * q).to(F32).flatten(-2)
    b = x.unflatten(-1, (-1, 256))
    amax = b.abs().amax(-1, keepdim=True)
    inv = torch.where(amax > 0, 127.0 / amax.to(F64), 0.0).to(F32)
    d = torch.where(amax > 0, 1.0 / inv.to(F64), 0.0).to(F32)
    return (d * torch.round(b * inv)).flatten(-2)


def _values(raw, type_):
    """The values of a matrix's rows."""
    if type_ == "q4_0":
        b = raw.unflatten(-1, (-1, 18))
        d = b[..., :2].contiguous().view(torch.float16).to(F32)
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).to(F32) - 8.0
        return (d * q).flatten(-2)
    b = raw.unflatten(-1, (-1, 144))
    d = b[..., :2].contiguous().view(torch.float16).to(F32)[..., None]
    dm = b[..., 2:4].contiguous().view(torch.float16).to(F32)[..., None]
    lo, hi = b[..., 4:12], b[..., 12:16]
    sc = torch.cat([lo[..., :4] & 63, (hi & 15) | ((lo[..., :4] >> 6) << 4)], -1).to(F32)[..., None]
    mn = torch.cat([lo[..., 4:] & 63, (hi >> 4) | ((lo[..., 4:] >> 6) << 4)], -1).to(F32)[..., None]
    c = b[..., 16:].unflatten(-1, (4, 32))
    q = torch.stack([c & 15, c >> 4], -2).flatten(-3, -2).to(F32)
    return (d * sc * q - dm * mn).flatten(-3)


# ---------------------------------------------------------------- what it takes
_ROW = {"q4_0": 18 / 32, "q4_K": 144 / 256, "q8_0": 34 / 32, "q8_K": 292 / 256, "f32": 4.0}


def work(case):
    T = case["T"]
    if case["op"] == "route":
        E, K = case["E"], case["K"]
        return {"bytes": 4.0 * T * E + 8.0 * T * K + 4.0 * E * (case["bias"] + case["expert_scale"]), "flops": 20.0 * T * E}
    if case["op"] == "norm":
        n = T * case["D"]
        # the codes are written and read once more where their values are returned
        out = 4.0 if case["out"] == "f32" else 2 * _ROW[case["out"]] + 4.0
        return {"bytes": n * (12.0 + out) + 4.0 * case["D"] * (2 if case["kind"] == "layer" else 1), "flops": 8.0 * n}
    N, n = case["N"], case["n"]
    b = N * n * _ROW[case["type"]] + 4.0 * T * N + 4.0 * T * n
    f = 2.0 * T * N * n
    if case["op"] == "chain":
        b += T * n * 8.0 + 4.0 * n * (2 if case["kind"] == "layer" else 1)
        f += 8.0 * T * n
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _exact_route(case, s):
    """Expert by expert: its place among the choices that are left, from how many come before it."""
    T, E, K, G = case["T"], case["E"], case["K"], case["groups"]
    logits = s["logits"].to(F64)
    score = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, -1)
    # what is ranked are numbers of 32 bits, by the definition
    choice = score.to(F32)
    if case["score"] == "softmax":
        top = s["logits"].max(-1, keepdim=True).values
        e = torch.exp((s["logits"] - top).to(F64)).to(F32)
        choice = (e.to(F64) * (1 / e.to(F64).sum(-1, keepdim=True)).to(F32).to(F64)).to(F32)
    if "bias" in s:
        choice = (choice.to(F64) + s["bias"].to(F64)).to(F32)
    if G > 1:
        g = choice.reshape(T, G, -1).to(F64)
        value = g.topk(case["top"], -1).values.sum(-1).to(F32)
        before = (value[:, None, :] > value[:, :, None]) | (
            (value[:, None, :] == value[:, :, None]) & (torch.arange(G, device=value.device)[None, :] < torch.arange(G, device=value.device)[:, None]))
        gone = before.sum(-1) >= case["kept"]
        choice = choice.masked_fill(gone.repeat_interleave(E // G, 1), -math.inf)
    ids = torch.empty((T, K), dtype=torch.int64, device=choice.device)
    at = torch.arange(E, device=choice.device)
    for t in range(0, T, 512):
        c = choice[t:t + 512]
        before = ((c[:, None, :] > c[:, :, None]) | ((c[:, None, :] == c[:, :, None]) & (at[None, :] < at[:, None]))).sum(-1)
        ids[t:t + 512] = before.argsort(-1)[:, :K]
    w = score.gather(1, ids)
    if case["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + GATE_EPS)
    w = w * case["scaling"]
    if "scale" in s:
        w = w * s["scale"].to(F64)[ids]
    return [ids.to(torch.int32), w]


def _exact_rows8(x, type_):
    """The 8-bit forms by their definitions (32-bit quotients, codes, the scale as it is held)."""
    n = x.shape[-1]
    size = 32 if type_ == Q8_0 else 256
    v = x.reshape(-1, size).to(F64)
    top = v.abs().max(1, keepdim=True).values
    if type_ == Q8_0:
        d = (top / 127).to(F32).to(F64)
        inv = torch.where(d == 0, torch.zeros_like(d), 1 / d).to(F32).to(F64)
        p = (v * inv).to(F32).to(F64)
        code = torch.where(p < 0, torch.ceil(p - 0.5), torch.floor(p + 0.5))
        return (code * d.to(torch.float16).to(F64)).reshape(-1, n)
    inv = torch.where(top == 0, torch.zeros_like(top), 127 / top).to(F32).to(F64)
    d = torch.where(inv == 0, torch.zeros_like(inv), 1 / inv).to(F32).to(F64)
    p = (v * inv).to(F32).to(F64)
    low = torch.floor(p)
    up = (p - low > 0.5) | ((p - low == 0.5) & (torch.remainder(low, 2) == 1))
    return ((low + up.to(F64)) * d).reshape(-1, n)


def _exact_matrix(raw, type_):
    if type_ == "q4_0":
        b = raw.reshape(raw.shape[0], -1, 18)
        out = torch.empty((*b.shape[:2], 32), dtype=F64, device=raw.device)
        codes = b[..., 2:].to(torch.int64)
        out[..., :16] = (codes % 16 - 8).to(F64)
        out[..., 16:] = (codes.div(16, rounding_mode="floor") - 8).to(F64)
        return (out * b[..., :2].contiguous().view(torch.float16).to(F64)).reshape(raw.shape[0], -1)
    b = raw.reshape(raw.shape[0], -1, 144)
    d = b[..., 0:2].contiguous().view(torch.float16).to(F64)[..., 0]
    dm = b[..., 2:4].contiguous().view(torch.float16).to(F64)[..., 0]
    p = b.to(torch.int64)
    out = torch.empty((*b.shape[:2], 256), dtype=F64, device=raw.device)
    for j in range(8):
        if j < 4:
            scale, low = p[..., 4 + j] % 64, p[..., 8 + j] % 64
        else:
            scale = p[..., 8 + j] % 16 + 16 * (p[..., j].div(64, rounding_mode="floor"))
            low = p[..., 8 + j].div(16, rounding_mode="floor") + 16 * (p[..., 4 + j].div(64, rounding_mode="floor"))
        codes = p[..., 16 + 32 * (j // 2):48 + 32 * (j // 2)]
        codes = codes % 16 if j % 2 == 0 else codes.div(16, rounding_mode="floor")
        out[..., 32 * j:32 * j + 32] = (d * scale)[..., None] * codes - (dm * low)[..., None]
    return out.reshape(raw.shape[0], -1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "route":
        return _exact_route(case, s)

    def product(rows):
        step = max(1, (1 << 25) // case["n"])
        return torch.cat([rows @ _exact_matrix(m, case["type"]).T for m in s["matrix"].split(step)], -1)

    if case["op"] == "product":
        return product(_exact_rows8(s["x"], EIGHT[case["type"]]))
    h = s["x"].to(F64) + s["add"].to(F64)
    if case["op"] == "norm" and case["out"] == "f32":
        c = h if case["kind"] == "rms" else h - h.mean(-1, keepdim=True)
        y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS) * s["w"].to(F64)
        return [h, y + s["b"].to(F64) if "b" in s else y]
    # rows that go to codes: 32-bit steps with sums in 64 bits, as the norm is defined
    r = h.to(F32)
    n = r.shape[-1]
    c = r if case["kind"] == "rms" else r - (r.to(F64).sum(-1, keepdim=True) / n).to(F32)
    ms = ((c * c).to(F64).sum(-1, keepdim=True) / n).to(F32) + EPS
    y = (c * (1 / torch.sqrt(ms.to(F64)).to(F32).to(F64)).to(F32)) * s["w"]
    y = y + s["b"] if "b" in s else y
    if case["op"] == "norm":
        return [h, _exact_rows8(y, Q8_0 if case["out"] == "q8_0" else Q8_K)]
    return [h, product(_exact_rows8(y, EIGHT[case["type"]]))]
