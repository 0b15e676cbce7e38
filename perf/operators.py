"""The MXFP4 operators of the MoE layer library: their plain forms, and the calls that a user makes.

MXFP4 is ggml's type 39: 32 values in 17 bytes, one E8M0 scale byte e and 16 bytes of E2M1 codes (value j in the low
nibble of byte j, value 16 + j in the high one); a value is 2^(e - 127) times one of +-{0, .5, 1, 1.5, 2, 3, 4, 6}.

  requant   mi_quantize to MXFP4, then mi_dequantize: what a row's blocks stand for
  product   mi_mul_mat_id with an MXFP4 expert table: rows in Q8_0 (ggml's vec_dot_type of MXFP4) times the table
  layer     a few tokens through whole MoE layers of MXFP4 tables (mi_moe_forward / _norm / _router_input)

The shapes are the library's: moondream3 (D 2048, 64 experts, top-8, inner 1024, fused [h | g]), qwen3omni (D 2048,
128 experts, top-8, inner 768), diffusiongemma (D 2816, inner 704: 22 blocks a row) and nemotronomni (D 2688, inner
1856, top-6, relu^2, a shared expert of 3712).
"""
import math
import pathlib
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
MXFP4 = 39
MODELS = {
    "moondream3": dict(D=2048, E=64, K=8, I=1024, fused=True, act="gelu_erf_gp1", norm="layer", gating="topk", shared=0),
    "qwen3omni": dict(D=2048, E=128, K=8, I=768, fused=False, act="silu", norm="rms", gating="topk", shared=0),
    "diffusiongemma": dict(D=2816, E=128, K=8, I=704, fused=False, act="gelu_tanh", norm="rms", gating="all", shared=0),
    "nemotronomni": dict(D=2688, E=128, K=6, I=1856, fused=False, act="relu_sqr", norm="rms", gating="sigmoid", shared=3712),
}
EPS, GATE_EPS, SCALING = 1e-6, 1e-20, 2.5


def _requant(name, rows, n):
    return {"name": name, "op": "requant", "rows": rows, "n": n}


def _product(name, model, table, T, zipf=False):
    return {"name": name, "op": "product", "model": model, "table": table, "T": T, "zipf": zipf}


def _layer(name, model, T, call, layers=1):
    return {"name": name, "op": "layer", "model": model, "T": T, "call": call, "layers": layers}


def listed():
    return [
        # a few rows checked against their originals: the call's own cost
        _requant("requant_3x2816", 3, 2816),
        # one small matrix with an odd number of blocks in a row
        _requant("requant_1000x1056", 1000, 1056),
        # a layer's fused gate/up table quantized at load
        _requant("requant_table", 64 * 2048, 2048),
        # one token's gate/up product
        _product("product_1_gate", "moondream3", "gate", 1),
        # a small decode batch's down product, each slot with a row of its own
        _product("product_13_down", "qwen3omni", "down", 13),
        # an image's tokens, rows of 22 blocks
        _product("product_301_down", "diffusiongemma", "down", 301),
        # a prefill with a few hot experts
        _product("product_1024_hot", "qwen3omni", "gate", 1024, zipf=True),
        # a long prefill
        _product("product_2048_gate", "moondream3", "gate", 2048),
        # text generation: one token through the layers of a stack, the norm in front of each
        _layer("layer_1_stack", "qwen3omni", 1, "norm", layers=6),
        # one token on a row that is normalized already, without the residual (the program adds it)
        _layer("layer_1", "moondream3", 1, "forward"),
        # a handful of sequences decoded together, relu^2 experts and the shared one
        _layer("layer_3_shared", "nemotronomni", 3, "norm"),
        # a larger decode batch
        _layer("layer_15", "moondream3", 15, "norm"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["requant", "product", "product", "layer", "layer"])
    if kind == "requant":
        n = 32 * _log_int(rng, 1, 128)
        c = _requant("", _log_int(rng, 1, 64 * 2048 * 2048 // max(n, 1024) // 2), n)
    elif kind == "product":
        model = rng.choice(["moondream3", "qwen3omni", "diffusiongemma", "nemotronomni"])
        c = _product("", model, rng.choice(["gate", "down"]), _log_int(rng, 1, 1500), rng.random() < 0.3)
    else:
        model = rng.choice(["moondream3", "qwen3omni", "qwen3omni", "diffusiongemma", "nemotronomni"])
        call = "router_input" if model == "diffusiongemma" else rng.choice(["forward", "norm"])
        c = _layer("", model, _log_int(rng, 1, 16), call, rng.randint(1, 3))
    del c["name"]
    return c


# ---------------------------------------------------------------- the format
def _steps(like):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=like.device, dtype=like.dtype)


def _pow2(e):
    """2^e in float64, by its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(F64)


def _scale_and_codes(x):
    """x [..., n] float32 -> (E8M0 bytes [..., n/32, 1], magnitude steps 0..7, negative) of its 32-value blocks: the
    scale's exponent is that of the block's largest value less 2, values go to the nearest step, ties to the smaller,
    above 6 to 6; a block that holds an infinity or a NaN is a NaN block (scale byte 255)."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax)[1] + (127 - 1 - 2)
    e = torch.where(amax > 0, e, 0).clamp(0, 254)
    e = torch.where(torch.isfinite(b.sum(-1, keepdim=True) * 0), e, 255)
    r = b.abs().to(F64) * _pow2(127 - e)
    m = sum((r > t).to(torch.uint8) for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
    return e, m, b < 0


def _pack(x):
    """The rows' bytes [..., n/32 * 17]."""
    e, m, neg = _scale_and_codes(x)
    c = m | (neg.to(torch.uint8) << 3)
    return torch.cat([e.to(torch.uint8), c[..., :16] | (c[..., 16:] << 4)], -1).flatten(-2)


def _values(raw, dtype):
    """What rows of bytes stand for."""
    b = raw.unflatten(-1, (-1, 17))
    c = torch.cat([b[..., 1:] & 15, b[..., 1:] >> 4], -1).to(torch.int32)
    v = _steps(torch.empty(0, device=raw.device, dtype=dtype))[c & 7] * (1 - 2 * (c >> 3))
    e = b[..., :1].to(torch.int32) - 127
    return (v * _pow2(e).to(dtype) + torch.where(e == 128, math.nan, 0.0)).flatten(-2)


def _rows8(x):
    """x [..., n] float32 as the product takes it: Q8_0 (per 32 values d = amax / 127 held in 16 bits, codes
    round(x / d) in 8), in the values that it stands for. Quotients in 64 bits, then rounded to 32 as they are defined."""
    b = x.unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1, keepdim=True).to(F64) / 127.0).to(F32)
    inv = torch.where(d > 0, 1.0 / d.to(F64), 0.0).to(F32)
    q = (b * inv).to(F64)
    q = torch.sign(q) * torch.floor(q.abs() + 0.5)
    return (d.to(torch.float16).to(F64) * q).flatten(-2)


# ---------------------------------------------------------------- inputs
def _gen(seed, *salt):
    v = seed
    for s in salt:
        v = (v * 1000003 + s + 1) % (1 << 62)
    return torch.Generator(device="cuda").manual_seed(v)


def _normal(shape, seed, *salt, std=1.0):
    return torch.randn(shape, generator=_gen(seed, *salt), device="cuda") * std


def _table(E, N, n, seed, *salt):
    """An expert table [E][N rows of n values], its bytes."""
    step = max(1, (1 << 26) // (N * n))
    return torch.cat([_pack(_normal((min(step, E - e), N, n), seed, *salt, e, std=0.02)) for e in range(0, E, step)])


def _rows(T, n, seed, *salt):
    """Rows of a residual stream: channels of different sizes, a few of them large."""
    size = torch.exp(0.4 * _normal((n,), seed, *salt, 1))
    size[torch.randperm(n, generator=_gen(seed, *salt, 2), device="cuda")[:4]] *= 8.0
    return _normal((T, n), seed, *salt, 3) * size


def _shape(case):
    """(values of a row, rows of a matrix, whether each slot has a row of its own) of a product's table."""
    m = MODELS[case["model"]]
    return (m["D"], m["I"] * (2 if m["fused"] else 1), False) if case["table"] == "gate" else (m["I"], m["D"], True)


def _inputs(case, seed):
    """What prepare() and exact() both start from."""
    if case["op"] == "requant":
        rows, n = case["rows"], case["n"]
        return {"x": _normal((rows, n), seed, 1) * torch.exp(_normal((rows, 1), seed, 2)) * 0.02}
    m, T = MODELS[case["model"]], case["T"]
    D, E, K, I = m["D"], m["E"], m["K"], m["I"]
    if case["op"] == "product":
        n, N, own_rows = _shape(case)
        score = torch.rand((T, E), generator=_gen(seed, 4), device="cuda")
        if case["zipf"]:
            rank = torch.randperm(E, generator=_gen(seed, 5), device="cuda") + 1
            score = -torch.log(score.clamp_min(1e-30)) * rank ** 1.2
        ids = score.argsort(-1)[:, :K].to(torch.int32).contiguous()
        return {"b": _rows(T * K if own_rows else T, n, seed, 6).reshape(T, -1, n), "ids": ids, "w": _table(E, N, n, seed, 7)}
    got = []
    for i in range(case["layers"]):
        h = _rows(T, D, seed, i, 10)
        t = {"h": h, "router_w": _normal((E, D), seed, i, 11, std=0.02), "gate": _table(E, I * (2 if m["fused"] else 1), D, seed, i, 12),
             "down": _table(E, D, I, seed, i, 13), "norm_w": 1.0 + 0.1 * _normal((D,), seed, i, 14)}
        t["x"] = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)) * t["norm_w"]
        if not m["fused"] and m["act"] != "relu_sqr":
            t["up"] = _table(E, I, D, seed, i, 15)
        if m["norm"] == "layer":
            t["norm_b"] = 0.05 * _normal((D,), seed, i, 16)
        if case["call"] == "router_input":
            t["x_router"] = _normal((T, D), seed, i, 17)
        if m["gating"] == "sigmoid":
            t["sel_bias"] = _normal((E,), seed, i, 18, std=0.05)
        if m["gating"] == "all":
            t["expert_scale"] = 0.5 + torch.rand((E,), generator=_gen(seed, i, 19), device="cuda")
        if m["shared"]:
            t["sh_gate"] = _table(1, m["shared"], D, seed, i, 20)
            t["sh_down"] = _table(1, D, m["shared"], seed, i, 21)
        got.append(t)
    return {"layers": got}


# ---------------------------------------------------------------- the calls
def _library():
    at = str(pathlib.Path.cwd() / "skyvision.cpp_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mimoe
    return mimoe


def _describe(state):
    """The handle and the descriptors that a user's program keeps."""
    M, case = _library(), state["case"]
    ctx = M.Context(0)
    state["ctx"] = ctx
    if case["op"] == "requant":
        state["rows"] = torch.empty(case["rows"] * case["n"] // 32 * 17, dtype=torch.uint8, device="cuda")
        state["out"] = torch.empty_like(state["x"])
        return
    m, T = MODELS[case["model"]], case["T"]
    D, E, K, I = m["D"], m["E"], m["K"], m["I"]
    ctx.reserve(T, D, I, E, K)
    if case["op"] == "product":
        n, N, _ = _shape(case)
        state["out"] = torch.empty((T, K, N), device="cuda")
        state["desc"] = (M.tensor(state["w"].data_ptr(), MXFP4, [n, N, E]), M.tensor(state["b"].data_ptr(), M.TYPE_F32, [n, state["b"].shape[1], T]),
                         M.tensor(state["ids"].data_ptr(), M.TYPE_I32, [K, T]), M.tensor(state["out"].data_ptr(), M.TYPE_F32, [N, K, T]))
        return
    acts = {"silu": M.ACT_SILU, "gelu_erf_gp1": M.ACT_GELU_ERF_GP1, "gelu_tanh": M.ACT_GELU_TANH, "relu_sqr": M.ACT_RELU_SQR}
    for t in state["layers"]:
        layer = M.make_layer(D, E, K, I, t["router_w"].data_ptr(), None,
                             M.tensor(t["gate"].data_ptr(), MXFP4, [D, I * (2 if m["fused"] else 1), E]),
                             M.tensor(t["up"].data_ptr(), MXFP4, [D, I, E]) if "up" in t else None,
                             M.tensor(t["down"].data_ptr(), MXFP4, [I, D, E]), m["fused"], acts[m["act"]])
        layer.gating = {"topk": M.GATING_SOFTMAX_TOPK, "sigmoid": M.GATING_SIGMOID_BIAS, "all": M.GATING_SOFTMAX_ALL}[m["gating"]]
        if "sel_bias" in t:
            layer.sel_bias, layer.routed_scaling, layer.gate_eps = t["sel_bias"].data_ptr(), SCALING, GATE_EPS
        if "expert_scale" in t:
            layer.expert_scale = t["expert_scale"].data_ptr()
        if m["shared"]:
            layer.sh_n_ff, layer.sh_act = m["shared"], acts[m["act"]]
            layer.sh_gate = M.tensor(t["sh_gate"].data_ptr(), MXFP4, [D, m["shared"]])
            layer.sh_down = M.tensor(t["sh_down"].data_ptr(), MXFP4, [m["shared"], D])
        t["layer"], t["out"] = layer, torch.empty((T, D), device="cuda")
        t["norm"] = M.make_norm(M.NORM_LAYER if m["norm"] == "layer" else M.NORM_RMS, EPS, t["norm_w"].data_ptr(),
                                t["norm_b"].data_ptr() if "norm_b" in t else None)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        _describe(state)
    if case["op"] == "product":
        # the rows that the fullest expert has: a padded batch's size
        state["most"] = int(torch.bincount(state["ids"].flatten().long()).max())
    torch.cuda.synchronize()
    return state


def run(state):
    case = state["case"]
    if own:
        return _call(state)
    if case["op"] == "requant":
        e, m, neg = _scale_and_codes(state["x"])
        v = _steps(state["x"])[m.long()] * torch.where(neg, -1.0, 1.0) * _pow2(e - 127).to(F32)
        return (v + torch.where(e == 255, math.nan, 0.0)).flatten(-2)
    if case["op"] == "product":
        x = _rows8(state["b"]).to(F32).expand(-1, state["ids"].shape[1], -1)
        return _expert_product(state["w"], x, state["ids"], state["most"], F32)
    return [_plain_layer(MODELS[case["model"]], case["call"], t) for t in state["layers"]]


def _call(state):
    case, ctx = state["case"], state["ctx"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "requant":
        rows, n = case["rows"], case["n"]
        rc = ctx.quantize(MXFP4, state["x"].data_ptr(), state["rows"].data_ptr(), rows, n, stream)
        rc = rc or ctx.dequantize(MXFP4, state["rows"].data_ptr(), state["out"].data_ptr(), rows, n, stream)
    elif case["op"] == "product":
        rc = ctx.mul_mat_id(*state["desc"], stream)
    else:
        for t in state["layers"]:
            rc = _call_layer(ctx, case, t, stream)
            if rc:
                break
    if rc:
        raise RuntimeError("%s: status %d" % (case["op"], rc))
    return [t["out"] for t in state["layers"]] if case["op"] == "layer" else state["out"]


def _call_layer(ctx, case, t, stream):
    T, h, out = case["T"], t["h"].data_ptr(), t["out"].data_ptr()
    if case["call"] == "norm":
        return ctx.forward_norm(t["layer"], t["norm"], h, T, h, out, None, stream)
    if case["call"] == "forward":
        return ctx.forward(t["layer"], t["x"].data_ptr(), T, None, out, None, stream)
    return ctx.forward_router_input(t["layer"], t["x"].data_ptr(), t["x_router"].data_ptr(), T, h, out, None, stream)


# ---------------------------------------------------------------- plain forms
def _expert_product(raw, x, ids, most, dtype):
    """y[t, k] = table[ids[t, k]] @ x[t, k] (x [T, K, n], table rows raw [E, N, bytes])."""
    T, K = ids.shape
    E, rows, flat = raw.shape[0], T * K, ids.flatten().long()
    if rows <= E:      # a matrix for each slot
        return (_values(raw[flat], dtype) @ x.reshape(rows, -1, 1).to(dtype)).reshape(T, K, -1)
    # the slots of each expert as a batch, padded to the fullest expert's
    order = torch.argsort(flat, stable=True)
    first = torch.searchsorted(flat[order], torch.arange(E, device=ids.device))
    place = torch.arange(rows, device=ids.device) - first[flat[order]]
    batch = torch.zeros((E, most, x.shape[-1]), device=ids.device, dtype=dtype)
    batch[flat[order], place] = x.reshape(rows, -1)[order].to(dtype)
    y = torch.bmm(_values(raw, dtype), batch.transpose(1, 2).contiguous())       # [E, N, most]
    out = torch.empty((rows, y.shape[1]), device=ids.device, dtype=dtype)
    out[order] = y[flat[order], :, place]
    return out.reshape(T, K, -1)


def _glu(act, a, b):
    if act == "relu_sqr":
        return torch.relu(a) ** 2
    if act == "silu":
        return a / (1.0 + torch.exp(-a)) * b
    if act == "gelu_tanh":
        return 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * a * (1.0 + 0.044715 * a * a))) * b
    return 0.5 * a * (1.0 + torch.erf(a * math.sqrt(0.5))) * (b + 1.0)


def _norm(m, t):
    """The row norm: sums in 64 bits (each later value's code depends on them), everything else in 32."""
    h = t["h"]
    if m["norm"] == "rms":
        d = h
    else:
        d = h - h.to(F64).mean(-1, keepdim=True).to(F32)
    var = (d * d).to(F64).mean(-1, keepdim=True).to(F32) + EPS
    y = d * (1.0 / torch.sqrt(var.to(F64)).to(F32).to(F64)).to(F32) * t["norm_w"]
    return y + t["norm_b"] if "norm_b" in t else y


def _route(m, t, x):
    logits = (x.to(F64) @ t["router_w"].to(F64).T).to(F32)
    K = m["K"]
    if m["gating"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-logits))
        ids = torch.sort(s + t["sel_bias"], dim=-1, descending=True, stable=True)[1][:, :K]
        w = s.gather(1, ids)
        return ids, w / (w.sum(-1, keepdim=True) + GATE_EPS) * SCALING
    ids = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :K]
    top = logits.gather(1, ids)
    w = torch.exp(top - top[:, :1])
    w = w / w.sum(-1, keepdim=True)
    return ids, w * t["expert_scale"][ids] if "expert_scale" in t else w


def _plain_layer(m, call, t):
    """The layer. The values between the two products are rounded to 8-bit codes, so they are computed in 64 bits:
    one that is off in its last bits next to a border between two codes would move the code."""
    x = _norm(m, t) if call == "norm" else t["x"]
    ids, w = _route(m, t, t["x_router"] if call == "router_input" else x)
    T, K = ids.shape

    def ffn(gate, up, down, i):
        a = _expert_product(gate, _rows8(x)[:, None, :].expand(-1, i.shape[1], -1), i, T, F64)
        if m["fused"]:
            a, b = a.chunk(2, -1)
        else:
            b = None if up is None else _expert_product(up, _rows8(x)[:, None, :].expand(-1, i.shape[1], -1), i, T, F64)
        return _expert_product(down, _rows8(_glu(m["act"], a, b).to(F32)), i, T, F64)

    y = (ffn(t["gate"], t.get("up"), t["down"], ids).to(F32) * w[..., None]).to(F64).sum(1)
    if m["shared"]:
        y = y + ffn(t["sh_gate"], None, t["sh_down"], torch.zeros((T, 1), device=ids.device, dtype=ids.dtype))[:, 0]
    return y.to(F32) if call == "forward" else t["h"] + y.to(F32)


# ---------------------------------------------------------------- what it takes
def work(case):
    if case["op"] == "requant":
        n = case["rows"] * case["n"]
        return {"bytes": 2.0 * n * (4 + 17 / 32), "flops": 2.0 * n}
    m, T = MODELS[case["model"]], case["T"]
    D, E, K, I = m["D"], m["E"], m["K"], m["I"]
    hit = E * (1.0 - (1.0 - K / E) ** T)             # experts that some token chose, evenly spread
    if case["op"] == "product":
        n, N, own_rows = _shape(case)
        if case["zipf"]:                              # the same with the ranks' weights
            p = [r ** -1.2 for r in range(1, E + 1)]
            hit = sum(1.0 - (1.0 - min(1.0, K * q / sum(p))) ** T for q in p)
        return {"bytes": hit * N * n / 32 * 17 + 4.0 * T * ((K if own_rows else 1) * n + K * N + K), "flops": 2.0 * T * K * N * n}
    products = 1 if m["act"] == "relu_sqr" else 2
    b = hit * (products + 1) * D * I / 32 * 17 + 4.0 * E * D + 4.0 * T * D * {"norm": 2, "forward": 2, "router_input": 4}[case["call"]]
    f = 2.0 * T * K * (products + 1) * D * I + 2.0 * T * E * D
    b += 2.0 * D * m["shared"] / 32 * 17
    f += 4.0 * T * D * m["shared"]
    return {"bytes": case["layers"] * b, "flops": case["layers"] * f}


# ---------------------------------------------------------------- in 64 bits, from the definitions
_ALL = [s * v for s in (1.0, -1.0) for v in (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)]


def _exact_block_values(raw):
    """Rows of bytes in float64, each code looked up in the table of all sixteen."""
    n = raw.shape[-1] // 17
    out = torch.empty((*raw.shape[:-1], n, 32), device=raw.device, dtype=F64)
    table = torch.tensor(_ALL, device=raw.device, dtype=F64)
    blocks = raw.reshape(*raw.shape[:-1], n, 17).long()
    scale = torch.tensor([2.0 ** k for k in range(-127, 129)], device=raw.device, dtype=F64)[blocks[..., 0]][..., None]
    out[..., :16] = table[blocks[..., 1:] % 16] * scale
    out[..., 16:] = table[blocks[..., 1:].div(16, rounding_mode="floor")] * scale
    return out.reshape(*raw.shape[:-1], n * 32)


def _exact_rows8(x):
    """Q8_0 of float32 rows, by its definition: 32-bit quotients, a 16-bit scale, 8-bit codes."""
    n = x.shape[-1]
    v = x.reshape(-1, 32).to(F64)
    d = (v.abs().max(1, keepdim=True).values / 127).to(F32).to(F64)
    inv = torch.where(d == 0, torch.zeros_like(d), 1 / d).to(F32).to(F64)
    p = (v * inv).to(F32).to(F64)
    code = torch.where(p < 0, torch.ceil(p - 0.5), torch.floor(p + 0.5))
    return (code * d.to(torch.float16).to(F64)).reshape(*x.shape[:-1], n)


def _exact_product(raw, x, ids):
    out = torch.zeros((*ids.shape, raw.shape[1]), device=raw.device, dtype=F64)
    for e in torch.unique(ids).tolist():
        at = ids == e
        out[at] = x[at] @ _exact_block_values(raw[e]).T
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "requant":
        # the nearest of the values that the block's scale allows, the smaller of two
        def rows(x):
            v = x.reshape(-1, 32).to(F64)
            top = v.abs().max(1, keepdim=True).values
            e = torch.where(top > 0, torch.floor(torch.log2(top.clamp_min(1e-300))) - 2, torch.full_like(top, -127.0)).clamp(-127, 127)
            e = torch.tensor([2.0 ** k for k in range(-127, 128)], device=x.device, dtype=F64)[e.long() + 127]
            steps = torch.tensor(_ALL[:8], device=x.device, dtype=F64)
            r = v.abs() / e
            best = (r[..., None] - steps).abs().argmin(-1)
            return (torch.sign(v) * steps[best] * e).reshape(x.shape)
        return torch.cat([rows(x) for x in s["x"].split(max(1, (1 << 23) // case["n"]))])
    if case["op"] == "product":
        K = s["ids"].shape[1]
        x = _exact_rows8(s["b"])
        return _exact_product(s["w"], x.expand(-1, K, -1), s["ids"])
    m = MODELS[case["model"]]
    K, outs = m["K"], []
    for t in s["layers"]:
        x, h64 = t["x"], t["h"].to(F64)
        if case["call"] == "norm":      # float32 steps with sums in float64, as the norm is defined
            c = t["h"] if m["norm"] == "rms" else t["h"] - (h64.sum(-1, keepdim=True) / m["D"]).to(F32)
            ms = ((c * c).to(F64).sum(-1, keepdim=True) / m["D"]).to(F32) + EPS
            root = torch.sqrt(ms.to(F64)).to(F32)
            x = (c * (1 / root.to(F64)).to(F32)) * t["norm_w"]
            x = x + t["norm_b"] if "norm_b" in t else x
        logits = t.get("x_router", x).to(F64) @ t["router_w"].to(F64).T
        if m["gating"] == "sigmoid":
            p = torch.sigmoid(logits)
            ids = (p + t["sel_bias"].to(F64)).topk(K).indices
            w = p.gather(1, ids)
            w = w / (w.sum(-1, keepdim=True) + GATE_EPS) * SCALING
        else:
            ids = logits.topk(K).indices
            w = torch.softmax(logits.gather(1, ids), -1)
            if "expert_scale" in t:
                w = w * t["expert_scale"].to(F64)[ids]
        xq = _exact_rows8(x)[:, None, :]

        def ffn(gate, up, down, i):
            a = _exact_product(gate, xq.expand(-1, i.shape[1], -1), i)
            if m["act"] == "relu_sqr":
                v = a.clamp_min(0) ** 2
            else:
                a, b = (a[..., :m["I"]], a[..., m["I"]:]) if m["fused"] else (a, _exact_product(up, xq.expand(-1, i.shape[1], -1), i))
                if m["act"] == "silu":
                    v = a * torch.sigmoid(a) * b
                elif m["act"] == "gelu_tanh":
                    v = 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))) * b
                else:
                    v = 0.5 * a * (1 + torch.erf(a / math.sqrt(2))) * (b + 1)
            return _exact_product(down, _exact_rows8(v.to(F32)), i)

        y = (ffn(t["gate"], t.get("up"), t["down"], ids) * w[..., None]).sum(1)
        if m["shared"]:
            y = y + ffn(t["sh_gate"], None, t["sh_down"], torch.zeros_like(ids[:, :1]))[:, 0]
        outs.append(y if case["call"] == "forward" else h64 + y)
    return outs
