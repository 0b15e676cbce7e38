"""Plain float64 forms of the MXFP4 operators, from the format's definition."""
from __future__ import annotations

import math

import numpy as np

STEPS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x: np.ndarray) -> np.ndarray:
    """float32 [..., n] -> bytes [..., n / 32 * 17]: every code by trying all steps, the first of the nearest."""
    b = np.asarray(x, np.float32).reshape(-1, 32)
    out = np.zeros((len(b), 17), np.uint8)
    for i, row in enumerate(b):
        if not np.isfinite(row).all():
            out[i, 0] = 255
            continue
        amax = float(np.abs(row).max())
        e = max(0, math.frexp(amax)[1] - 3 + 127) if amax > 0 else 0
        r = np.abs(row.astype(np.float64)) * 2.0 ** (127 - e)
        c = np.abs(r[:, None] - STEPS).argmin(1)
        c = np.where((row < 0) & (c > 0), c | 8, c).astype(np.uint8)
        out[i, 0] = e
        out[i, 1:] = c[:16] | (c[16:] << 4)
    return out.reshape(*np.shape(x)[:-1], -1)


def values(raw: np.ndarray) -> np.ndarray:
    """bytes [..., n / 32 * 17] -> float64 [..., n]"""
    b = np.asarray(raw, np.uint8).reshape(-1, 17)
    c = np.concatenate([b[:, 1:] & 15, b[:, 1:] >> 4], 1)
    v = STEPS[c & 7] * np.where(c & 8, -1.0, 1.0) * 2.0 ** (b[:, :1].astype(np.float64) - 127)
    v[b[:, 0] == 255] = np.nan
    return v.reshape(*np.shape(raw)[:-1], -1)


def q8_0(x: np.ndarray) -> np.ndarray:
    """float32 [..., n] -> the float64 values of its Q8_0 (32-bit quotients, fp16 scale, codes rounded half away)."""
    with np.errstate(all="ignore"):
        b = np.ascontiguousarray(x, np.float32).reshape(-1, 32)
        d = (np.abs(b).max(1, keepdims=True) / np.float32(127)).astype(np.float32)
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        p = (b * inv).astype(np.float64)
        q = np.copysign(np.floor(np.abs(p) + 0.5), p)
        v = d.astype(np.float16).astype(np.float64) * q
        v[~np.isfinite(d.astype(np.float16)[:, 0])] = np.nan
    return v.reshape(np.shape(x))


def product(raw: np.ndarray, b: np.ndarray, ids: np.ndarray, size: bool = False) -> np.ndarray:
    """table bytes [E, N, row], b float32 [T, 1 | K, n], ids [T, K] -> float64 [T, K, N] (rows of ids outside: 0);
    size: the sums of the terms' sizes instead"""
    T, K = ids.shape
    x = np.broadcast_to(q8_0(b), (T, K, b.shape[-1]))
    x = np.abs(x) if size else x
    out = np.zeros((T, K, raw.shape[1]))
    with np.errstate(all="ignore"):
        for e in np.unique(ids):
            if 0 <= e < raw.shape[0]:
                at, w = ids == e, values(raw[e])
                out[at] = x[at] @ (np.abs(w) if size else w).T
    return out


def product_sizes(raw, b, ids):
    return product(raw, b, ids, True)


_erf = np.vectorize(math.erf)


def act(kind: int, a, b):
    """mi_act in float64"""
    if kind == 4:
        return np.where(a > 0, a, np.where(np.isnan(a), a, 0.0)) ** 2
    if kind == 0:
        return a / (1 + np.exp(-a)) * b
    if kind == 2:
        return 0.5 * a * (1 + np.tanh(math.sqrt(2 / math.pi) * a * (1 + 0.044715 * a * a))) * b
    return 0.5 * a * (1 + _erf(a / math.sqrt(2))) * (b + 1 if kind == 1 else b)


def ffn_slots(L: dict, x, ids_gu, ids_dn) -> np.ndarray:
    """the slots' outputs: L has gate, up (or None), down bytes, fused, act, I; x float32 [T, D]; float64 [T, K, D]"""
    I = L["I"]
    with np.errstate(all="ignore"):
        a = product(L["gate"], x[:, None, :], ids_gu)
        b = None
        if L["act"] != 4:
            a, b = (a[..., :I], a[..., I:]) if L["fused"] else (a, product(L["up"], x[:, None, :], ids_gu))
        v = act(L["act"], a, b).astype(np.float32)
        return product(L["down"], v, ids_dn)


def ffn(L: dict, x, ids_gu, ids_dn, w) -> np.ndarray:
    """the routed sum, float64 [T, D]"""
    y = ffn_slots(L, x, ids_gu, ids_dn)
    live = (ids_gu >= 0) & (ids_gu < len(L["gate"])) & (ids_dn >= 0) & (ids_dn < len(L["down"]))
    return np.where(live[..., None], y * w[..., None].astype(np.float64), 0.0).sum(1)
