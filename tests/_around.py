"""Plain forms of the operators around the experts (grouped routing, residual norm, dense products of 4-bit matrices),
from their definitions: routing scores, norm steps and codes as they are defined in 32 bits, everything else in 64."""
from __future__ import annotations

import numpy as np

import pyoracle as O

F32, F64 = np.float32, np.float64


# ------------------------------------------------------------------ routing
def scores(logits, sigmoid: bool):
    """float32 [T, E]: each evaluated in 64 bits and rounded"""
    l = np.asarray(logits, F32)
    with np.errstate(all="ignore"):
        if sigmoid:
            return (1.0 / (1.0 + np.exp(-l.astype(F64)))).astype(F32)
        top = np.fmax.reduce(l, axis=1, keepdims=True)
        e = np.exp((l - top).astype(F32).astype(F64)).astype(F32)
        return e * (1.0 / e.astype(F64).sum(1, keepdims=True)).astype(F32)


def route(logits, K, sigmoid, groups=1, kept=1, top=1, renorm=True, eps=0.0, scaling=1.0, bias=None, scale=None):
    """(ids int32 [T, K], weights float64 [T, K]), one token and one slot after another"""
    s = scores(logits, sigmoid)
    T, E = s.shape
    with np.errstate(all="ignore"):
        c = s if bias is None else s + np.asarray(bias, F32)
    gs = E // groups
    ids, w = np.zeros((T, K), np.int32), np.zeros((T, K))
    for t in range(T):
        ok = np.ones(E, bool)
        if 1 < groups and kept < groups:
            vals = []
            for g in range(groups):
                v = sorted((x for x in c[t, g * gs:(g + 1) * gs] if not np.isnan(x)), reverse=True)
                vals.append(np.nan if not v else v[0] if top == 1 else F32(v[0] + v[1]) if len(v) > 1 else -np.inf)
            order = sorted(range(groups), key=lambda g: (np.isnan(vals[g]), -vals[g] if not np.isnan(vals[g]) else 0, g))
            ok[:] = False
            for g in order[:kept]:
                ok[g * gs:(g + 1) * gs] = True
        live = [e for e in range(E) if ok[e] and not np.isnan(c[t, e])]
        chosen = sorted(live, key=lambda e: (-c[t, e], e))[:K]
        sw = [float(s[t, e]) for e in chosen]
        while len(chosen) < K:
            chosen.append(next(e for e in range(E) if e not in chosen))
            sw.append(np.nan)
        sw = np.array(sw, F64)
        with np.errstate(all="ignore"):
            if renorm:
                sw = sw / (sw.sum() + F64(F32(eps)))
            sw = sw * F64(F32(scaling))
            if scale is not None:
                sw = sw * np.asarray(scale, F32).astype(F64)[chosen]
        ids[t], w[t] = chosen, sw
    return ids, w


# ------------------------------------------------------------------ norm
def add_norm(x, add, layer: bool, eps, w=None, b=None):
    """(h, y) float32: sums in 64 bits, each other step rounded to 32"""
    h = np.asarray(x, F32) if add is None else np.asarray(x, F32) + np.asarray(add, F32)
    D = h.shape[1]
    with np.errstate(all="ignore"):
        d = h - (h.astype(F64).sum(1, keepdims=True) / D).astype(F32) if layer else h
        var = ((d * d).astype(F64).sum(1, keepdims=True) / D).astype(F32)
        y = d * (F32(1) / np.sqrt(var + F32(eps)))
        if w is not None:
            y = y * np.asarray(w, F32)
        if layer and b is not None:
            y = y + np.asarray(b, F32)
    return h, y


def q8_bytes(y, type_):
    """rows of y in Q8_0 or Q8_K: ggml's quantizer, NaN blocks (scale NaN, codes 0) where a value is not finite"""
    T, D = y.shape
    size, bytes_ = (32, 34) if type_ == O.TYPE_Q8_0 else (256, 292)
    bad = ~np.isfinite(y.reshape(T, -1, size)).all(2)
    raw = O.quantize(type_, np.where(np.isfinite(y), y, 0).astype(F32)).reshape(T, -1, bytes_).copy()
    raw[bad] = 0
    raw[bad, :2 if size == 32 else 4] = np.frombuffer(F32(np.nan).tobytes() if size == 256 else b"\x00\x7e", np.uint8)
    return raw.reshape(T, -1)


# ------------------------------------------------------------------ products
def values8(raw, type_, n):
    """float64 [T, n] of rows in Q8_0 / Q8_K; blocks whose scale is not finite are NaN"""
    T = raw.shape[0]
    if type_ == O.TYPE_Q8_0:
        blk = np.ascontiguousarray(raw).reshape(T, -1, 34)
        d = np.ascontiguousarray(blk[..., :2]).view(np.float16).astype(F64)
        q = blk[..., 2:].view(np.int8).astype(F64)
    else:
        blk = np.ascontiguousarray(raw).reshape(T, -1, 292)
        d = np.ascontiguousarray(blk[..., :4]).view(F32).astype(F64)
        q = blk[..., 4:260].view(np.int8).astype(F64)
    d = np.where(np.isfinite(d), d, np.nan)
    return (d * q).reshape(T, n)


def matrix_parts(raw, type_, n):
    """(values, minima) float64 [N, n]: a value is values - minima"""
    N = raw.shape[0]
    if type_ == O.TYPE_Q4_0:
        blk = np.ascontiguousarray(raw).reshape(N, -1, 18)
        d = np.ascontiguousarray(blk[..., :2]).view(np.float16).astype(F64)
        q = np.concatenate([blk[..., 2:] & 15, blk[..., 2:] >> 4], -1).astype(F64) - 8
        return (d * q).reshape(N, n), np.zeros((N, n))
    blk = np.ascontiguousarray(raw).reshape(N, -1, 144)
    d = np.ascontiguousarray(blk[..., :2]).view(np.float16).astype(F64)
    dm = np.ascontiguousarray(blk[..., 2:4]).view(np.float16).astype(F64)
    s = blk[..., 4:16].astype(np.int64)
    sc = np.concatenate([s[..., :4] & 63, (s[..., 8:] & 15) | ((s[..., :4] >> 6) << 4)], -1)
    mn = np.concatenate([s[..., 4:8] & 63, (s[..., 8:] >> 4) | ((s[..., 4:8] >> 6) << 4)], -1)
    c = blk[..., 16:].reshape(N, -1, 4, 32)
    q = np.stack([c & 15, c >> 4], -2).reshape(N, -1, 8, 32).astype(F64)
    return (((d * sc)[..., None]) * q).reshape(N, n), np.repeat(dm * mn, 32, -1).reshape(N, n)


def mul_mat(raw, type_, rows8, n):
    """(products float64 [T, N], the bound of a float32 sum over the blocks' exact parts): every block's part is
    rounded at most three times (its scale, the product, the sum; a part of the minima likewise) and enters at most
    blocks + 4 additions, each off by at most 2^-24 of the sizes added so far."""
    x = values8(rows8, O.TYPE_Q8_0 if type_ == O.TYPE_Q4_0 else O.TYPE_Q8_K, n)
    v, m = matrix_parts(raw, type_, n)
    blocks = n // (32 if type_ == O.TYPE_Q4_0 else 256)
    with np.errstate(all="ignore"):
        size = np.abs(x) @ (np.abs(v) + np.abs(m)).T
        return x @ (v - m).T, size * (2 * blocks + 8) * 2.0 ** -24
