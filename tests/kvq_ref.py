"""The operators of caches in fewer bits (include/orc.h: orc_rope_table,
orc_kvq_store, orc_kvq_load, orc_attn_kvq) from their definitions, in 64 bits."""
import math

import numpy as np

import orc

LEVELS = {orc.KV_Q8: 127, orc.KV_Q4: 7}


def frequencies(rot, base, sc=None):
    """(frequencies, factor of the table's values); sc: (kind, factor, low, high, orig, mscale)"""
    f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    kind, factor, low, high, orig, mscale = sc or (orc.ROPE_PLAIN, 1, 0, 0, 0, 0)
    if kind == orc.ROPE_LINEAR:
        return f / factor, 1.0
    if kind == orc.ROPE_BANDS:
        turns = orig * f / (2 * math.pi)
        mid = (turns - low) / (high - low)
        return np.where(turns > high, f, np.where(turns < low, f / factor, mid * f + (1 - mid) * f / factor)), 1.0
    if kind == orc.ROPE_YARN:
        at = [rot * math.log(orig / (2 * math.pi * t)) / (2 * math.log(base)) for t in (high, low)]
        a, b = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
        slow = np.clip((np.arange(rot // 2) - a) / max(b - a, 0.001), 0, 1)
        return (1 - slow) * f + slow * f / factor, mscale or 0.1 * math.log(factor) + 1
    return f, 1.0


def table(pos0, n, rot, base, sc=None):
    f, m = frequencies(rot, base, sc)
    th = (pos0 + np.arange(n, dtype=np.float64))[:, None] * f[None]
    return np.stack([np.cos(th) * m, np.sin(th) * m], -1)


def rotate(x, cs, layout, rot):
    """x [..., hd] by the pairs cs [..., rot / 2, 2], rounded once to fp32"""
    y = x.astype(np.float64)
    if rot:
        a = slice(0, rot // 2) if layout == orc.ROPE_HALF else slice(0, rot, 2)
        b = slice(rot // 2, rot) if layout == orc.ROPE_HALF else slice(1, rot, 2)
        co, si = cs[..., 0].astype(np.float64), cs[..., 1].astype(np.float64)
        u, v = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
        y[..., a], y[..., b] = u * co - v * si, u * si + v * co
    return y.astype(np.float32)


#: the finite scales up to the largest that a group takes
SCALES = (np.arange(227, dtype=np.uint16) << 7).view(np.float16).astype(np.float64) / 16


def quantised(ty, x):
    """What a cache of type ty holds for the fp32 rows x [..., hd]"""
    if ty == orc.F16:
        with np.errstate(over="ignore"):
            return np.where(np.isfinite(x), np.clip(x, -65504, 65504), x).astype(np.float16).astype(np.float64)
    m = LEVELS[ty]
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(g).all(-1, keepdims=True)
    g = np.clip(np.where(np.isfinite(g), g, 0), -4064, 4064)
    d = SCALES[np.searchsorted(SCALES * m, np.abs(g).max(-1, keepdims=True))]
    y = np.where(d > 0, np.rint(g / np.where(d > 0, d, 1)) * d, 0)
    return np.where(bad, np.nan, y).reshape(x.shape)


def attention(q, pk, pv, k, v, starts, limit):
    """q [S][T][H][hd]; prefix pk, pv [KV][P][hd]; own k, v [S][KV][ctx][hd]. Returns (out, sum of w |v|, largest
    sum of |q k| / sqrt(hd) of each row, sum of |v|) in 64 bits."""
    S, T, H, hd = q.shape
    KV, P = k.shape[1], pk.shape[1]
    G = H // KV
    out, scale, size, total = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3] + (1,)), np.zeros(q.shape)
    live = [s for s in range(S) if 0 <= starts[s] < limit]
    for g in range(KV):
        hs = slice(g * G, (g + 1) * G)
        qg = q[:, :, hs].astype(np.float64) / math.sqrt(hd)
        pkg, pvg = pk[g].astype(np.float64), pv[g].astype(np.float64)
        sp, ap = qg @ pkg.T, (np.abs(qg) @ np.abs(pkg).T).max(-1, initial=0)
        for s in live:
            n = min(T, limit - starts[s])
            end = starts[s] + n
            kk, vv = k[s, g, :end].astype(np.float64), v[s, g, :end].astype(np.float64)
            hide = (np.arange(end)[None] > starts[s] + np.arange(n)[:, None])[:, None]
            sc = np.concatenate([sp[s, :n], np.where(hide, -np.inf, qg[s, :n] @ kk.T)], -1)
            w = np.exp(sc - sc.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[s, :n, hs] = w[..., :P] @ pvg + w[..., P:] @ vv
            scale[s, :n, hs] = w[..., :P] @ np.abs(pvg) + w[..., P:] @ np.abs(vv)
            total[s, :n, hs] = np.abs(pvg).sum(0) + np.where(hide, 0.0, 1.0) @ np.abs(vv)
            size[s, :n, hs, 0] = np.maximum(ap[s, :n], np.where(hide, 0, np.abs(qg[s, :n]) @ np.abs(kk).T).max(-1))
    return out, scale, size, total
