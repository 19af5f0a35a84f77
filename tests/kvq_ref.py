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
    KV = k.shape[1]
    out, scale, size, total = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3] + (1,)), np.zeros(q.shape)
    q = q.astype(np.float64)
    for s in range(S):
        for t in range(T):
            p = starts[s] + t
            if starts[s] < 0 or starts[s] >= limit or p >= limit:
                continue
            for g in range(KV):
                kk = np.concatenate([pk[g], k[s, g, :p + 1]]).astype(np.float64)
                vv = np.concatenate([pv[g], v[s, g, :p + 1]]).astype(np.float64)
                hs = slice(g * H // KV, (g + 1) * H // KV)
                sc = q[s, t, hs] @ kk.T / math.sqrt(hd)
                w = np.exp(sc - sc.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[s, t, hs], scale[s, t, hs] = w @ vv, w @ np.abs(vv)
                total[s, t, hs] = np.abs(vv).sum(0)
                size[s, t, hs, 0] = (np.abs(q[s, t, hs]) @ np.abs(kk).T).max(-1) / math.sqrt(hd)
    return out, scale, size, total
