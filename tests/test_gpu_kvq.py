"""Caches in fewer bits: the rotary table, the quantising write, the read-back
and the attention (csrc/orc_kvq.hip, csrc/orc_attn_kvq.hip) against their
definitions in 64 bits.

Bounds, set before the first run:
* the table is rounded once: half a step of fp32 (2^-24 of the value) and what 64-bit sines leave at the far angles
  (2^-53 of an angle below 2^25: 4e-9);
* rotated q rows, codes and values read back are exact: rotations are sums of two exact products, rounded once, and
  the scales and codes are defined without a rounding of their own;
* attention, relative to sum w |v| of the row: the scores' error in natural units is at most 2^-22 (split q) and 8
  roundings of the matrix cores at 2^-23 each of S = max over keys of sum |q k| / sqrt(hd), 1.2e-6 S, which moves weights
  and their sum (2.4e-6 S); apart from that the exponent's rounding (2^-24 of an argument below 16, times ln 2: 6.6e-7),
  the exponential (1.2e-7), the weights' split (2.4e-7), 4 roundings of 2^-23 per block (4.8e-7), and one of 2^-24 for
  each of up to 24 additions of blocks and partial sums, in the weighted and in the plain sum (2.9e-6): 4.4e-6. Held:
  5e-6 + 2.5e-6 S; and 2^-39 of sum |v|: a weight carries 2^15 and its lower half ends at fp16's last place, 2^-24, so
  next to the largest weight, 1, each weight is off by up to 2^-39 however small it is itself.
"""
import ctypes as C

import numpy as np
import pytest

import kvq_ref as ref
import orc

pytestmark = pytest.mark.gpu

TYPES = [orc.F16, orc.KV_Q8, orc.KV_Q4]
SCALINGS = [None, (orc.ROPE_LINEAR, 4.0, 0.0, 0.0, 0, 0.0), (orc.ROPE_BANDS, 8.0, 1.0, 4.0, 8192, 0.0),
            (orc.ROPE_YARN, 4.0, 1.0, 32.0, 32768, 0.0), (orc.ROPE_YARN, 16.0, 2.0, 16.0, 4096, 1.25)]


def _table(dev, pos0, n, rot, base, sc=None):
    out = dev.alloc(max(1, n * rot * 4))
    c = C.byref(orc.RopeScaling(*sc)) if sc else None
    dev.check(dev.L.orc_rope_table(out.ptr, pos0, n, rot, base, c, None))
    return out


@pytest.mark.parametrize("sc", SCALINGS)
@pytest.mark.parametrize("pos0,n,rot,base", [(0, 1, 2, 1e4), (0, 300, 64, 5e5), (131000, 77, 128, 1e6),
                                             (8191, 65, 58, 1e4), (3, 4097, 6, 1e6)])
def test_rope_table(dev, sc, pos0, n, rot, base):
    print(f"[gpu] rope table {pos0} {n} {rot} {sc}", flush=True)
    got = _table(dev, pos0, n, rot, base, sc).read(np.float32).reshape(n, rot // 2, 2)
    want = ref.table(pos0, n, rot, base, sc)
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 4e-9)


def test_rope_table_of_no_positions(dev):
    dev.check(dev.L.orc_rope_table(None, 5, 0, 64, 1e4, None, None))


class Caches:
    """K and V caches of one kind, every byte 0xFF at first (NaN in each type)."""

    def __init__(self, dev, ty, seqs, kv, ctx, hd):
        self.dev, self.ty, self.shape = dev, ty, (seqs, kv, hd, ctx)
        self.bytes = dev.L.orc_kvq_bytes(ty, seqs, kv, ctx, hd)
        assert self.bytes == seqs * kv * ctx * {orc.F16: 2 * hd, orc.KV_Q8: hd + hd // 32, orc.KV_Q4: hd // 2 + hd // 32}[ty]
        self.k, self.v = dev.alloc(self.bytes), dev.alloc(self.bytes)
        for c in (self.k, self.v):
            dev.check(dev.L.orc_fill(c.ptr, 0xFF, self.bytes, None))

    def load(self, n, pos=None, off=0):
        seqs, kv, hd, ctx = self.shape
        out = [self.dev.alloc(4 * seqs * kv * n * hd) for _ in range(2)]
        d = self.dev.upload(np.asarray(pos, np.int32)) if pos is not None else None
        self.dev.check(self.dev.L.orc_kvq_load(self.ty, self.k.ptr, self.v.ptr, seqs, kv, hd, ctx, d and d.ptr, off, n,
                                               out[0].ptr, out[1].ptr, None))
        self.dev.sync()
        return [o.read(np.float32).reshape(seqs, kv, n, hd) for o in out]

    def store(self, qkv, n_tok, heads, rope=None, rot=0, layout=orc.ROPE_HALF, pos=None, off=0, rope_off=0, stream=None,
              in_place=False):
        """qkv [seqs * n_tok][ld]; returns the rotated q rows [.. ][heads * hd + 4] (4 floats of padding)"""
        seqs, kv, hd, ctx = self.shape
        x = self.dev.upload(qkv)
        ldq = qkv.shape[1] if in_place else heads * hd + 4
        q = x if in_place else self.dev.upload(np.full((seqs * n_tok, ldq), 7.5, np.float32))
        d = self.dev.upload(np.asarray(pos, np.int32)) if pos is not None else None
        self.dev.sync()
        self.dev.check(self.dev.L.orc_kvq_store(self.ty, x.ptr, qkv.shape[1], seqs, n_tok, heads, kv, hd, layout, rot,
                                                rope and rope.ptr, rope_off, d and d.ptr, off, q.ptr, ldq, self.k.ptr,
                                                self.v.ptr, ctx, stream))
        self.dev.sync()
        if not in_place:
            assert np.array_equal(x.read(np.uint32).reshape(qkv.shape), qkv.view(np.uint32))
        return q.read(np.float32).reshape(seqs * n_tok, ldq)


def _same(a, b):
    return np.array_equal(a.astype(np.float64), b.astype(np.float64), equal_nan=True)


# sequences, tokens, query and kv heads, ctx, starts, layout, rotated dims
STORES = [(1, 1, 2, 1, 64, [0], orc.ROPE_HALF, None), (1, 1, 14, 2, 128, [63], orc.ROPE_PAIRS, None),
          (3, 1, 4, 2, 192, [64, -1, 191], orc.ROPE_HALF, 32), (2, 5, 3, 3, 128, [61, 125], orc.ROPE_PAIRS, 6),
          (1, 130, 4, 1, 192, [7], orc.ROPE_HALF, 58), (2, 64, 2, 2, 256, [0, 100], orc.ROPE_PAIRS, 0),
          (2, 200, 1, 2, 256, [64, -3], orc.ROPE_HALF, None), (1, 70, 3, 2, 128, [30], orc.ROPE_PAIRS, 34),
          (3, 16, 2, 1, 64, [48, 49, 3], orc.ROPE_PAIRS, None), (1, 15, 5, 1, 64, [50], orc.ROPE_HALF, 20)]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", STORES)
def test_store_and_load(dev, ty, hd, case):
    """Codes, scales and rotated rows equal the definition's; rows that were not written keep their bytes."""
    S, T, H, KV, ctx, starts, layout, rot = case
    rot = hd if rot is None else rot
    print(f"[gpu] kvq store {ty} {hd} {case}", flush=True)
    rng = np.random.default_rng(S * 1000 + T)
    qkv = rng.normal(0, 1, (S * T, (H + 2 * KV) * hd + 8)).astype(np.float32)
    qkv[:, ::17] *= 30  # channels of another size
    qkv[::3] *= 1e-4    # rows near the smallest scales
    qkv[::7, : -8 - KV * hd] = 0
    rope = _table(dev, 40, ctx, rot, 1e4) if rot else None
    c = Caches(dev, ty, S, KV, ctx, hd)
    before = c.load(ctx)
    assert all(np.isnan(b).all() for b in before)
    q = c.store(qkv, T, H, rope, rot, layout, starts)
    cs = rope.read(np.float32).reshape(ctx, rot // 2, 2) if rot else np.zeros((ctx, 0, 2), np.float32)
    x = qkv[:, :-8].reshape(S, T, H + 2 * KV, hd)
    wk, wv = (np.full((S, KV, ctx, hd), np.nan) for _ in range(2))
    wq = np.full((S, T, H * hd + 4), 7.5)
    for s in range(S):
        for t in range(T):
            p = starts[s] + t
            if starts[s] < 0 or p >= ctx:
                continue
            wq[s, t, :-4] = ref.rotate(x[s, t, :H], cs[p], layout, rot).ravel()
            wk[s, :, p] = ref.quantised(ty, ref.rotate(x[s, t, H:H + KV], cs[p], layout, rot))
            wv[s, :, p] = ref.quantised(ty, x[s, t, H + KV:])
    assert _same(q, wq.reshape(S * T, -1))
    k, v = c.load(ctx)
    assert _same(k, wk) and _same(v, wv)
    # a window of rows, some of them outside the cache: zeros
    at = [p - 2 for p in starts]
    for got, want in zip(c.load(T + 3, at, 1), (wk, wv)):
        for s in range(S):
            for j in range(T + 3):
                p = at[s] + 1 + j
                assert _same(got[s, :, j], want[s, :, p] if 0 <= p < ctx else np.zeros((KV, hd)))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_values_at_the_borders_of_the_formats(dev, ty, hd):
    """Ties between codes, magnitudes at and next to a scale's reach, zeros, subnormals, the largest values, infinities
    and NaN."""
    rng = np.random.default_rng(5)
    n, KV = 64, 2
    x = np.zeros((n, KV, hd // 32, 32), np.float32)
    m = ref.LEVELS.get(ty, 127)
    for i in range(n):
        for g in range(KV):
            for b in range(hd // 32):
                kind, d = (i + g + b) % 8, ref.SCALES[rng.integers(1, 200)]
                u = rng.integers(-2 * m, 2 * m + 1, 32) / 2  # ties
                u[0] = m
                y = (u * d).astype(np.float32)
                if kind == 1:
                    y[0] = np.nextafter(np.float32(m * d), np.float32(np.inf))
                elif kind == 2:
                    y[0] = np.nextafter(np.float32(m * d), np.float32(0))
                elif kind == 3:
                    y = rng.normal(0, 1, 32).astype(np.float32) * np.float32(10.0 ** rng.integers(-42, -4))
                elif kind == 4:
                    y = rng.normal(0, 1, 32).astype(np.float32) * np.float32(10.0 ** rng.integers(3, 38))
                elif kind == 5:
                    y[rng.integers(32)] = [np.inf, -np.inf, np.nan][i % 3]
                elif kind == 6:
                    y = np.nextafter(y, np.float32(rng.choice([-1e9, 1e9])))
                x[i, g, b] = y
    x = x.reshape(n, KV, hd)
    qkv = np.concatenate([rng.normal(0, 1, (n, hd)).astype(np.float32), x.reshape(n, -1), x[::-1].reshape(n, -1)], 1)
    c = Caches(dev, ty, 1, KV, 64, hd)
    c.store(qkv, n, 1)
    few = Caches(dev, ty, 1, KV, 64, hd)  # the same rows by calls of a few tokens each: the same values
    for a in range(0, n, 9):
        few.store(qkv[a:a + 9], min(9, n - a), 1, off=a)
    k, v = c.load(64)
    assert all(_same(p, q) for p, q in zip(few.load(64), (k, v)))
    want = ref.quantised(ty, x)
    assert _same(k[0].transpose(1, 0, 2), want) and _same(v[0].transpose(1, 0, 2), want[::-1])


def test_store_in_place_and_one_cache_read_back(dev):
    rng = np.random.default_rng(8)
    S, T, H, KV, hd, ctx = 2, 3, 4, 2, 64, 128
    qkv = rng.normal(0, 1, (S * T, (H + 2 * KV) * hd)).astype(np.float32)
    rope = _table(dev, 0, ctx + 50, hd, 1e4)
    a, b = (Caches(dev, orc.KV_Q8, S, KV, ctx, hd) for _ in range(2))
    q = a.store(qkv, T, H, rope, hd, orc.ROPE_HALF, [9, 70], rope_off=50)
    y = b.store(qkv, T, H, rope, hd, orc.ROPE_HALF, [9, 70], rope_off=50, in_place=True)
    assert np.array_equal(y[:, :H * hd], q[:, :-4]) and np.array_equal(y[:, H * hd:], qkv[:, H * hd:])
    assert np.array_equal(a.k.read(np.uint8), b.k.read(np.uint8)) and np.array_equal(a.v.read(np.uint8), b.v.read(np.uint8))
    cs = rope.read(np.float32).reshape(-1, hd // 2, 2)
    assert _same(q[0, :-4], ref.rotate(qkv[0, :H * hd].reshape(H, hd), cs[59], orc.ROPE_HALF, hd).ravel())
    k, v = a.load(ctx)
    one = dev.alloc(k.nbytes)
    for buf, d_k, d_v, want in ((a.k, one.ptr, None, k), (a.v, None, one.ptr, v)):
        dev.check(dev.L.orc_kvq_load(orc.KV_Q8, d_k and buf.ptr, d_v and buf.ptr, S, KV, hd, ctx, None, 0, ctx, d_k,
                                     d_v, None))
        dev.sync()
        assert _same(one.read(np.float32).reshape(want.shape), want)


def _attend(dev, own, q, heads, T, prefix=None, P=0, pos=None, off=0, limit=None, pad=4, stream=None):
    """The call on q [S][T][H][hd], rows `pad` floats longer; the output's padding must stay."""
    S, KV, hd, ctx = own.shape
    limit = ctx if limit is None else limit
    n = heads * hd
    rows = np.full((S * T, n + pad), 3.25, np.float32)
    rows[:, :n] = q.reshape(S * T, n)
    dq, do = dev.upload(rows), dev.upload(np.full((S * T, n + 2 * pad), 7.5, np.float32))
    size = dev.L.orc_attn_kvq_workspace(S, T, heads, KV, hd, P, limit)
    work = dev.alloc(size + 64)
    dev.check(dev.L.orc_fill(work.ptr, 0xFF, size + 64, None))
    d = dev.upload(np.asarray(pos, np.int32)) if pos is not None else None
    dev.sync()
    dev.check(dev.L.orc_attn_kvq(own.ty, dq.ptr, n + pad, S, T, heads, KV, hd, prefix and prefix.k.ptr,
                                 prefix and prefix.v.ptr, P, prefix.shape[3] if prefix else 0, own.k.ptr, own.v.ptr, ctx,
                                 d and d.ptr, off, limit, do.ptr, n + 2 * pad, work.ptr if size else None, stream))
    dev.sync()
    assert np.all(work.read(np.uint8, 64, size) == 0xFF)
    got = do.read(np.float32).reshape(S * T, n + 2 * pad)
    assert np.all(got[:, n:] == 7.5)
    return got[:, :n].reshape(S, T, heads, hd)


def _filled(dev, ty, seqs, kv, ctx, hd, lens, rng, amp=1.0):
    """A cache whose sequence i holds lens[i] rows (NaN behind them), and its values"""
    c = Caches(dev, ty, seqs, kv, ctx, hd)
    n = max(max(lens), 1)
    qkv = np.zeros((seqs, n, (1 + 2 * kv) * hd), np.float32)
    qkv[:, :, hd:] = rng.normal(0, amp, (seqs, n, 2 * kv * hd))
    # the longest first, then every shorter sequence's rows behind its end are refilled with NaN by a store of NaN rows
    c.store(qkv.reshape(seqs * n, -1), n, 1, pos=[0 if m else -1 for m in lens])
    if min(lens) < n:
        bad = np.full((seqs * (n - min(lens)), (1 + 2 * kv) * hd), np.nan, np.float32)
        c.store(bad, n - min(lens), 1, pos=lens)
    k, v = c.load(ctx)
    for i, m in enumerate(lens):
        assert np.isfinite(k[i, :, :m]).all() and np.isnan(k[i, :, m:]).all() and np.isnan(v[i, :, m:]).all()
    return c, k, v


def _held(got, want, scale, size, total):
    err = np.abs(got - want)
    bound = (5e-6 + 2.5e-6 * size) * scale + 2.0 ** -39 * total
    assert np.all(err <= bound), float(np.max(err / bound))


# sequences, tokens, query heads, kv heads, prefix rows, starts, pos_limit (None: ctx), ctx
ATTENTIONS = [
    (1, 1, 1, 1, 0, [0], None, 64),                       # one key
    (1, 1, 8, 2, 0, [62], None, 64), (1, 1, 8, 2, 0, [63], 64, 128), (1, 1, 14, 2, 0, [64], None, 128),
    (1, 1, 4, 4, 0, [700], None, 1024),                   # several chunks
    (1, 1, 24, 2, 1, [0], None, 64), (1, 2, 32, 2, 130, [5], None, 192),  # a prefix of one sequence
    (1, 9, 7, 1, 0, [331], None, 512),                    # a verify pass
    (1, 70, 4, 2, 0, [0], None, 128), (1, 131, 3, 1, 65, [10], None, 192),  # prompts
    (2, 300, 4, 2, 64, [0, 33], None, 384),
    (3, 1, 8, 2, 63, [0, -1, 40], None, 64), (2, 1, 2, 2, 64, [127, 0], 128, 256), (5, 1, 4, 1, 65, [3, 64, 9, 0, 63], 66, 128),
    (17, 1, 8, 2, 1000, list(range(0, 68, 4)), None, 128),  # a shared prompt
    (4, 3, 28, 4, 200, [0, 126, -1, 61], 128, 128),       # tokens behind the limit, an idle slot
    (2, 20, 6, 3, 300, [44, -5], None, 64), (40, 2, 16, 2, 513, [7] * 40, 9, 64),
    (2, 1, 4, 2, 0, [-1, -1], None, 64), (3, 1, 4, 2, 70, [-1, -1, -1], None, 64),  # nothing to attend to
]
# enough rows and keys for the forms that share more: 64-row tiles by one key group, 128-row tiles behind long contexts and
# over long shared prefixes (own rows by 16 and by 32), chunks by the dozen
LARGE = [
    (16, 400, 8, 4, 0, [0] * 15 + [3], 640, 640), (4, 70, 16, 8, 0, [3000, 2999, 2950, 17], None, 3136),
    (400, 1, 8, 8, 6200, [i % 61 - 1 for i in range(400)], None, 64), (40, 5, 32, 8, 3601, list(range(40)), 64, 64),
    (1, 1, 8, 2, 0, [5000], None, 5056),
    # own rows of several blocks a wave beside a prefix's tiles
    (17, 1, 8, 2, 1000, [37 * i for i in range(17)], None, 640), (4, 3, 28, 4, 200, [600, 331, -1, 63], None, 640),
    # chunks by the hundred, of own rows and of a prefix
    (1, 1, 8, 1, 0, [33000], None, 33024), (3, 1, 8, 1, 17000, [9000, 5, 8999], None, 9024), (5, 1, 8, 1, 70001, [40, 0, 7, 63, -1], None, 64),
    (100, 1, 16, 4, 12300, [3 * i for i in range(100)], None, 320), (25, 5, 16, 4, 12300, [12 * i for i in range(25)], None, 320),
]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", ATTENTIONS + LARGE)
def test_attention(dev, ty, hd, case):
    S, T, H, KV, P, starts, limit, ctx = case
    print(f"[gpu] attn_kvq {ty} {hd} {case}", flush=True)
    rng = np.random.default_rng(S * 10000 + T * 100 + P)
    end = limit or ctx
    own, k, v = _filled(dev, ty, S, KV, ctx, hd, [min(s + T, end) if s >= 0 else 0 for s in starts], rng)
    pre, pk, pv = None, np.zeros((KV, 0, hd)), np.zeros((KV, 0, hd))
    if P:
        pre, a, b = _filled(dev, ty, 1, KV, (P + 63) // 64 * 64, hd, [P], rng)
        pk, pv = a[0, :, :P], b[0, :, :P]
    q = rng.normal(0, 1, (S, T, H, hd)).astype(np.float32)
    got = _attend(dev, own, q, H, T, pre, P, starts, 0, limit)
    _held(got, *ref.attention(q, pk, pv, k, v, starts, end))


# every attention kernel, with tokens of one sequence that see different keys (the last: three blocks of them in a tile)
ODD = [(1, 5, 3, 1, 0, [61], None, 128), (2, 5, 4, 1, 0, [62, 0], None, 128), (1, 9, 7, 1, 70, [331], None, 512),
       (16, 400, 8, 4, 0, [0] * 15 + [3], 640, 640), (4, 70, 16, 8, 0, [3000, 2999, 2950, 17], None, 3136),
       (17, 3, 8, 2, 1000, [20 * i for i in range(17)], None, 384), (4, 3, 28, 4, 200, [600, 331, -1, 63], None, 640),
       (50, 2, 16, 4, 12300, [3 * i for i in range(50)], None, 320), (25, 5, 16, 4, 12300, [12 * i for i in range(25)], None, 320),
       (8, 130, 8, 8, 0, [2999, 3000, 3001, 2950, 3040, 3050, 3062, 7], None, 3200)]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", ODD)
def test_nan_in_a_new_row_reaches_only_the_tokens_that_see_it(dev, ty, hd, case):
    """NaN and infinities in the V rows of some of the call's own tokens, and NaN in a K row: the tokens before them are as
    they should be, the ones from there on not finite where the row is not."""
    S, T, H, KV, P, starts, limit, ctx = case
    print(f"[gpu] attn_kvq, odd rows {ty} {hd} {case}", flush=True)
    rng = np.random.default_rng(S * 10000 + T * 100 + P + 1)
    end, G = limit or ctx, H // KV
    own, k, v = _filled(dev, ty, S, KV, ctx, hd, [min(s + T, end) if s >= 0 else 0 for s in starts], rng)
    pre, pk, pv = None, np.zeros((KV, 0, hd)), np.zeros((KV, 0, hd))
    if P:
        pre, a, b = _filled(dev, ty, 1, KV, (P + 63) // 64 * 64, hd, [P], rng)
        pk, pv = a[0, :, :P], b[0, :, :P]
    q = rng.normal(0, 1, (S, T, H, hd)).astype(np.float32)
    # row t of sequence s anew: V with NaN (dim 3), an infinity (the last dim) and, in one kv head, K with NaN
    marks = []
    for s in range(S):
        if starts[s] < 0:
            continue
        t = int(rng.integers(T))
        row = np.zeros((1, (1 + 2 * KV) * hd), np.float32)
        kk, vv = k[s, :, starts[s] + t].copy(), v[s, :, starts[s] + t].copy()
        vv[0, 3], vv[KV - 1, hd - 1] = np.nan, np.inf
        if s % 2 and KV > 1:
            kk[1, 7] = np.nan
        row[0, hd:] = np.concatenate([kk.ravel(), vv.ravel()])
        one = [-1] * S
        one[s] = starts[s] + t
        own.store(np.repeat(row, S, 0), 1, 1, pos=one)
        marks.append((s, t))
    k2, v2 = own.load(ctx)
    # (the row's other values as the cache now holds them: quantised a second time, they may have moved)
    want, scale, size, total = ref.attention(q, pk, pv, *(np.nan_to_num(x, posinf=0) for x in (k2, v2)), starts, end)
    got = _attend(dev, own, q, H, T, pre, P, starts, 0, limit)
    for s, t in marks:
        p = starts[s] + t
        bad = ~np.isfinite(v2[s, :, p])  # [KV][hd]
        bad |= ~np.isfinite(k2[s, :, p]).all(-1)[:, None]
        assert bad[0, 3] and bad[KV - 1, hd - 1]
        bad = np.repeat(bad, G, 0)
        assert not np.isfinite(got[s, t:][:, bad]).any(), (s, t)  # an infinity: NaN or infinite
        got[s, t:][:, bad] = want[s, t:][:, bad]
    assert np.isfinite(got).all()
    _held(got, want, scale, size, total)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("amp", [1e-6, 1e-3, 30.0, 3e4])
def test_attention_of_large_and_small_queries(dev, ty, amp):
    """Queries of any size: softmax from even to one key only."""
    S, T, H, KV, hd, P, ctx = 2, 2, 4, 2, 64, 100, 128
    rng = np.random.default_rng(int(amp * 10) + ty)
    own, k, v = _filled(dev, ty, S, KV, ctx, hd, [102, 32], rng)
    pre, pk, pv = _filled(dev, ty, 1, KV, 128, hd, [P], rng)
    q = (rng.normal(0, 1, (S, T, H, hd)) * amp).astype(np.float32)
    q[0, 1, 2] = 0  # even weights
    got = _attend(dev, own, q, H, T, pre, P, [100, 30])
    want, scale, size, total = ref.attention(q, pk[0, :, :P], pv[0, :, :P], k, v, [100, 30], ctx)
    err = np.abs(got - want)
    # weights far from the largest key's may be off by more than their first-order change: one whole sum w |v| at most
    bound = np.minimum(np.expm1(5e-6 + 2.5e-6 * size), 2.0) * scale + 2.0 ** -39 * total
    if amp <= 30:
        assert np.all(err <= bound), float(np.max(err / bound))
    else:  # the scores' rounding passes 1: what is left is that the result is a mean of rows
        assert np.isfinite(got).all() and np.abs(got).max() <= max(np.nanmax(np.abs(v)), np.nanmax(np.abs(pv))) * 1.0001


def test_a_row_of_nan_or_infinite_queries_stays_alone(dev):
    S, T, H, KV, hd, ctx = 1, 3, 4, 1, 128, 256
    rng = np.random.default_rng(12)
    own, k, v = _filled(dev, orc.KV_Q8, S, KV, ctx, hd, [203], rng)
    q = rng.normal(0, 1, (S, T, H, hd)).astype(np.float32)
    want, scale, size, total = ref.attention(q, np.zeros((KV, 0, hd)), np.zeros((KV, 0, hd)), k, v, [200], ctx)
    q[0, 1, 2, 5], q[0, 2, 0, 0] = np.nan, np.inf
    got = _attend(dev, own, q, H, T, pos=[200])
    for t, h in ((1, 2), (2, 0)):
        assert np.isnan(got[0, t, h]).all()
        got[0, t, h] = want[0, t, h]
    _held(got, want, scale, size, total)


def test_host_positions_and_another_stream(dev):
    S, T, H, KV, hd, ctx = 2, 3, 8, 2, 128, 320
    rng = np.random.default_rng(13)
    s = C.c_void_p()
    dev.check(dev.L.orc_stream_create(C.byref(s)))
    own, k, v = _filled(dev, orc.KV_Q4, S, KV, ctx, hd, [290, 290], rng)
    q = rng.normal(0, 1, (S, T, H, hd)).astype(np.float32)
    none = np.zeros((KV, 0, hd))
    got = _attend(dev, own, q, H, T, off=287, limit=290, stream=s)
    _held(got, *ref.attention(q, none, none, k, v, [287, 287], 290))
    again = _attend(dev, own, q, H, T, pos=[280, 285], off=4, limit=290, stream=s)
    _held(again, *ref.attention(q, none, none, k, v, [284, 289], 290))
    dev.check(dev.L.orc_stream_destroy(s))


@pytest.mark.parametrize("ty", TYPES)
def test_same_call_twice_gives_the_same_bits(dev, ty):
    rng = np.random.default_rng(14)
    own, k, v = _filled(dev, ty, 9, 2, 192, 128, [150 + i for i in range(9)], rng)
    pre, _, _ = _filled(dev, ty, 1, 2, 640, 128, [600], rng)
    q = rng.normal(0, 1, (9, 2, 8, 128)).astype(np.float32)
    a, b = (_attend(dev, own, q, 8, 2, pre, 600, [148 + i for i in range(9)]) for _ in range(2))
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_agrees_with_the_attention_over_fp32_rows(dev):
    """orc_attn_gqa on the rows read back: the same values, both within fp32 rounding of the exact result."""
    H, KV, hd, ctx, P = 8, 2, 64, 448, 400
    rng = np.random.default_rng(15)
    own, k, v = _filled(dev, orc.KV_Q8, 1, KV, ctx, hd, [P + 1], rng)
    q = rng.normal(0, 1, (1, 1, H, hd)).astype(np.float32)
    got = _attend(dev, own, q, H, 1, pos=[P])
    dq, dk, dv = dev.upload(q), dev.upload(np.nan_to_num(k)), dev.upload(np.nan_to_num(v))
    out, work = dev.alloc(4 * H * hd), dev.alloc(dev.L.orc_attn_workspace(1, H, hd, ctx))
    dev.check(dev.L.orc_attn_gqa(dq.ptr, H * hd, 1, H, KV, hd, P, dk.ptr, dv.ptr, ctx, out.ptr, H * hd, work.ptr, None))
    dev.sync()
    other = out.read(np.float32).reshape(got.shape)
    none = np.zeros((KV, 0, hd))
    want, scale, size, total = ref.attention(q, none, none, k, v, [P], ctx)
    _held(got, want, scale, size, total)
    assert np.all(np.abs(got - other) <= 2 * (5e-6 + 2.5e-6 * size) * scale)


@pytest.mark.parametrize("ty,hd,layout", [(orc.F16, 64, orc.ROPE_HALF), (orc.KV_Q8, 128, orc.ROPE_HALF),
                                          (orc.KV_Q4, 128, orc.ROPE_PAIRS)])
def test_continuations_of_one_prompt(dev, ty, hd, layout):
    """The operators as they are used: a scaled table, a prompt stored and attended to in two passes, then decode
    steps of several continuations, captured once and replayed with positions that advance on the device."""
    H, KV, S, P, ctx, rot = 8, 2, 5, 150, 64, hd // 2
    rng = np.random.default_rng(hd + ty)
    dev_, L, ld = dev, dev.L, (H + 2 * KV) * hd
    rope = _table(dev, 0, 192 + ctx, rot, 1e4, (orc.ROPE_BANDS, 4.0, 1.0, 4.0, 64, 0.0))
    cs = rope.read(np.float32).reshape(-1, rot // 2, 2)
    pre, own = Caches(dev, ty, 1, KV, 192, hd), Caches(dev, ty, S, KV, ctx, hd)
    none = np.zeros((KV, 0, hd))
    prompt = rng.normal(0, 1, (P, ld)).astype(np.float32)
    for a, b in ((0, 100), (100, P)):
        q = pre.store(prompt[a:b], b - a, H, rope, rot, layout, off=a)[:, :-4].reshape(1, b - a, H, hd)
        assert _same(q[0, 3], ref.rotate(prompt[a + 3, :H * hd].reshape(H, hd), cs[a + 3], layout, rot))
        k, v = pre.load(192)
        _held(_attend(dev, pre, q, H, b - a, off=a), *ref.attention(q, none, none, k, v, [a], 192))
    k, v = pre.load(192)
    pk, pv = k[0, :, :P], v[0, :, :P]
    starts = np.array([0, 3, -1, 1, 0], np.int32)  # one slot idle; the others hold a few rows already
    first = rng.normal(0, 1, (S * 3, ld)).astype(np.float32)
    own.store(first, 3, H, rope, rot, layout, [0, 0, -1, 0, 0], rope_off=P)
    # one captured step: write, attend
    x, q, out = dev.alloc(4 * S * ld), dev.alloc(4 * S * H * hd), dev.alloc(4 * S * H * hd)
    pos, work = dev.upload(starts), dev.alloc(max(16, L.orc_attn_kvq_workspace(S, 1, H, KV, hd, P, ctx)))
    s, graph = C.c_void_p(), C.c_void_p()
    dev.check(L.orc_stream_create(C.byref(s)))

    def step():
        dev.check(L.orc_kvq_store(ty, x.ptr, ld, S, 1, H, KV, hd, layout, rot, rope.ptr, P, pos.ptr, 0, q.ptr, H * hd,
                                  own.k.ptr, own.v.ptr, ctx, s))
        dev.check(L.orc_attn_kvq(ty, q.ptr, H * hd, S, 1, H, KV, hd, pre.k.ptr, pre.v.ptr, P, 192, own.k.ptr, own.v.ptr,
                                 ctx, pos.ptr, 0, ctx, out.ptr, H * hd, work.ptr, s))

    dev.check(L.orc_graph_begin(s))
    step()
    dev.check(L.orc_graph_end(s, C.byref(graph)))
    for i in range(4):
        rows = rng.normal(0, 1, (S, ld)).astype(np.float32)
        x.write(rows)
        q.write(np.zeros((S, H * hd), np.float32))
        pos.write(starts)
        dev.sync()
        dev.check(L.orc_graph_launch(graph, s))
        dev.check(L.orc_stream_sync(s))
        got = out.read(np.float32).reshape(S, 1, H, hd)
        qr = q.read(np.float32).reshape(S, 1, H, hd)
        k, v = own.load(ctx)
        for n in range(S):
            if starts[n] >= 0:
                p = starts[n]
                kv = rows[n, H * hd:].reshape(2, KV, hd)
                assert _same(k[n, :, p], ref.quantised(ty, ref.rotate(kv[0], cs[P + p], layout, rot)))
                assert _same(v[n, :, p], ref.quantised(ty, kv[1]))
        _held(got, *ref.attention(qr, pk, pv, k, v, starts, ctx))
        assert np.all(got[2] == 0)
        out.write(np.zeros_like(got))
        step()  # the same step launched from the host
        dev.check(L.orc_stream_sync(s))
        assert np.array_equal(out.read(np.uint32), got.view(np.uint32).ravel())
        starts = np.where(starts >= 0, starts + 1, starts).astype(np.int32)
    dev.check(L.orc_graph_destroy(graph))
    dev.check(L.orc_stream_destroy(s))


@pytest.mark.parametrize("T,layout,rot", [(20, orc.ROPE_HALF, 128), (20, orc.ROPE_HALF, 40), (33, orc.ROPE_PAIRS, 128), (2, orc.ROPE_PAIRS, 40)])
def test_store_in_place_of_every_form(dev, T, layout, rot):
    rng = np.random.default_rng(T + rot)
    S, H, KV, hd, ctx = 2, 4, 2, 128, 128
    qkv = rng.normal(0, 1, (S * T, (H + 2 * KV) * hd)).astype(np.float32)
    rope = _table(dev, 0, ctx, rot, 1e4)
    a, b = (Caches(dev, orc.KV_Q4, S, KV, ctx, hd) for _ in range(2))
    q = a.store(qkv, T, H, rope, rot, layout, [9, 70])
    y = b.store(qkv, T, H, rope, rot, layout, [9, 70], in_place=True)
    assert np.array_equal(y[:, :H * hd], q[:, :-4]) and np.array_equal(y[:, H * hd:], qkv[:, H * hd:])
    assert np.array_equal(a.k.read(np.uint8), b.k.read(np.uint8)) and np.array_equal(a.v.read(np.uint8), b.v.read(np.uint8))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,layout,rot", [(5, orc.ROPE_HALF, None), (6, orc.ROPE_PAIRS, None), (7, orc.ROPE_PAIRS, 38),
                                          (14, orc.ROPE_HALF, None), (3, orc.ROPE_HALF, 38)])
def test_a_prompt_is_written_as_its_tokens_one_by_one(dev, hd, H, layout, rot):
    rng = np.random.default_rng(H)
    S, T, KV, ctx, rot = 2, 41, 1, 128, rot or hd
    starts = np.array([3, 70])
    qkv = rng.normal(0, 1, (S, T, (H + 2 * KV) * hd)).astype(np.float32)
    rope = _table(dev, 0, ctx, rot, 1e4)
    a, b, c = (Caches(dev, orc.KV_Q8, S, KV, ctx, hd) for _ in range(3))
    q = a.store(qkv.reshape(S * T, -1), T, H, rope, rot, layout, starts)[:, :H * hd].reshape(S, T, -1)
    y = b.store(qkv.reshape(S * T, -1), T, H, rope, rot, layout, starts, in_place=True)[:, :H * hd].reshape(S, T, -1)
    assert np.array_equal(q, y)
    for t in range(T):
        one = c.store(np.ascontiguousarray(qkv[:, t]), 1, H, rope, rot, layout, starts + t)
        assert np.array_equal(one[:, :H * hd], q[:, t])
    for other in (b, c):
        assert np.array_equal(a.k.read(np.uint8), other.k.read(np.uint8)) and np.array_equal(a.v.read(np.uint8), other.v.read(np.uint8))


@pytest.mark.parametrize("ty", [orc.F16, orc.KV_Q8])
def test_a_cache_of_more_than_4_gb(dev, ty):
    """The last rows of the last of three sequences of 2^20 (F16; 8 bits: 2^21) positions, zeros before them: the rows
    read back, and attention, whose zero keys weigh exp(0) each.

    Bound: as the others', with up to 2^21 / 64 / 64 = 512 blocks added up per chunk at 2^-24 each, in two sums: 6.1e-5.
    """
    S, H, KV, hd, T = 3, 8, 8, 128, 3
    ctx = 1 << (20 if ty == orc.F16 else 21)
    rng = np.random.default_rng(21)
    print(f"[gpu] caches of {dev.L.orc_kvq_bytes(ty, S, KV, ctx, hd) / 2 ** 30:.1f} GB", flush=True)
    c = Caches(dev, ty, S, KV, ctx, hd)
    assert c.bytes > 4 << 30
    for b in (c.k, c.v):
        dev.check(dev.L.orc_fill(b.ptr, 0, c.bytes, None))
    if ty != orc.F16:  # code 128 is zero; byte 0 of a group whose scale is zero stands for zero too
        assert not np.any(c.load(4)[0])
    pos = [-1, -1, ctx - T]
    qkv = rng.normal(0, 1, (S * T, (H + 2 * KV) * hd)).astype(np.float32)
    c.store(qkv, T, H, pos=pos)
    x = qkv.reshape(S, T, H + 2 * KV, hd)[2]
    k, v = (ref.quantised(ty, x[:, a:a + KV]) for a in (H, H + KV))
    got_k, got_v = c.load(T + 2, [0, ctx - T - 2, ctx - T - 2])
    for got, want in ((got_k, k), (got_v, v)):
        assert _same(got[2, :, 2:].transpose(1, 0, 2), want) and not np.any(got[2, :, :2]) and not np.any(got[:2])
    q = (x[:, :H] * 3).astype(np.float32)  # the last keys count against 2^20 zeros
    full = np.zeros((S, T, H, hd), np.float32)
    full[2] = q
    got = _attend(dev, c, full, H, T, pos=pos)
    assert not np.any(got[:2])
    for t in range(T):
        for h in range(H):
            s = (k[:t + 1, h] @ q[t, h].astype(np.float64)) / np.sqrt(hd)
            n0 = ctx - T
            m = max(s.max(), 0)
            w, z = np.exp(s - m), n0 * np.exp(-m)
            total = w.sum() + z
            size = (np.abs(k[:t + 1, h]) @ np.abs(q[t, h])).max() / np.sqrt(hd)
            err = np.abs(got[2, t, h] - w @ v[:t + 1, h] / total)
            assert np.all(err <= (6.6e-5 + 2.5e-6 * size) * (w @ np.abs(v[:t + 1, h]) / total) + 2.0 ** -39 * np.abs(v[:t + 1, h]).sum(0)), (t, h)


def test_calls_on_two_streams_at_once(dev):
    """Different shapes on two streams, each with a workspace of its own: the bits of the same calls one by one."""
    rng = np.random.default_rng(30)
    hd, KV = 128, 2
    jobs = []
    for S, T, H, P, starts, ctx in ((9, 1, 8, 900, list(range(9)), 64), (1, 90, 4, 0, [300], 448)):
        own, _, _ = _filled(dev, orc.KV_Q8, S, KV, ctx, hd, [s + T for s in starts], rng)
        pre = _filled(dev, orc.KV_Q8, 1, KV, (P + 63) // 64 * 64, hd, [P], rng)[0] if P else None
        q = rng.normal(0, 1, (S, T, H, hd)).astype(np.float32)
        want = _attend(dev, own, q, H, T, pre, P, starts, pad=0)
        s = C.c_void_p()
        dev.check(dev.L.orc_stream_create(C.byref(s)))
        size = dev.L.orc_attn_kvq_workspace(S, T, H, KV, hd, P, ctx)
        jobs.append((s, dev.upload(q), dev.alloc(q.nbytes), dev.alloc(size + 16), dev.upload(np.asarray(starts, np.int32)), want,
                     (S, T, H, P, ctx, own, pre)))
    dev.sync()
    for _ in range(20):
        for s, q, out, work, pos, _, (S, T, H, P, ctx, own, pre) in jobs:
            dev.check(dev.L.orc_attn_kvq(orc.KV_Q8, q.ptr, H * hd, S, T, H, KV, hd, pre and pre.k.ptr, pre and pre.v.ptr, P,
                                         pre.shape[3] if pre else 0, own.k.ptr, own.v.ptr, ctx, pos.ptr, 0, ctx, out.ptr,
                                         H * hd, work.ptr, s))
    dev.sync()
    for s, q, out, work, pos, want, _ in jobs:
        assert np.array_equal(out.read(np.uint32), want.view(np.uint32).ravel())
        dev.check(dev.L.orc_stream_destroy(s))
