"""The 8-bit cache and trees of drafted tokens (norm_rope_kv, kv_read, atencion_mx8, atencion_arbol, kv_ramal) against float64.

Stored blocks, f16 rounding and moved rows are exact.  Rotated values: norms (a sum of 128 squares in a tree: 8 roundings, a
division, a root, two products), the sine or cosine (a reduced angle's rounding and the polynomial's, 2^-22 together) and the
rotation (3 roundings) add up to at most ROT = 24 roundings of 2^-24 of |a| + |b|, a and b the normed pair.
Attention: keys and values are exact, queries and probabilities 22 bits, scores sums of 8 (hd = 128: twice 4 steps) float32
additions, so a score is off by at most e = 2^-20 sum |q k| scale and an output by (2 e + 2^-19) max |v| (2^-19: probabilities,
the sums over up to 2000 keys, the shares' weights)."""
import ctypes

import numpy as np
import pytest

from quipullm_amd import capi
import mx8
from mx8 import F16, F32, MX8
from test_gpu_ops import dev  # noqa: F401

pytestmark = pytest.mark.gpu
ROT = 24 * 2.0 ** -24
FMTS = [F32, F16, MX8]


def table(nrot, base=500000.0):
    e = np.float32(-2.0) * np.arange(max(1, nrot // 2), dtype=np.float32) / np.float32(max(1, nrot))
    return np.power(base, e.astype(np.float64)).astype(np.float32)


def rotate(x, w, pos, nrot, neox, esc=1.0, eps=1e-6):
    """x [T][heads][hd] normed (w given) and rotated -> (values float64, |a| + |b| of each value's pair)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float32(eps)) * w.astype(np.float64)
    half = nrot // 2
    ang = ((pos.astype(np.float32) * np.float32(esc))[:, None] * table(nrot)[None, :half]).astype(np.float64)[:, None]
    j = np.arange(half)
    i0, i1 = (j, j + half) if neox else (2 * j, 2 * j + 1)
    a, b = x[..., i0], x[..., i1]
    y, size = x.copy(), np.abs(x)
    y[..., i0], y[..., i1] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
    size[..., i0] = size[..., i1] = np.abs(a) + np.abs(b)
    return y, size


def store(quipu, dev, q, k, v, pos0, rows, fmt, cap=0, neox=0, nrot=0, qn=None, kn=None, pos=None, esc=0, fill=0x5a, inplace=False, T=None):
    """norm_rope_kv into caches of `fill` bytes; returns (qo, kc, vc as raw bytes, handles)."""
    nt, nh, hd = q.shape
    nkv = k.shape[1]
    n = mx8.nbytes(fmt, rows, nkv, hd)
    kc, vc = (dev.buf(np.full(n, fill, np.uint8)) for _ in "kv")
    qb = dev.buf(q)
    qo = qb if inplace else dev.buf(np.full(q.shape, 7.0, np.float32))
    opt = [dev.buf(x) if x is not None else 0 for x in (qn, kn)]
    quipu.dispatch("norm_rope_kv", [("u", hd), ("u", nh), ("u", nkv), ("u", neox), ("f", 1e-6), ("u", nrot), ("f", esc), ("u", cap),
                                    ("u", fmt), ("u", rows)],
                   [dev.paso(nt if T is None else T, pos0), qb, dev.buf(k), dev.buf(v), qo, kc, vc] + opt +
                   [dev.buf(table(nrot)) if nrot else 0, dev.buf(pos.astype(np.uint32)) if pos is not None else 0], (nh, nt))
    return dev.get(qo, q.shape), dev.get(kc, (n,), np.uint8), dev.get(vc, (n,), np.uint8), (kc, vc)


def read(quipu, dev, hs, nkv, hd, fmt, rows, p0, n, cap=0, half=0):
    t = np.float16 if half else np.float32
    out = [dev.buf(np.full((n + 1, nkv, hd), 3.0, t)) for _ in "kv"]
    quipu.dispatch("kv_read", [("u", hd), ("u", nkv), ("u", cap), ("u", fmt), ("u", rows), ("u", p0), ("u", n), ("u", half)],
                   [0, hs[0], hs[1]] + out, (nkv, max(1, n)))
    got = [dev.get(h, (n + 1, nkv, hd), t) for h in out]
    assert all(np.all(g[n] == 3.0) for g in got)   # nothing past the rows
    return got[0][:n], got[1][:n]


def awkward(rng, shape):
    """Rows whose blocks hold every kind of magnitude: zeros, denormals, borders of the scale, ties of the rounding."""
    x = (rng.standard_normal(shape) * 10.0 ** rng.integers(-6, 4, shape[:-1] + (1,))).astype(np.float32)
    b = x.reshape(-1, 32)
    for i, kind in enumerate(rng.integers(0, 9, b.shape[0])):
        if kind == 0:
            b[i] = 0
        elif kind == 1:
            b[i] *= np.float32(1e-40 / max(1e-30, np.abs(b[i]).max()))
        elif kind == 2:
            b[i] = np.float32(0.25) * (rng.integers(-509, 510, 32)).astype(np.float32) * np.float32(2.0 ** rng.integers(-30, 30))
            b[i, 0] = 0.25 * 509 * np.abs(b[i]).max() / max(1e-30, np.abs(b[i]).max())
        elif kind == 3:
            b[i, 5] = np.float32(127.5 * 2.0 ** rng.integers(-20, 20))   # a scale's border
        elif kind == 4:
            b[i, 5] = np.nextafter(np.float32(127.5), np.float32(0))
        elif kind == 5:
            b[i, 7] = np.float32(3.0e38)
        elif kind == 6:
            b[i, 9] = (np.nan, np.inf, -np.inf)[i % 3]
        elif kind == 7:
            b[i] = rng.integers(-127, 128, 32) + np.float32(0.5)          # ties at a step of 1
            b[i, 3] = 100.0
    return x


@pytest.mark.parametrize("hd,nkv,T,pos0,rows,cap", [(128, 8, 1, 0, 1, 0), (128, 2, 1, 4100, 4101, 0), (64, 3, 37, 30, 70, 0),
                                                    (128, 1, 70, 5, 77, 0), (64, 5, 50, 90, 61, 61), (128, 4, 33, 1000, 40, 40)])
def test_blocks_are_exact(quipu, dev, hd, nkv, T, pos0, rows, cap):
    """The 8-bit cache's bytes after a store without norms or rotation, other slots as they were; kv_read gives what they
    stand for."""
    rng = np.random.default_rng(5)
    k, v = awkward(rng, (T, nkv, hd)), awkward(rng, (T, nkv, hd))
    q = rng.standard_normal((T, 2 * nkv, hd)).astype(np.float32)
    qo, kc, vc, hs = store(quipu, dev, q, k, v, pos0, rows, MX8, cap)
    assert np.array_equal(qo, q)
    R = mx8.slots32(rows)
    slots = (pos0 + np.arange(T)) % (cap or 1 << 30)
    for got, x, lay in ((kc, k, mx8.k_bytes), (vc, v, mx8.v_bytes)):
        q8, e8 = np.full((R, nkv, hd), 0x5a, np.uint8), np.full((R, nkv, hd // 32), 0x5a, np.uint8)
        q8[slots], e8[slots] = mx8.quantise(x)
        assert np.array_equal(got, lay(q8, e8))
    for half in (0, 1):
        gk, gv = read(quipu, dev, hs, nkv, hd, MX8, rows, pos0, T, cap, half)
        for got, x in ((gk, k), (gv, v)):
            with np.errstate(over="ignore"):
                want = mx8.dequantise(*mx8.quantise(x)).astype(np.float16 if half else np.float32)
            assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,nh,nkv,T,pos0,nrot,neox,norm", [
    (128, 32, 8, 1, 4100, 128, 0, 0), (128, 4, 4, 5, 0, 128, 1, 1), (64, 6, 2, 33, 31, 64, 1, 0), (64, 1, 1, 3, 7, 64, 0, 1),
    (128, 3, 1, 40, 130000, 128, 0, 1), (128, 6, 2, 9, 12, 64, 1, 1), (64, 5, 5, 17, 3, 22, 0, 0), (128, 2, 2, 2, 0, 34, 1, 0)])
def test_rotation(quipu, dev, fmt, hd, nh, nkv, T, pos0, nrot, neox, norm):
    """Norms, rotation (all channels or the first of them) and storing, against the formula; q in place and apart from it."""
    rng = np.random.default_rng(6)
    q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) for h in (nh, nkv, nkv))
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in "qk") if norm else (None, None)
    rows = pos0 + T + 3
    qo, kc, vc, hs = store(quipu, dev, q, k, v, pos0, rows, fmt, 0, neox, nrot, qn, kn, inplace=bool(T % 2))
    pos = pos0 + np.arange(T)
    want, size = rotate(q, qn, pos, nrot, neox)
    assert np.all(np.abs(qo - want) <= ROT * size)
    gk, gv = read(quipu, dev, hs, nkv, hd, fmt, rows, pos0, T)
    want, size = rotate(k, kn, pos, nrot, neox)
    if fmt == F32:
        assert np.all(np.abs(gk - want) <= ROT * size) and np.array_equal(gv, v)
    elif fmt == F16:
        assert np.all(np.abs(gk - want) <= ROT * size + 2.0 ** -11 * np.abs(want) + 2.0 ** -25)
        assert np.array_equal(gv, v.astype(np.float16))
    else:
        # half a step of the block's scale; one step more only where the value is that near to a border
        step = 2.0 ** (mx8.quantise(want.astype(np.float32))[1].astype(np.float64) - 133).repeat(32, -1)
        assert np.all(np.abs(gk - want) <= 0.5 * step + 2 * ROT * size + 0.5 * step * (np.abs(want) > 63 * step))
        assert np.array_equal(gv, mx8.dequantise(*mx8.quantise(v)).astype(np.float32))


def test_rotation_at_given_positions(quipu, dev):
    """Positions of the tokens' own (the depths of a tree), far ones, a repeated one, linear RoPE scaling; rows that the
    dispatch or the Paso does not cover stay as they were."""
    rng = np.random.default_rng(7)
    T, nh, nkv, hd = 6, 3, 1, 128
    q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) for h in (nh, nkv, nkv))
    pos = np.array([10, 11, 11, 12, 1000003, 0])
    qo, _, _, hs = store(quipu, dev, q, k, v, 20, 40, F32, 0, 1, hd, None, None, pos, 0.125, fill=0)
    want, size = rotate(q, None, pos, hd, 1, 0.125)
    assert np.all(np.abs(qo - want) <= ROT * size)
    gk, _ = read(quipu, dev, hs, nkv, hd, F32, 40, 19, 8)
    want, size = rotate(k, None, pos, hd, 1, 0.125)
    assert np.all(np.abs(gk[1:7] - want) <= ROT * size) and np.all(gk[[0, 7]] == 0)
    qo, _, _, hs = store(quipu, dev, q, k, v, 20, 40, F32, 0, 0, hd, fill=0, T=4)
    assert np.all(qo[4:] == 7.0) and not np.any(qo[:4] == 7.0)
    assert np.all(read(quipu, dev, hs, nkv, hd, F32, 40, 24, 2)[0] == 0)
    # slots past the cache are not written, the others are
    _, kc, vc, hs = store(quipu, dev, q, k, v, 37, 40, MX8, 0, 0, 0)
    assert np.array_equal(read(quipu, dev, hs, nkv, hd, MX8, 40, 37, 3)[1], mx8.dequantise(*mx8.quantise(v[:3])).astype(np.float32))


@pytest.mark.parametrize("fmt", [F32, F16])
def test_read_of_rings(quipu, dev, fmt):
    rng = np.random.default_rng(8)
    rows, nkv, hd, cap = 45, 2, 64, 43
    k, v = (rng.standard_normal((rows, nkv, hd)) for _ in "kv")
    kc, vc, kh, vh = mx8.cache(fmt, k, v)
    hs = dev.buf(kc), dev.buf(vc)
    at = (1000 + np.arange(cap)) % cap
    for half in (0, 1):
        gk, gv = read(quipu, dev, hs, nkv, hd, fmt, rows, 1000, cap, cap, half)
        t = np.float16 if half else np.float32
        assert np.array_equal(gk, kh[at].astype(t)) and np.array_equal(gv, vh[at].astype(t))
    assert read(quipu, dev, hs, nkv, hd, fmt, rows, 45, 0)[0].size == 0


def bound(q, k, v, see, scale):
    """Allowed error of each (t, h): the docstring's, over the keys that the row sees."""
    T, nh, hd = q.shape
    out = np.zeros((T, nh, 1))
    for t in range(T):
        on = np.flatnonzero(see[t])
        for h in range(nh if len(on) else 0):
            kk, vv = (np.abs(x[on, h * k.shape[1] // nh]) for x in (k, v))
            out[t, h] = (2 * 2.0 ** -20 * (kk @ np.abs(q[t, h].astype(np.float64))).max() * scale + 2.0 ** -19) * vv.max()
    return out


def causal(T, pos0, swa, n):
    p, at = np.arange(n)[None], (pos0 + np.arange(T))[:, None]
    return (p <= at) & ((p > at - swa) if swa else True)


def run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, fmt, rows, swa=0, cap=0, mask=None, where=None, ns=0, noalloc=False, cover=None):
    nh, hd = q.shape[1:]
    o = dev.buf(np.full((q.shape[0] + 1, nh, hd), 9.0, np.float32))
    scale = float(np.float32(1 / np.sqrt(hd)))
    b = [dev.paso(T, pos0), dev.buf(q), dev.buf(kc), dev.buf(vc), o]
    parts = dev.zeros(ns * q.shape[0] * nh * (4 * hd + 8)) if ns > 1 else 0
    u = [("u", hd), ("u", nh), ("u", nkv), ("u", swa), ("f", scale), ("u", cap)]
    if mask is None:
        quipu.dispatch("atencion_mx8", u + [("u", 0), ("u", 0), ("u", fmt), ("u", rows), ("u", ns)], b + [parts], (nh, cover or T), noalloc=noalloc)
    else:
        quipu.dispatch("atencion_arbol", u + [("u", fmt), ("u", rows), ("u", ns)],
                       b + [dev.buf(mask), dev.buf(where.astype(np.uint32)) if where is not None else 0, parts], (nh, cover or T), noalloc=noalloc)
    got = dev.get(o, (q.shape[0] + 1, nh, hd))
    assert np.all(got[-1] == 9.0)
    return got[:-1], scale


SHAPES = [
    (128, 8, 8, 1, 0, 0, 0),          # one key
    (64, 1, 1, 2, 0, 0, 0),           # one head
    (64, 6, 2, 5, 31, 0, 0),          # a group of 3 heads, 15 rows, keys to a tile's edge
    (128, 8, 4, 8, 1000, 0, 0),       # 16 rows, keys shared out
    (128, 10, 2, 7, 64, 0, 0),        # 35 rows: the second block of 32 nearly empty
    (64, 32, 1, 3, 500, 0, 0),        # 32 heads per KV head
    (128, 4, 2, 70, 130, 33, 0),      # a window narrower than a block, no ring
    (64, 8, 2, 24, 200, 64, 88),      # a ring of 88 slots (no multiple of 32) that the keys wrap in
    (128, 4, 4, 1, 500, 100, 132),    # one token of a ring
    (64, 4, 4, 40, 0, 64, 104),       # a ring that is not full yet
    (128, 4, 1, 300, 0, 0, 0),        # many blocks of rows
]


def ring_rows(k, v, n, pos0, swa, cap, rows, junk):
    """The rows of a cache that holds the positions below n in a ring of cap slots (or as they are), junk elsewhere: in slots
    not written, and in keys before every row's window."""
    kc, vc = (np.full((rows,) + k.shape[1:], junk) for _ in "kv")
    for p in range(max(0, n - cap) if cap else 0, n):
        if not swa or p > pos0 - swa:
            kc[p % (cap or n)], vc[p % (cap or n)] = k[p], v[p]
    return kc, vc


@pytest.mark.parametrize("hd,nh,nkv,T,pos0,swa,cap", SHAPES)
def test_attention(quipu, dev, hd, nh, nkv, T, pos0, swa, cap):
    """atencion_mx8 against float64 over what the cache holds; keys that a row does not see are NaN in the cache."""
    rng = np.random.default_rng(9)
    n = pos0 + T
    rows = cap or n + 9
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)) * 10.0 ** rng.uniform(-2, 1, (n, 1, 1)) for _ in "kv")
    kc, vc, _, _ = mx8.cache(MX8, *ring_rows(k, v, n, pos0, swa, cap, rows, np.nan))
    kh, vh = (mx8.dequantise(*mx8.quantise(x.astype(np.float32))) for x in (k, v))
    see = causal(T, pos0, swa, n)
    for ns in (0, 1, 3):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, MX8, rows, swa, cap, ns=ns)
        assert np.all(np.abs(got - mx8.attend(q, kh, vh, see, scale)) <= bound(q, kh, vh, see, scale)), ns
    got2, _ = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, MX8, rows, swa, cap, noalloc=True)
    assert np.all(np.abs(got2 - mx8.attend(q, kh, vh, see, scale)) <= bound(q, kh, vh, see, scale))


def random_tree(rng, T, full):
    """Mask words of T drafted tokens [T][ceil(T / 32)], what they see [T][T], and their depths: a random tree, or (not full)
    any sets, empty ones among them, with bits set past the T tokens."""
    see, depth = np.zeros((T, T), bool), np.zeros(T, int)
    for t in range(T):
        p = rng.integers(-1, t) if t else -1
        if full:
            if p >= 0:
                see[t], depth[t] = see[p], depth[p] + 1
            see[t, t] = True
        else:
            see[t] = rng.random(T) < 0.3
            see[t] &= t % 4 != 1
    W = (T + 31) // 32
    bits = np.zeros((T, 32 * W), np.uint64)
    bits[:, :T] = see
    if not full:
        bits[:, T:] = 1
    words = (bits.reshape(T, W, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
    return words, see, depth


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("hd,nh,nkv,T,pos0,swa,cap", [
    (128, 8, 8, 1, 0, 0, 0),          # one token without a past
    (64, 4, 2, 33, 0, 0, 0),          # a tree without a past: rows that see nothing
    (128, 8, 4, 7, 4100, 0, 0),       # a long past, shared out
    (64, 6, 2, 70, 45, 0, 0),         # three words of mask, not at a tile's edge
    (128, 32, 4, 64, 33, 0, 0),       # 512 rows
    (128, 4, 4, 20, 300, 40, 0),      # a window
    (64, 8, 2, 40, 200, 64, 110),     # a ring that the drafted tokens wrap in
])
def test_tree(quipu, dev, hd, nh, nkv, T, pos0, swa, cap, full, fmt):
    """atencion_arbol against float64.  What a row must not see is not finite in the cache: slots never written, keys before
    every window, and (not full) some drafted tokens that few rows see, which make exactly those rows' outputs NaN."""
    rng = np.random.default_rng(10)
    n = pos0 + T
    rows = cap or n + 5
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in "kv")
    mask, drafts, depth = random_tree(rng, T, full)
    where = pos0 + depth
    see = np.zeros((T, n), bool)
    see[:, pos0:] = drafts
    see[:, :pos0] = (np.arange(pos0)[None] > (where - swa)[:, None]) if swa else True
    kr, vr = ring_rows(k, v, n, pos0, swa, cap, rows, np.nan)
    kc, vc, _, _ = mx8.cache(fmt, kr, vr)
    held = [mx8.cache(fmt, x, x)[2] for x in (k, v)]
    got, scale = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, fmt, rows, swa, cap, mask, where)
    want, lim = mx8.attend(q, *held, see, scale), bound(q, *held, see, scale)
    assert np.all(np.abs(got - want) <= lim)
    assert np.all(got[~see.any(1)] == 0)
    got, _ = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, fmt, rows, swa, cap, mask, where, ns=5)
    assert np.all(np.abs(got - want) <= lim)
    if T < 3:
        return
    for kind in ("k", "v"):
        bad = [x.copy() for x in (k, v)]
        bad["kv".index(kind)][pos0 + T - 2, :, 3::64] = np.nan if kind == "k" else np.inf
        kr, vr = ring_rows(*bad, n, pos0, swa, cap, rows, np.nan)
        kc, vc, _, _ = mx8.cache(fmt, kr, vr)
        got, _ = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, fmt, rows, swa, cap, mask, where)
        hit = see[:, n - 2]
        assert np.all(np.abs(got[~hit] - want[~hit]) <= lim[~hit])
        assert not np.isfinite(got[hit][..., 3::64]).any()


def test_tree_is_causal_attention_of_a_chain(quipu, dev):
    """A chain of drafted tokens gives what atencion_mx8 gives for the same rows."""
    rng = np.random.default_rng(11)
    T, nh, nkv, hd, pos0 = 40, 8, 2, 128, 77
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((pos0 + T, nkv, hd)) for _ in "kv")
    kc, vc, _, _ = mx8.cache(MX8, k, v)
    words = np.array([[((1 << (t + 1)) - 1) >> (32 * w) & 0xffffffff for w in range(2)] for t in range(T)], np.uint32)
    a, _ = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, MX8, pos0 + T, ns=1)
    b, _ = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, MX8, pos0 + T, mask=words, ns=1)
    assert np.all(np.abs(a - b) <= 2.0 ** -18 * np.abs(v).max())


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("hd,nh,nkv,T,pos0,swa,cap", [(128, 8, 4, 24, 40, 0, 0), (64, 4, 4, 9, 300, 40, 64), (128, 6, 2, 1, 700, 600, 0)])
@pytest.mark.parametrize("kind", ["k_not_finite", "k_huge", "v_huge", "v_without_weight", "q_spread", "blocks", "zeros_first", "tiny"])
def test_unlike_magnitudes(quipu, dev, hd, nh, nkv, T, pos0, swa, cap, kind, tree):
    """Keys and values far larger or smaller than the others: a row that does not see such a key, or gives it no weight, has
    the result that it would have without it."""
    rng = np.random.default_rng(12)
    n = pos0 + T
    rows = cap or n + 9
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    q[..., 0] = 4.0
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in "kv")
    late = pos0 + T // 2  # seen by the later half only (one token: by that token)
    if kind == "k_not_finite":
        k[late, :, 5] = np.inf
    elif kind == "k_huge":
        k[late, :, 7] = 2.0 ** 60
    elif kind == "v_huge":
        v *= 1e-3
        v[late] = 2.0 ** 60
    elif kind == "v_without_weight":
        v *= 1e-3
        v[pos0 - 3] = 2.0 ** 60
        k[pos0 - 3] = 0
        k[pos0 - 3, :, 0] = -3000
    elif kind == "blocks":  # magnitudes that change forth and back along the keys
        k[::37] *= 1e-6
        v[n // 2:n // 2 + 200] *= 1e-7
    elif kind == "zeros_first":
        k[:n // 2], v[:n // 2] = 0, 0
    elif kind == "tiny":
        v *= 1e-30
        k *= 1e-20
        q *= np.float32(1e18)
    else:
        q[T // 2:, :, 3] *= np.float32(2.0 ** 30)
        k[:, :, 3] = 0
    kc, vc, _, _ = mx8.cache(MX8, *ring_rows(k, v, n, pos0, swa, cap, rows, np.nan))
    kh, vh = (mx8.dequantise(*mx8.quantise(x.astype(np.float32))) for x in (k, v))
    see = causal(T, pos0, swa, n)
    mask = where = None
    if tree:
        mask = np.array([[(1 << (t + 1)) - 1] for t in range(T)], np.uint32)
        where = pos0 + np.arange(T)
    got, scale = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, MX8, rows, swa, cap, mask, where)
    for t in range(T):
        on = np.flatnonzero(see[t])
        for h in range(nh):
            kk, vv = kh[on, h * nkv // nh], vh[on, h * nkv // nh]
            s = kk @ q[t, h].astype(np.float64) * scale
            if not np.isfinite(s).all():
                assert not np.isfinite(got[t, h]).any(), (t, h)
                continue
            w = np.exp(s - s.max())
            w /= w.sum()
            near = w > 1e-36  # (below it a weight is 0 in float32)
            e = 2.0 ** -20 * (np.abs(kk[near]) @ np.abs(q[t, h].astype(np.float64))).max() * scale
            assert np.all(np.abs(got[t, h] - w[near] @ vv[near]) <= (2 * e + 2.0 ** -19) * np.abs(vv[near]).max()), (t, h)


def test_tokens_past_the_dispatch(quipu, dev):
    """A Paso of more tokens than the dispatch covers: the others' outputs stay as they were."""
    rng = np.random.default_rng(13)
    q = rng.standard_normal((9, 2, 64)).astype(np.float32)
    k, v = (rng.standard_normal((600, 1, 64)) for _ in "kv")
    kc, vc, _, _ = mx8.cache(MX8, k, v)
    got, _ = run_attention(quipu, dev, q, kc, vc, 9, 500, 1, MX8, 600, cover=2)
    assert np.all(got[2:] == 9.0) and not np.any(got[:2] == 9.0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,nkv,T,pos0,rows,cap,idx,layers", [
    (128, 8, 64, 333, 400, 0, [0, 3, 9, 17, 40, 63], 3), (64, 1, 2, 0, 2, 0, [1], 1), (64, 3, 30, 31, 61, 0, list(range(1, 30)), 2),
    (128, 2, 20, 75, 51, 51, [2, 3, 8, 11, 12, 13, 17, 18, 19], 2), (64, 2, 5, 10, 20, 0, [0, 1, 2], 64)])
def test_path(quipu, dev, fmt, hd, nkv, T, pos0, rows, cap, idx, layers):
    """kv_ramal moves the rows, in every layer, and nothing else."""
    rng = np.random.default_rng(14)
    n = mx8.nbytes(fmt, rows, nkv, hd)
    R, kvd = mx8.slots32(rows), nkv * hd
    caches, hs = [], []
    for _ in range(layers):
        k, v = (rng.standard_normal((rows, nkv, hd)) for _ in "kv")
        kc, vc, kh, vh = mx8.cache(fmt, k, v)
        caches.append((kh, vh))
        hs += [dev.buf(kc), dev.buf(vc)]
    raw = [dev.get(h, (rows * kvd * (4 if fmt == F32 else 2) if fmt != MX8 else n,), np.uint8) for h in hs]
    quipu.dispatch("kv_ramal", [("u", hd), ("u", nkv), ("u", cap), ("u", fmt), ("u", rows), ("u", len(idx))],
                   [dev.paso(T, pos0), dev.buf(np.array(idx, np.uint32))] + hs, (len(idx),))
    for i, (kh, vh) in enumerate(caches):
        gk, gv = read(quipu, dev, (hs[2 * i], hs[2 * i + 1]), nkv, hd, fmt, rows, 0, rows)
        src, dst = ((pos0 + np.array(x)) % (cap or 1 << 30) for x in (idx, range(len(idx))))
        for got, x in ((gk, kh), (gv, vh)):
            want = x.copy()
            want[dst] = x[src]
            assert np.array_equal(got, want.astype(np.float32))
    if fmt == MX8:  # slots past the rows hold what they held
        got = dev.get(hs[0], (n,), np.uint8)
        assert np.array_equal(got[nkv * R * hd:].reshape(nkv, R, hd // 32)[:, rows:], raw[0][nkv * R * hd:].reshape(nkv, R, hd // 32)[:, rows:])


def test_path_beyond_the_tree_moves_nothing(quipu, dev):
    """Indices past the drafted tokens, and slots past the cache, are left out."""
    rng = np.random.default_rng(15)
    k, v = (rng.standard_normal((20, 1, 64)) for _ in "kv")
    kc, vc, kh, vh = mx8.cache(F32, k, v)
    hs = dev.buf(kc), dev.buf(vc)
    quipu.dispatch("kv_ramal", [("u", 64), ("u", 1), ("u", 0), ("u", F32), ("u", 20), ("u", 3)],
                   [dev.paso(6, 15), dev.buf(np.array([2, 5, 9], np.uint32)), *hs], (3,))
    want = kh.copy()
    want[15] = kh[17]   # (15 + 5 lies past the cache, 9 past the tree)
    assert np.array_equal(read(quipu, dev, hs, 1, 64, F32, 20, 0, 20)[0], want.astype(np.float32))


@pytest.mark.parametrize("fmt", FMTS)
def test_a_tree_pass_in_two_graphs(quipu, dev, fmt):
    """Store, tree attention (its shares in a buffer of the graph's own) and the path, captured twice with other trees, and
    replayed in turn with eager work between: every replay gives the eager results."""
    rng = np.random.default_rng(16)
    T, nh, nkv, hd, pos0 = 12, 8, 2, 128, 700
    rows, scale = pos0 + T + 4, float(np.float32(1 / np.sqrt(hd)))
    k0, v0 = (rng.standard_normal((rows, nkv, hd)) for _ in "kv")
    kc0, vc0, _, _ = mx8.cache(fmt, k0, v0)
    paso, freq = dev.paso(T, pos0), dev.buf(table(hd))

    def build(seed):
        r = np.random.default_rng(seed)
        mask, _, depth = random_tree(r, T, True)
        b = {n: dev.buf(r.standard_normal((T, h, hd)).astype(np.float32)) for n, h in (("q", nh), ("k", nkv), ("v", nkv))}
        b.update(qo=dev.zeros(4 * T * nh * hd), o=dev.zeros(4 * T * nh * hd), kc=dev.buf(kc0), vc=dev.buf(vc0), mask=dev.buf(mask),
                 pos=dev.buf((pos0 + depth).astype(np.uint32)), parts=dev.zeros(4 * T * nh * (4 * hd + 8)),
                 idx=dev.buf(np.array([0, 2, 5, 11], np.uint32)))

        def go():
            quipu.dispatch("norm_rope_kv", [("u", hd), ("u", nh), ("u", nkv), ("u", 0), ("f", 1e-6), ("u", hd), ("f", 0), ("u", 0), ("u", fmt), ("u", rows)],
                           [paso, b["q"], b["k"], b["v"], b["qo"], b["kc"], b["vc"], 0, 0, freq, b["pos"]], (nh, T))
            quipu.dispatch("atencion_arbol", [("u", hd), ("u", nh), ("u", nkv), ("u", 0), ("f", scale), ("u", 0), ("u", fmt), ("u", rows), ("u", 4)],
                           [paso, b["qo"], b["kc"], b["vc"], b["o"], b["mask"], b["pos"], b["parts"]], (nh, T))
            quipu.dispatch("kv_ramal", [("u", hd), ("u", nkv), ("u", 0), ("u", fmt), ("u", rows), ("u", 4)], [paso, b["idx"], b["kc"], b["vc"]], (4,))

        def out():
            n = kc0.nbytes
            return [dev.get(b["o"], (T, nh, hd)), dev.get(b["kc"], (n,), np.uint8), dev.get(b["vc"], (vc0.nbytes,), np.uint8)]
        return b, go, out

    two = [build(s) for s in (21, 22)]
    want, graphs = [], []
    for b, go, out in two:
        go()
        want.append(out())
        quipu.upload(b["kc"], kc0)
        quipu.upload(b["vc"], vc0)
        quipu.graph_begin()
        try:
            go()
        finally:
            graphs.append(quipu.graph_end())
    try:
        for step in range(4):
            b, go, out = two[step % 2]
            quipu.upload(b["kc"], kc0)
            quipu.upload(b["vc"], vc0)
            quipu.upload(b["o"], np.zeros((T, nh, hd), np.float32))
            quipu.graph_launch(graphs[step % 2])
            for g, w in zip(out(), want[step % 2]):
                assert np.array_equal(g, w), step
            run_attention(quipu, dev, np.ones((3, nh, hd), np.float32), kc0, vc0, 3, 300, nkv, fmt, rows,
                          mask=np.full((3, 1), 7, np.uint32))   # eager work in the library's workspace
    finally:
        for g in graphs:
            quipu.graph_free(g)


def test_one_share_while_capturing(quipu, dev):
    """Without a buffer for the shares a captured atencion_mx8 takes one share; its replays give its eager result."""
    rng = np.random.default_rng(17)
    nh, nkv, hd, pos0 = 4, 1, 64, 900
    q = rng.standard_normal((1, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((pos0 + 1, nkv, hd)) for _ in "kv")
    kc, vc, _, _ = mx8.cache(MX8, k, v)
    want, scale = run_attention(quipu, dev, q, kc, vc, 1, pos0, nkv, MX8, pos0 + 1, ns=1)
    o = dev.zeros(4 * nh * hd)
    b = [dev.paso(1, pos0), dev.buf(q), dev.buf(kc), dev.buf(vc), o]
    quipu.graph_begin()
    try:
        quipu.dispatch("atencion_mx8", [("u", hd), ("u", nh), ("u", nkv), ("u", 0), ("f", scale), ("u", 0), ("u", 0), ("u", 0), ("u", MX8), ("u", pos0 + 1)], b, (nh, 1))
    finally:
        g = quipu.graph_end()
    try:
        for _ in range(3):
            quipu.upload(o, np.zeros(nh * hd, np.float32))
            quipu.graph_launch(g)
            assert np.array_equal(dev.get(o, (1, nh, hd)), want)
    finally:
        quipu.graph_free(g)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("power", [19, 20, 21, 22, 23, 24, 25, 26, 27, 28, 40])
def test_scores_past_their_last_place(quipu, dev, power, wide):
    """Scores around 2^power, in units of log2, that grow by 15.5 from tile to tile, where the sum of a score and a few units is
    rounded by more than a unit.  Each tile has one key whose score is not -2^power.  A row's largest score leads the others by
    15.5 less the rounding of both (2^-22 of 2^power together: two sums of products, two products with the unit), so that its
    key's value is the output up to 2^(that - 15.5) (1 + 2^-15) of two values' difference."""
    hd, nh, nkv = 128, 32 if wide else 4, 8 if wide else 1
    T, n = (256, 4224) if wide else (1, 160)
    pos0 = n - T
    rng = np.random.default_rng(power)
    k, v = np.zeros((n, nkv, hd)), rng.standard_normal((n, nkv, hd)).astype(np.float32)
    q = np.zeros((T, nh, hd), np.float32)
    per = np.sqrt(hd) * np.log(2.0)  # q k of one unit of log2
    tile = np.arange(n) // 32
    # three blocks of channels: 2^power, then 15.5 for each tile of 64, then 15.5 for each 64 tiles
    q[..., 0], q[..., 32], q[..., 64] = 2.0 ** (power - 14) * per, 15.5 * per, 15.5 * per
    k[:, :, 0], k[:, :, 32], k[:, :, 64] = -(2.0 ** 14), (tile % 64)[:, None], 64 * (tile // 64)[:, None]
    k[5::32, :, 0] = 2.0 ** 14
    kc, vc, _, held = mx8.cache(mx8.MX8, k, v)
    o, _ = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, mx8.MX8, n)
    last = (pos0 + np.arange(T) - 5) // 32 * 32 + 5  # the last key with a score that the token sees
    want = held[last][:, np.arange(nh) * nkv // nh]
    most = np.abs(held).max()
    off = 2.0 ** (power - 22)
    if off < 15:
        assert np.all(np.abs(o - want) <= 2.0 ** (off - 15.5) * 1.01 * 2 * most + 1e-5), np.abs(o - want).max()
    assert np.isfinite(o).all() and np.abs(o).max() <= most * (1 + 1e-5)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T", [1, 40])
def test_keys_and_queries_in_the_thousands(quipu, dev, T, fmt):
    """Scores up to 1e9, as the keys and queries of some models make them: nearly one key for each row.  A score is off by 2^-20
    of the sum of its products' magnitudes; rows whose two largest differ by less are within the values, and not compared."""
    hd, nh, nkv, n = 128, 8, 2, 500
    rng = np.random.default_rng(T)
    q = (rng.standard_normal((T, nh, hd)) * 5000).astype(np.float32)
    k, v = rng.standard_normal((n, nkv, hd)) * 5000, rng.standard_normal((n, nkv, hd)) * 1000
    kc, vc, kh, vh = mx8.cache(fmt, k, v)
    see = causal(T, n - T, 0, n)
    mask = np.zeros((T, (T + 31) // 32), np.uint32)
    for t in range(T):
        for j in range(t + 1):
            mask[t, j // 32] |= np.uint32(1 << (j % 32))
    o, scale = run_attention(quipu, dev, q, kc, vc, T, n - T, nkv, fmt, n, mask=mask)
    want = mx8.attend(q.astype(np.float64), kh, vh, see, scale)
    kk = np.repeat(kh, nh // nkv, 1)
    scores = np.einsum("thc,nhc->thn", q.astype(np.float64), kk) * scale
    size = np.einsum("thc,nhc->thn", np.abs(q).astype(np.float64), np.abs(kk)) * scale
    top = np.sort(np.where(see[:, None], scores, -np.inf), -1)
    clear = top[..., -1] - top[..., -2] > size.max() * 2.0 ** -20 + 20
    assert clear.mean() > 0.9
    most = np.abs(vh).max()
    assert np.all(np.abs(o - want)[clear] <= 1e-5 * most)
    assert np.isfinite(o).all() and np.abs(o).max() <= most * (1 + 1e-5)


def sampled(rng, T, most=20):
    """Some of T rows: the first, the last, those at the edges of blocks, others."""
    edges = [x for x in (0, 1, 15, 16, 31, 32, 33, T // 2, T - 2, T - 1) if 0 <= x < T]
    return np.unique(np.concatenate([edges, rng.integers(0, T, most - 10)])).astype(int)


@pytest.mark.parametrize("hd,nh,nkv,T,pos0,swa,cap", [
    (128, 32, 8, 256, 4200, 0, 0),      # blocks of 16 rows
    (128, 32, 8, 256, 5300, 0, 0),      # blocks of 128 rows and shares of the keys
    (128, 32, 8, 1100, 0, 0, 0),        # blocks of 128 rows, the last with 48, no shares
    (64, 24, 8, 1500, 37, 0, 0),        # groups of 3 heads: blocks that begin inside a token
    (64, 32, 8, 1100, 3000, 300, 1500), # a ring
    (128, 16, 16, 700, 9000, 1024, 0),  # a window, no ring, shares
    (128, 12, 4, 90, 9000, 0, 0),       # blocks of 16 rows, many shares
])
def test_attention_over_many_blocks(quipu, dev, hd, nh, nkv, T, pos0, swa, cap):
    """As test_attention, the rows of some tokens, where launches are large."""
    rng = np.random.default_rng(19)
    n = pos0 + T
    rows = cap or n + 9
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)) * 10.0 ** rng.uniform(-2, 1, (n, 1, 1)) for _ in "kv")
    kc, vc, _, _ = mx8.cache(MX8, *ring_rows(k, v, n, pos0, swa, cap, rows, np.nan))
    kh, vh = (mx8.dequantise(*mx8.quantise(x.astype(np.float32))) for x in (k, v))
    some = sampled(rng, T)
    see = causal(T, pos0, swa, n)[some]
    for noalloc in (False, True):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, MX8, rows, swa, cap, noalloc=noalloc)
        assert np.all(np.abs(got[some] - mx8.attend(q[some], kh, vh, see, scale)) <= bound(q[some], kh, vh, see, scale)), noalloc
        assert np.isfinite(got).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,nh,nkv,T,pos0,swa,cap", [
    (128, 32, 8, 128, 10400, 0, 0),     # 512 rows: blocks of 128 (8 bits), of 32 (f32, f16), shares
    (64, 16, 16, 300, 9000, 600, 0),    # a window, ten words of mask
])
def test_tree_over_many_blocks(quipu, dev, hd, nh, nkv, T, pos0, swa, cap, fmt):
    """As test_tree, the rows of some tokens, where launches are large."""
    rng = np.random.default_rng(20)
    n = pos0 + T
    rows = n + 5
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in "kv")
    mask, drafts, depth = random_tree(rng, T, True)
    where = pos0 + depth
    some = sampled(rng, T)
    see = np.zeros((T, n), bool)
    see[:, pos0:] = drafts
    see[:, :pos0] = (np.arange(pos0)[None] > (where - swa)[:, None]) if swa else True
    for bad in (False, True):
        if bad:  # a drafted token whose value is not finite, seen by few
            v[pos0 + T // 3, :, 5::64] = np.inf
        kc, vc, _, _ = mx8.cache(fmt, *ring_rows(k, v, n, pos0, swa, cap, rows, np.nan))
        if not bad:
            held = [mx8.cache(fmt, x, x)[2] for x in (k, v)]
        got, scale = run_attention(quipu, dev, q, kc, vc, T, pos0, nkv, fmt, rows, swa, cap, mask, where)
        want, lim = mx8.attend(q[some], *held, see[some], scale), bound(q[some], *held, see[some], scale)
        hit = see[:, pos0 + T // 3] & bad
        assert np.all(np.abs(got[some] - want)[~hit[some]] <= lim[~hit[some]])
        assert np.isfinite(got[~hit]).all() and not np.isfinite(got[hit][..., 5::64]).any()


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("T,cover,pos0", [(3, 40, 200), (1, 2, 0), (100, 300, 4000)])
def test_rows_past_the_tokens_may_hold_anything(quipu, dev, T, cover, pos0, tree):
    """A call for `cover` tokens of which the Paso has T: the queries behind them are NaN, and their outputs stay as they were."""
    hd, nh, nkv, n = 128, 16, 4, pos0 + T
    rng = np.random.default_rng(21)
    q = np.full((cover, nh, hd), np.nan, np.float32)
    q[:T] = rng.standard_normal((T, nh, hd))
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in "kv")
    kc, vc, kh, vh = mx8.cache(MX8, k, v)
    rows = pos0 + cover + 9
    pad = lambda x: np.concatenate([x, np.zeros((rows - n, nkv, hd))])   # noqa: E731
    grown = mx8.cache(MX8, pad(k), pad(v))[:2]
    mask = np.zeros((cover, (cover + 31) // 32), np.uint32)
    for t in range(cover):
        for j in range(t + 1):
            mask[t, j // 32] |= np.uint32(1 << (j % 32))
    got, scale = run_attention(quipu, dev, q, *grown, T, pos0, nkv, MX8, rows, mask=mask if tree else None, cover=cover)
    see = causal(T, pos0, 0, n)
    assert np.all(np.abs(got[:T] - mx8.attend(q[:T], kh, vh, see, scale)) <= bound(q[:T], kh, vh, see, scale))
    assert np.all(got[T:] == 9.0)


@pytest.mark.parametrize("rows", [1, 2, 7])
@pytest.mark.parametrize("n", [1, 1000, 128256])
def test_argmax_of_rows(quipu, dev, rows, n):
    rng = np.random.default_rng(n)
    v = rng.standard_normal((rows, n)).astype(np.float32)
    v[:, n // 2] = v[:, n - 1] = 9.0   # ties: the lowest index
    v[:, 0] = np.nan if n > 1 else v[:, 0]
    out = dev.buf(np.full(rows + 1, 77, np.uint32))
    quipu.dispatch("argmax", [("u", n), ("u", rows)], [0, dev.buf(v), out])
    got = dev.get(out, (rows + 1,), np.uint32)
    assert got[:rows].tolist() == [n // 2] * rows and got[rows] == 77


@pytest.mark.parametrize("T,n,nh,nkv", [(1, 90, 4, 1), (1, 3000, 8, 2), (24, 900, 8, 2), (260, 5600, 32, 8)])
def test_values_near_the_largest(quipu, dev, T, n, nh, nkv):
    """Values up to 2^127: sums of probabilities times values leave f32's range, the outputs do not."""
    hd = 128
    rng = np.random.default_rng(22)
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = rng.standard_normal((n, nkv, hd)), rng.uniform(0.5, 1, (n, nkv, hd)) * 2.0 ** 127
    k[::7] *= 3
    kc, vc, kh, vh = mx8.cache(MX8, k, v)
    some = sampled(rng, T)
    see = causal(T, n - T, 0, n)[some]
    for ns in (0, 1):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, n - T, nkv, MX8, n, ns=ns)
        assert np.isfinite(got).all()
        assert np.all(np.abs(got[some] - mx8.attend(q[some], kh, vh, see, scale)) <= bound(q[some], kh, vh, see, scale))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,nh,nkv,T,pos0,nrot,neox,norm,cap", [
    (128, 30, 7, 400, 11, 128, 0, 1, 0),      # groups of four with two and three heads in the last ones
    (128, 30, 7, 403, 0, 128, 1, 1, 450),     # halves apart (through LDS), a ring
    (64, 27, 5, 901, 5, 64, 1, 1, 0),         # two tokens for each wavefront, the last alone; three and one heads
    (64, 27, 5, 950, 1000, 22, 0, 0, 951),
    (128, 1, 31, 301, 3, 34, 1, 0, 0),        # one head of q
    (64, 33, 16, 700, 77, 0, 0, 1, 0),        # norms alone
])
def test_stores_of_many_tokens(quipu, dev, fmt, hd, nh, nkv, T, pos0, nrot, neox, norm, cap):
    """As test_rotation, with tokens enough that a wavefront takes four heads (64 wavefronts for each of 256 CUs); the rows
    behind the Paso's tokens stay as they were."""
    assert T * (nh + 2 * nkv) * hd // 128 >= 64 * 256
    rng = np.random.default_rng(23)
    q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) for h in (nh, nkv, nkv))
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in "qk") if norm else (None, None)
    rows = cap or pos0 + T + 3
    n = T - 5  # the Paso's
    qo, kc, vc, hs = store(quipu, dev, q, k, v, pos0, rows, fmt, cap, neox, nrot, qn, kn, T=n, fill=0)
    pos = pos0 + np.arange(T)
    want, size = rotate(q, qn, pos, nrot, neox)
    assert np.all(np.abs(qo - want)[:n] <= ROT * size[:n]) and np.all(qo[n:] == 7.0)
    gk, gv = (x.astype(np.float64) for x in read(quipu, dev, hs, nkv, hd, fmt, rows, pos0, n, cap))
    want, size = (x[:n] for x in rotate(k, kn, pos, nrot, neox))
    if fmt == F32:
        assert np.all(np.abs(gk - want) <= ROT * size) and np.array_equal(gv, v[:n])
    elif fmt == F16:
        assert np.all(np.abs(gk - want) <= ROT * size + 2.0 ** -11 * np.abs(want) + 2.0 ** -25)
        assert np.array_equal(gv, v[:n].astype(np.float16))
    else:
        step = 2.0 ** (mx8.quantise(want.astype(np.float32))[1].astype(np.float64) - 133).repeat(32, -1)
        assert np.all(np.abs(gk - want) <= 0.5 * step + 2 * ROT * size + 0.5 * step * (np.abs(want) > 63 * step))
        assert np.array_equal(gv, mx8.dequantise(*mx8.quantise(v[:n])))
    inplace = store(quipu, dev, q, k, v, pos0, rows, fmt, cap, neox, nrot, qn, kn, T=n, inplace=True)[0]
    assert np.array_equal(inplace[:n], qo[:n]) and np.array_equal(inplace[n:], q[n:])
