"""Attention over 8-bit caches and drafted trees where magnitudes lie far apart or near float32's largest: outputs that are
finite stay finite, and a row has the precision that it would have without the keys that it gives no weight.

Tolerances.  A score is a sum of hd products added one by one at worst (the float32 matrix instructions): off by at most
e = 2^-24 hd sum |q k| scale.  An output is a sum over the keys seen, each added with a rounding, and its state is met with
others and moved from tile to tile with at most 4 roundings each: (2 e + (2 n + 256) 2^-24) max |v| for n keys, max |v| over the
keys whose weight float32 holds."""
import numpy as np
import pytest

import mx8
from mx8 import F32, MX8
from test_gpu_cache import causal, run_attention, sampled
from test_gpu_ops import dev  # noqa: F401

pytestmark = pytest.mark.gpu


def chain(T):
    """The mask of a chain of T drafted tokens."""
    W = (T + 31) // 32
    return np.array([[((1 << (t + 1)) - 1) >> (32 * w) & 0xffffffff for w in range(W)] for t in range(T)], np.uint32)


def check(got, q, kh, vh, see, scale, rows):
    """Rows `rows` of got against float64 over the held keys and values; a row that sees a NaN key is NaN."""
    nh, hd, nkv = q.shape[1], q.shape[2], kh.shape[1]
    worst = 0.0
    for t in rows:
        on = np.flatnonzero(see[t])
        for h in range(nh):
            kk, vv = kh[on, h * nkv // nh], vh[on, h * nkv // nh]
            if np.isnan(kk).any():
                assert np.isnan(got[t, h]).all(), (t, h)
                continue
            s = kk @ q[t, h].astype(np.float64) * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            near = w > 1e-36
            e = 2.0 ** -24 * hd * (np.abs(kk[near]) @ np.abs(q[t, h].astype(np.float64))).max() * scale
            lim = (2 * e + (2 * len(on) + 256) * 2.0 ** -24) * np.abs(vv[near]).max()
            assert np.isfinite(got[t, h]).all(), (t, h)
            off = np.abs(got[t, h] - w[near] @ vv[near]).max()
            assert off <= lim, (t, h, off, lim)
            worst = max(worst, off / lim)
    print("largest part of the tolerance: %.3g" % worst, flush=True)


SMALL, WIDE = (24, 90, 8, 2), (1040, 1100, 32, 8)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,n,nh,nkv", [SMALL, WIDE, (1, 3000, 8, 2)])
@pytest.mark.parametrize("kind", ["beside_ones", "nan_key"])
def test_values_near_the_largest_in_f32(quipu, dev, T, n, nh, nkv, hd, kind, tree):
    """Values up to 2^127 on the path that computes in float32: beside values around 1 in every tile, and behind a key that is
    not finite and that only the later half of the rows see."""
    rng = np.random.default_rng(31)
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = rng.standard_normal((n, nkv, hd)), rng.uniform(0.5, 1, (n, nkv, hd)) * 2.0 ** 127
    if kind == "beside_ones":
        v[1::2] = rng.standard_normal((len(v[1::2]), nkv, hd))
    elif T > 1:
        k[n - T // 2, :, 5] = np.nan
    kc, vc, kh, vh = mx8.cache(MX8, k, v)
    see = causal(T, n - T, 0, n)
    for ns in (0, 1, 5):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, n - T, nkv, MX8, n, ns=ns, mask=chain(T) if tree else None)
        check(got, q, kh, vh, see, scale, sampled(rng, T))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["falling", "rising_without_weight"])
@pytest.mark.parametrize("T,n,nh,nkv,run", [(24, 1700, 8, 2, 512), (1, 1300, 4, 1, 384), (1040, 1500, 32, 8, 128), (1, 100000, 4, 2, 8192)])
def test_values_that_move_the_scale_again_and_again(quipu, dev, T, n, nh, nkv, run, kind, hd, tree):
    """Values whose magnitudes fall by 2^54 three times along the keys, and ones that rise so from keys that alone have weight:
    each step is one that the sums bear, all together are not."""
    rng = np.random.default_rng(32)
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in "kv")
    level = np.minimum(np.arange(n) // run, 3)
    if kind == "falling":
        v *= 2.0 ** (100 - 54.0 * level)[:, None, None]
    else:
        v *= 2.0 ** (-100 + 54.0 * level)[:, None, None]
        q[..., 0] = 4
        k[:, :, 0] = np.where(level > 0, -3000, 0)[:, None]
        k[level > 0, :, 1:32] = 0
    kc, vc, kh, vh = mx8.cache(MX8, k, v)
    see = causal(T, n - T, 0, n)
    for ns in (1, 0):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, n - T, nkv, MX8, n, ns=ns, mask=chain(T) if tree else None)
        check(got, q, kh, vh, see, scale, sampled(rng, T))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,n,nh,nkv", [(1, 3, 1, 1), (1, 90, 4, 1), (24, 900, 8, 2), (100, 4000, 16, 8)])
@pytest.mark.parametrize("kind", ["alike", "beside_ones", "nan_key"])
@pytest.mark.parametrize("fmt", [F32, MX8])
def test_tree_values_near_the_largest(quipu, dev, fmt, T, n, nh, nkv, kind, hd):
    """atencion_arbol over values up to 2^127: sums of probabilities times values leave float32's range, the outputs do not."""
    rng = np.random.default_rng(33)
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    k, v = rng.standard_normal((n, nkv, hd)), rng.uniform(0.5, 1, (n, nkv, hd)) * 2.0 ** 127
    if n == 3:
        k[:] = 0
    if kind == "beside_ones":
        v[1::2] = rng.standard_normal((len(v[1::2]), nkv, hd))
    elif kind == "nan_key" and T > 1:
        k[n - T // 2, :, 5] = np.nan
    kc, vc, kh, vh = mx8.cache(fmt, k, v)
    see = causal(T, n - T, 0, n)
    for ns in (0, 1, 5):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, n - T, nkv, fmt, n, ns=ns, mask=chain(T))
        check(got, q, kh, vh, see, scale, sampled(rng, T))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,n,nh,nkv", [(24, 90, 8, 2), (1, 500, 4, 1), (1040, 1100, 32, 8)])
@pytest.mark.parametrize("op,fmt", [("mx8", MX8), ("tree", MX8), ("tree", F32)])
def test_magnitudes_whose_product_float32_does_not_hold(quipu, dev, op, fmt, T, n, nh, nkv, hd):
    """Queries of 2^40 in channels where the keys are 0, keys of 2^121 in channels where the queries are 0: scores of 0.  And
    one key with a score of 2^40."""
    rng = np.random.default_rng(34)
    q, k, v = np.zeros((T, nh, hd), np.float32), np.zeros((n, nkv, hd)), rng.standard_normal((n, nkv, hd))
    q[..., 0:hd:32], k[..., 1:hd:32] = 2.0 ** 40, 2.0 ** 121
    if fmt == MX8:
        k[..., 0:32] = 0
        q[..., 32:] = 0
    if T == 1:
        k[n // 2] = 0
        k[n // 2, :, 0] = 1
    kc, vc, kh, vh = mx8.cache(fmt, k, v)
    see = causal(T, n - T, 0, n)
    for ns in (0, 1, 5):
        got, scale = run_attention(quipu, dev, q, kc, vc, T, n - T, nkv, fmt, n, ns=ns, mask=chain(T) if op == "tree" else None)
        check(got, q, kh, vh, see, scale, sampled(rng, T))
