"""The 8-bit cache in numpy, written from its definition: blocks of 32 channels of a token's head, value = q 2^(x - 133),
q within +-127 held as the byte q + 128, x the smallest byte for which the block's largest magnitude times 2^(133 - x) lies
below 127.5; x = 255: a value of the block was not finite, and all of it is NaN.  And the three layouts of a cache."""
import numpy as np

F32, F16, MX8 = 0, 1, 2


def quantise(x):
    """x [..., c] f32 -> (bytes [..., c], scales [..., c / 32])."""
    b = np.asarray(x, np.float64).reshape(x.shape[:-1] + (-1, 32))
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(b).max(-1)
        bad = ~np.isfinite(top)
        m = np.where(bad, 0, top)
        # 127.5 2^(x - 133) for every x; the first one above m
        limits = 127.5 * 2.0 ** (np.arange(255) - 133.0)
        e = np.searchsorted(limits, m, side="right")
        q = np.rint(np.where(bad[..., None], 0, b) * 2.0 ** (133.0 - e)[..., None])
    return (q + 128).astype(np.uint8).reshape(x.shape), np.where(bad, 255, e).astype(np.uint8)


def dequantise(q, e):
    s = np.where(e == 255, np.nan, 2.0 ** (e.astype(np.float64) - 133.0))
    return ((q.reshape(q.shape[:-1] + (-1, 32)).astype(np.float64) - 128) * s[..., None]).reshape(q.shape)


def slots32(rows):
    return (rows + 31) // 32 * 32


def k_bytes(q, e):
    """Rows [rows][nkv][hd] bytes, [rows][nkv][hd / 32] scales (rows a multiple of 32) -> the K cache's bytes."""
    R, nkv, hd = q.shape
    t = q.reshape(R // 32, 2, 16, nkv, hd // 64, 4, 16).transpose(3, 0, 1, 4, 5, 2, 6)
    return np.concatenate([t.ravel(), e.transpose(1, 0, 2).ravel()])


def v_bytes(q, e):
    R, nkv, hd = q.shape
    t = q.reshape(R // 32, 2, 4, 4, nkv, 16, hd // 32, 2)   # tile, a, g, b, head, n, i, e
    s = e.reshape(R // 32, 2, 4, 4, nkv, hd // 32)
    return np.concatenate([t.transpose(4, 0, 6, 2, 5, 7, 1, 3).ravel(), s.transpose(4, 0, 5, 2, 1, 3).ravel()])


def cache(fmt, k, v):
    """Rows [rows][nkv][hd] of K and V as the two caches' memory, and the values that they hold ([rows][nkv][hd] float64)."""
    import refs
    rows, nkv, hd = k.shape
    kvd = nkv * hd
    with np.errstate(over="ignore", invalid="ignore"):
        if fmt == MX8:
            pad = ((0, slots32(rows) - rows), (0, 0), (0, 0))
            out, held = [], []
            for x, lay in ((k, k_bytes), (v, v_bytes)):
                q, e = quantise(x.astype(np.float32))
                held.append(dequantise(q, e))
                # slots past the rows hold anything: the largest bytes
                out.append(lay(np.pad(q, pad, constant_values=255), np.pad(e, pad, constant_values=255)))
            return out[0], out[1], held[0], held[1]
        if fmt == F16:
            kh, vh = k.astype(np.float16).reshape(rows, kvd), v.astype(np.float16).reshape(rows, kvd)
            return kh, refs.v_tiled(vh, kvd), *(a.astype(np.float64).reshape(k.shape) for a in (kh, vh))
    kf, vf = k.astype(np.float32), v.astype(np.float32)
    return kf, vf, kf.astype(np.float64), vf.astype(np.float64)


def nbytes(fmt, rows, nkv, hd):
    if fmt == MX8:
        return slots32(rows) * nkv * (hd + hd // 32)
    return slots32(rows) * nkv * hd * (2 if fmt == F16 else 4)


def attend(q, k, v, see, scale):
    """q [T][nh][hd], k, v [n][nkv][hd], see [T][n] -> [T][nh][hd] float64; a row that sees nothing is 0."""
    T, nh, hd = q.shape
    o = np.zeros((T, nh, hd))
    for t in range(T):
        on = np.flatnonzero(see[t])
        if not len(on):
            continue
        for h in range(nh):
            kk, vv = k[on, h * k.shape[1] // nh], v[on, h * k.shape[1] // nh]
            s = kk @ q[t, h].astype(np.float64) * scale
            w = np.exp(s - s.max())
            o[t, h] = (w / w.sum()) @ vv
    return o
