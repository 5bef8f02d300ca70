"""Operators of the 8-bit cache and of drafted trees, as cases that can be timed and compared.

A pass is one of

  store   norm_rope_kv, then kv_read of the rows just written: queries and keys normed per head, rotated and, with the
          values, stored into the cache (f32, f16 or 8-bit blocks), and read back
  attend  atencion_mx8: causal attention over the 8-bit cache, from one token to prompt chunks, windows on rings
  tree    atencion_arbol: a tree of drafted tokens over a cache of any type
  path    kv_ramal: the rows of a tree's accepted path moved to consecutive slots, in all layers' caches; 8-bit caches are
          read back with kv_read

`own` chooses between the backend's ops and their plain form in torch operations.
The ops run on the backend's own stream: the first pass over a state waits for what torch was asked for before, and a caller
waits for the device before torch reads what a pass gave or changes what it reads.

Cache layouts (R slots: the rows rounded up to 32; a tile is 32 slots).
  f32  K and V [slot][nkv hd]
  f16  K [slot][nkv hd]; V [tile][nkv hd][32], slot 16 a + 4 g + b of a tile at place 8 g + 4 a + b
  mx8  blocks of 32 channels of a token's head: value = q 2^(x - 133), q within +-127 and held as the byte q + 128, x the
       smallest byte for which the block's largest magnitude times 2^(133 - x) is below 127.5; 255: a value was not finite.
       K [nkv][tile][slot / 16][channel / 64][channel % 64 / 16][slot % 16][channel % 16], then x [nkv][slot][hd / 32]
       V [nkv][tile][i][g][n][e][a][b]: channel hd / 16 n + 2 i + e, slot 16 a + 4 g + b; x [nkv][tile][hd / 32][g][a][b]
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

F32, F16, MX8 = 0, 1, 2
EPS = 1e-6

_8B = dict(nh=32, nkv=8, hd=128)
_MOE = dict(nh=32, nkv=4, hd=128)
_WIN = dict(nh=16, nkv=8, hd=128)
_TINY = dict(nh=16, nkv=16, hd=64)


def listed():
    return [
        # one decoded token of the 8B shape: rotated and stored, all launch latency
        dict(kind="store", **_8B, T=1, pos=4100, rows=4400, fmt=MX8, neox=0, norm=0, name="store_1_8b_mx8"),
        # a long prompt of the mixture shape in one pass, with head norms and split-half rotation: bandwidth
        dict(kind="store", **_MOE, T=2048, pos=0, rows=4400, fmt=MX8, neox=1, norm=1, name="store_2048_moe_mx8"),
        # one token of the 8B shape behind the headline workload's context
        dict(kind="attend", **_8B, T=1, pos=4100, rows=4400, name="attend_1_8b_4k"),
        # one token behind a very long conversation: the cache's bytes are all of it
        dict(kind="attend", **_8B, T=1, pos=131000, rows=131072, name="attend_1_8b_128k"),
        # a prompt chunk in the engine's default setting, inside a conversation
        dict(kind="attend", **_8B, T=32, pos=480, rows=4096, name="attend_32_8b"),
        # a long prompt in one pass: the matrix cores
        dict(kind="attend", **_8B, T=2048, pos=0, rows=4400, name="attend_2048_8b"),
        # a prompt chunk of the sliding-window shape, its ring of 1024 + 512 slots wrapping
        dict(kind="attend", **_WIN, T=500, pos=2100, rows=1536, swa=1024, cap=1536, name="attend_500_window"),
        # a small tree behind the headline context, f16 cache: latency
        dict(kind="tree", **_8B, T=8, pos=4100, rows=4400, fmt=F16, width=3, name="tree_8_8b_f16"),
        # a wide tree of the mixture shape behind a long context, 8-bit cache
        dict(kind="tree", **_MOE, T=64, pos=32700, rows=32800, fmt=MX8, width=4, name="tree_64_moe_mx8_32k"),
        # the small model's tree right after a short prompt, f32 cache
        dict(kind="tree", **_TINY, T=25, pos=96, rows=512, fmt=F32, width=2, name="tree_25_tiny_f32"),
        # the accepted path of a 64-token tree in the 32 layers of the 8B shape
        dict(kind="path", **_8B, T=64, pos=333, rows=448, fmt=F16, n=6, layers=32, name="path_6_of_64_f16"),
        # the same in two layers of a small 8-bit cache, which is read back
        dict(kind="path", **_TINY, T=25, pos=96, rows=512, fmt=MX8, n=4, layers=2, name="path_4_of_25_mx8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "tree", "tree", "path"])
    nkv = rng.choice([1, 2, 4, 8])
    c = dict(kind=kind, nh=nkv * rng.choice([1, 2, 3, 4, 8]), nkv=nkv, hd=rng.choice([64, 128]))
    if kind == "store":
        T, pos = _log_int(rng, 1, 2048), rng.choice([0, _log_int(rng, 1, 100000)])
        cap = rng.choice([0, 0, T + rng.randint(0, 700)])
        return dict(c, T=T, pos=pos, rows=cap or pos + T + rng.randint(0, 300), cap=cap, fmt=rng.choice([F32, F16, MX8, MX8]),
                    neox=rng.choice([0, 1]), norm=rng.choice([0, 1]))
    if kind == "path":
        T = _log_int(rng, 2, 128)
        pos = _log_int(rng, 1, 500)
        fmt = rng.choice([F32, F16, MX8])
        return dict(c, T=T, pos=pos, rows=pos + T + rng.randint(0, 100), fmt=fmt, n=rng.randint(1, (T + 1) // 2),
                    layers=_log_int(rng, 1, 3 if fmt == MX8 else 32))
    T = 1 if kind == "attend" and rng.random() < 0.3 else _log_int(rng, 2, 1400 if kind == "attend" else 128)
    # (a scores matrix of the plain form and the cache stay below those of the largest listed cases)
    most = min(131000, 2048 * 2048 * 32 // (c["nh"] * T), 2 * 131000 * 1024 // (3 * nkv * c["hd"]))
    pos = min(most, rng.choice([0, _log_int(rng, 10, 130000)]))
    c.update(T=T, pos=pos, rows=pos + T + rng.randint(0, 200))
    if rng.random() < 0.25:
        swa = rng.choice([100, 512, 1024])
        cap = swa + T + rng.randint(0, 64)
        c.update(swa=swa, **(dict(cap=cap, rows=cap) if cap < c["rows"] else {}))
    if kind == "tree":
        c.update(fmt=rng.choice([F32, F16, MX8]), width=rng.randint(1, 5))
    return c


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def freq_table(hd, base=500000.0):
    e = (-2.0 * torch.arange(hd // 2, dtype=torch.float32, device="cuda") / hd).double()
    return torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), e).float()


def tree_parents(T, width):
    """Parent of each drafted token: `width` children of the last accepted token, then chains and forks below them."""
    return [-1] + [max(0, (i - 1) // width if i % 2 else i - width) for i in range(1, T)]


def tree_plan(case):
    """The tree as its program has it: mask words (uint32 as int32) [T][ceil(T / 32)] and positions [T]."""
    T, par = case["T"], tree_parents(case["T"], case["width"])
    seen, depth = [], []
    for i, p in enumerate(par):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    W = (T + 31) // 32
    words = torch.tensor([[(s >> 32 * w) & 0xFFFFFFFF for w in range(W)] for s in seen], dtype=torch.int64)
    return (words - ((words >> 31) << 32)).int().cuda(), (torch.tensor(depth, dtype=torch.int32) + case["pos"]).cuda()


def path_plan(case):
    """Drafted tokens of the accepted path, increasing: the first token, then tokens past the path's length."""
    n, T = case["n"], case["T"]
    rest = [n + i * (T - n) // max(1, n - 1) for i in range(n - 1)]
    return torch.tensor([0] + rest, dtype=torch.int32, device="cuda")


def _rows(g, n, nkv, hd):
    """Keys or values as models have them: unit variance, two channels of each head a few times larger."""
    x = torch.randn(n, nkv, hd, generator=g, device="cuda")
    x[:, :, 5] *= 6.0
    x[:, :, hd - 20] *= 4.0
    return x


def span(case):
    """Positions that the cache holds and the pass can read, [lo, hi)."""
    swa, hi = case.get("swa", 0), case["pos"] + case["T"]
    lo = max(0, case["pos"] + 1 - swa) if swa else 0
    return lo, hi


def slots_of(case, lo, hi):
    p = torch.arange(lo, hi, device="cuda")
    return p % case["cap"] if case.get("cap") else p


def quantise(x):
    """x [..., hd] -> (bytes [..., hd], scales [..., hd / 32]); 64 bits, since values lie next to borders."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.frexp(top)[1] + 126                        # top = m 2^(e - 126), 1/2 <= m < 1: top 2^(133 - e) in [64, 128)
    e = (e + (top * torch.exp2((133 - e).double()) >= 127.5)).clamp(0, 254).masked_fill(top == 0, 0)
    q = torch.round(b * torch.exp2((133 - e).double())[..., None])
    bad = ~torch.isfinite(top)
    return (q.masked_fill(bad[..., None], 0) + 128).to(torch.uint8).flatten(-2), e.masked_fill(bad, 255).to(torch.uint8)


def dequantise(q, e):
    """f32 values of the blocks (64 bits inside: 2^(x - 133) has no f32 of its own below 2^-126)."""
    s = torch.exp2(e.double() - 133.0).masked_fill(e == 255, math.nan)
    return ((q.unflatten(-1, (-1, 32)).double() - 128.0) * s[..., None]).flatten(-2).float()


def empty_cache(case, layers=1):
    """Caches of all `layers` as the program allocates them: K and V [layers][bytes or values], zeroed."""
    nkv, hd, rows, fmt = case["nkv"], case["hd"], case["rows"], case.get("fmt", MX8)
    R = (rows + 31) // 32 * 32
    if fmt == MX8:
        return tuple(torch.zeros(layers, nkv * R * (hd + hd // 32), dtype=torch.uint8, device="cuda") for _ in "kv")
    t = torch.float16 if fmt == F16 else torch.float32
    return (torch.zeros(layers, rows, nkv * hd, dtype=t, device="cuda"),
            torch.zeros(layers, R if fmt == F16 else rows, nkv * hd, dtype=t, device="cuda"))


def places(case, slots, which):
    """Elements of a cache that hold rows `slots`: [n][nkv][hd] (and, for mx8, their scales' [n][nkv][hd / 32])."""
    nkv, hd, fmt = case["nkv"], case["hd"], case.get("fmt", MX8)
    R = (case["rows"] + 31) // 32 * 32
    s = slots.view(-1, 1, 1).long()
    h = torch.arange(nkv, device="cuda").view(1, -1, 1)
    c = torch.arange(hd, device="cuda").view(1, 1, -1)
    tile, a, g, b = s // 32, s % 32 // 16, s % 16 // 4, s % 4
    if fmt != MX8:
        ch = h * hd + c
        return (tile * nkv * hd + ch) * 32 + 8 * g + 4 * a + b if fmt == F16 and which == "v" else s * nkv * hd + ch
    blk = torch.arange(hd // 32, device="cuda").view(1, 1, -1)
    base, tail = (h * (R // 32) + tile) * 32 * hd, nkv * R * hd
    if which == "k":
        return (base + (((a * (hd // 64) + c // 64) * 4 + c % 64 // 16) * 16 + s % 16) * 16 + c % 16,
                tail + (h * R + s) * (hd // 32) + blk)
    n, d = c // (hd // 16), c % (hd // 16)
    return (base + (((d // 2 * 4 + g) * 16 + n) * 2 + d % 2) * 8 + 4 * a + b,
            tail + (((h * (R // 32) + tile) * (hd // 32) + blk) * 4 + g) * 8 + 4 * a + b)


def put(case, cache, which, slots, x):
    """Stores rows x [n][nkv][hd] into one layer's cache; returns nothing."""
    flat, at = cache.view(-1), places(case, slots, which)
    if case.get("fmt", MX8) == MX8:
        q, e = quantise(x)
        flat[at[0]] = q
        flat[at[1]] = e
    else:
        flat[at] = x.to(cache.dtype)


def take(case, cache, which, slots):
    """Rows `slots` of one layer's cache as f32 [n][nkv][hd]."""
    flat, at = cache.view(-1), places(case, slots, which)
    if case.get("fmt", MX8) == MX8:
        return dequantise(flat[at[0]], flat[at[1]])
    return flat[at].float()


def inputs(case, seed):
    """Everything that the seed decides, in rows."""
    g, kind = _gen(seed), case["kind"]
    nh, nkv, hd, T = case["nh"], case["nkv"], case["hd"], case["T"]
    m = {}
    if kind == "store":
        m["q"] = torch.randn(T, nh, hd, generator=g, device="cuda") * 1.5
        m["k"], m["v"] = _rows(g, T, nkv, hd), _rows(g, T, nkv, hd)
        if case["norm"]:
            m["qnorm"], m["knorm"] = (1.0 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in "qk")
    elif kind == "path":
        m["kc"], m["vc"] = ([_rows(g, case["rows"], nkv, hd) for _ in range(case["layers"])] for _ in "kv")
    else:
        lo, hi = span(case)
        m["q"] = torch.randn(T, nh, hd, generator=g, device="cuda") * 1.5
        m["kc"], m["vc"] = [_rows(g, hi - lo, nkv, hd)], [_rows(g, hi - lo, nkv, hd)]
    return m


def prepare(case, seed):
    s = dict(inputs(case, seed), case=case)
    s["kcache"], s["vcache"] = empty_cache(case, case.get("layers", 1))
    if "kc" in s:
        lo, hi = (0, case["rows"]) if case["kind"] == "path" else span(case)
        at = slots_of(case, lo, hi)
        for i in range(len(s["kc"])):
            put(case, s["kcache"][i], "k", at, s["kc"][i])
            put(case, s["vcache"][i], "v", at, s["vc"][i])
        del s["kc"], s["vc"]
    s["freq"] = freq_table(case["hd"])
    s["paso"] = torch.tensor([case["T"], case["pos"], 0, 0], dtype=torch.int32, device="cuda")
    if case["kind"] == "tree":
        s["mask"], s["where"] = tree_plan(case)
    if case["kind"] == "path":
        s["idx"] = path_plan(case)
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms
def rotated(x, w, pos, freq, neox):
    """x [T][heads][hd] normed per head (w given) and rotated; the angle is the 32-bit product of position and table
    entry, as everywhere in this family, its sine and cosine are taken in 64 bits."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    th = (pos.float()[:, None] * freq[None]).double()[:, None]
    cos, sin = th.cos().float(), th.sin().float()
    a, b = x.chunk(2, -1) if neox else (x[..., 0::2], x[..., 1::2])
    r = (a * cos - b * sin, a * sin + b * cos)
    return torch.cat(r, -1) if neox else torch.stack(r, -1).flatten(-2)


def shown(case, mask=None, where=None):
    """Which positions lo .. hi of span() the T queries see: [T][hi - lo]."""
    T, pos, swa = case["T"], case["pos"], case.get("swa", 0)
    lo, hi = span(case)
    key, t = torch.arange(lo, hi, device="cuda")[None], torch.arange(T, device="cuda")
    at = (where if where is not None else t + pos)[:, None]
    old = (key < pos) if mask is not None else (key <= at)
    if swa:
        old = old & (key > at - swa)
    if mask is not None:
        old = old.expand(T, -1).clone()
        old[:, pos - lo:] = ((mask[:, t // 32] >> (t % 32)) & 1).bool()
    return old


def attention(q, k, v, see, scale):
    """q [T][nh][hd] over k, v [n][nkv][hd], see [T][n]; rows that see nothing are 0."""
    T, nh, hd = q.shape
    nkv = k.shape[1]
    qh = q.reshape(T, nkv, -1, hd).permute(1, 2, 0, 3).reshape(nkv, -1, hd).contiguous()   # [nkv][G T][hd]
    s = torch.bmm(qh, k.permute(1, 2, 0).contiguous()).view(nkv, -1, T, k.shape[0]) * scale
    s = s.masked_fill_(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(nkv, -1, k.shape[0]), v.permute(1, 0, 2).contiguous()).view(nkv, -1, T, hd) / den.masked_fill(den == 0, 1)
    return o.permute(2, 0, 1, 3).reshape(T, nh, hd)


def run_plain(s):
    c = s["case"]
    kind, T, pos = c["kind"], c["T"], c["pos"]
    if kind == "store":
        at = slots_of(c, pos, pos + T)
        p = torch.arange(pos, pos + T, device="cuda")
        qo = rotated(s["q"], s.get("qnorm"), p, s["freq"], c["neox"])
        put(c, s["kcache"][0], "k", at, rotated(s["k"], s.get("knorm"), p, s["freq"], c["neox"]))
        put(c, s["vcache"][0], "v", at, s["v"])
        back = torch.float32 if c["fmt"] == F32 else torch.float16
        return {"q": qo, "k": take(c, s["kcache"][0], "k", at).to(back), "v": take(c, s["vcache"][0], "v", at).to(back)}
    if kind == "path":
        src, dst = slots_of(c, pos, pos + T)[s["idx"].long()], slots_of(c, pos, pos + c["n"])
        for name, cache in (("k", s["kcache"]), ("v", s["vcache"])):
            at = places(c, src, name), places(c, dst, name)
            flat = cache.view(c["layers"], -1)
            for a, b in zip(*at) if c["fmt"] == MX8 else [at]:
                flat[:, b] = flat[:, a]
        if c["fmt"] == MX8:
            at = torch.arange(c["rows"], device="cuda")
            return {n: torch.stack([take(c, x, n, at).half() for x in s[n + "cache"]]) for n in "kv"}
        return {"k": s["kcache"], "v": s["vcache"]}
    lo, hi = span(c)
    at = slots_of(c, lo, hi)
    return attention(s["q"], take(c, s["kcache"][0], "k", at), take(c, s["vcache"][0], "v", at),
                     shown(c, s.get("mask"), s.get("where")), 1.0 / math.sqrt(c["hd"]))


# ------------------------------------------------------------------------------------------------- the backend's own ops
_gpu = None


class Plan:
    """Dispatches with their uniforms and bindings packed once, as the engine's bind groups are."""

    def __init__(self):
        global _gpu
        from quipullm_amd import capi
        _gpu = _gpu or capi.Quipu(0)
        self.capi, self.calls, self.out = capi, [], None

    def add(self, op, u, bufs, grid):
        ub = self.capi.uniform(u)
        hs = [b if isinstance(b, int) else b.data_ptr() for b in bufs]
        self.calls.append((_gpu.op(op), ctypes.create_string_buffer(ub, len(ub)), len(ub), (ctypes.c_uint64 * len(hs))(*hs),
                           len(hs)) + tuple(grid) + (1,) * (3 - len(grid)))

    def run(self):
        dispatch = _gpu.L.qp_dispatch
        for c in self.calls:
            if dispatch(*c):
                _gpu._check(1, "qp_dispatch")
        return self.out


def plan(s):
    c, p = s["case"], Plan()
    nh, nkv, hd, T, pos = c["nh"], c["nkv"], c["hd"], c["T"], c["pos"]
    cap, rows, fmt, swa = c.get("cap", 0), c["rows"], c.get("fmt", MX8), c.get("swa", 0)
    kc, vc = s["kcache"], s["vcache"]
    u = lambda *v: [("f" if isinstance(x, float) else "u", x) for x in v]   # noqa: E731
    if c["kind"] == "store":
        back = 0 if fmt == F32 else 1
        new = lambda *shape, t=torch.float32: torch.empty(*shape, dtype=t, device="cuda")   # noqa: E731
        t = torch.float16 if back else torch.float32
        p.out = {"q": new(T, nh, hd), "k": new(T, nkv, hd, t=t), "v": new(T, nkv, hd, t=t)}
        p.add("norm_rope_kv", u(hd, nh, nkv, c["neox"], EPS, hd, 1.0, cap, fmt, rows),
              [s["paso"], s["q"], s["k"], s["v"], p.out["q"], kc, vc, s.get("qnorm", 0), s.get("knorm", 0), s["freq"], 0], (nh, T))
        p.add("kv_read", u(hd, nkv, cap, fmt, rows, pos, T, back), [0, kc, vc, p.out["k"], p.out["v"]], (nkv, T))
    elif c["kind"] == "path":
        pairs = [x for i in range(c["layers"]) for x in (kc[i], vc[i])]
        p.out = {"k": kc, "v": vc}
        p.add("kv_ramal", u(hd, nkv, cap, fmt, rows, c["n"]), [s["paso"], s["idx"]] + pairs, (c["n"],))
        if fmt == MX8:
            p.out = {n: torch.empty(c["layers"], rows, nkv, hd, dtype=torch.float16, device="cuda") for n in "kv"}
            for i in range(c["layers"]):
                p.add("kv_read", u(hd, nkv, cap, fmt, rows, 0, rows, 1), [0, kc[i], vc[i], p.out["k"][i], p.out["v"][i]], (nkv, rows))
    else:
        p.out = torch.empty(T, nh, hd, device="cuda")
        scale = 1.0 / math.sqrt(hd)
        if c["kind"] == "tree":
            p.add("atencion_arbol", u(hd, nh, nkv, swa, scale, cap, fmt, rows),
                  [s["paso"], s["q"], kc, vc, p.out, s["mask"], s["where"]], (nh, T))
        else:
            p.add("atencion_mx8", u(hd, nh, nkv, swa, scale, cap, 0, 0, MX8, rows), [s["paso"], s["q"], kc, vc, p.out], (nh, T))
    return p


def run(s):
    if own:
        if "plan" not in s:
            s["plan"] = plan(s)
            torch.cuda.synchronize()   # the backend's stream does not wait for torch's: the inputs and the buffers are ready
        return s["plan"].run()
    return run_plain(s)


# ------------------------------------------------------------------------------------------------------- work and truth
def seen_keys(case):
    """(sum of the keys that the queries see, keys that the pass reads)."""
    T, pos, swa = case["T"], case["pos"], case.get("swa", 0)
    lo, hi = span(case)
    if case["kind"] == "tree":
        depth = []
        for p in tree_parents(T, case["width"]):
            depth.append(depth[p] + 1 if p >= 0 else 0)
        old = [min(pos, max(0, swa - 1 - d)) if swa else pos for d in depth]
        return sum(old) + sum(depth) + T, hi - lo
    return sum(min(pos + t + 1, swa or pos + t + 1) for t in range(T)), hi - lo


def work(case):
    nh, nkv, hd, T, fmt = case["nh"], case["nkv"], case["hd"], case["T"], case.get("fmt", MX8)
    row = 2 * nkv * (hd + hd // 32 if fmt == MX8 else hd * (2 if fmt == F16 else 4))   # bytes of a token's K and V
    if case["kind"] == "store":
        back = 4 if fmt == F32 else 2
        return {"bytes": T * (8 * nh * hd + 8 * nkv * hd + 2 * row + 2 * back * nkv * hd), "flops": T * (nh + nkv) * hd * (3 + 4 * case["norm"])}
    if case["kind"] == "path":
        back = case["rows"] * (row + 4 * nkv * hd) if fmt == MX8 else 0
        return {"bytes": case["layers"] * (2 * case["n"] * row + back), "flops": 0}
    total, read = seen_keys(case)
    return {"bytes": read * row + 8 * T * nh * hd, "flops": 4 * hd * nh * total}


def _blocks64(x):
    """What 8-bit blocks hold of x [..., hd], in 64 bits: the scale found by trying two neighbours."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    m = b.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(m.clamp_min(1e-300))) - 6
    for _ in range(2):
        e = torch.where(m / torch.exp2(e) >= 127.5, e + 1, e)
    for _ in range(2):
        e = torch.where(m / torch.exp2(e - 1) < 127.5, e - 1, e)
    e = e.clamp_min(-133)
    return (torch.round(b / torch.exp2(e)) * torch.exp2(e)).reshape(x.shape)


def _held(case, x):
    fmt = case.get("fmt", MX8)
    return _blocks64(x) if fmt == MX8 else (x.half() if fmt == F16 else x.float()).double()


def exact(case, seed):
    m, T, pos, hd = inputs(case, seed), case["T"], case["pos"], case["hd"]
    if case["kind"] == "path":
        src, n = path_plan(case).long(), case["n"]
        out = {}
        for name in ("k", "v"):
            x = _held(case, torch.stack(m[name + "c"]))
            x = x if case["fmt"] == MX8 else x.flatten(2)
            x[:, pos:pos + n] = x[:, pos + src].clone()
            if case["fmt"] == F16 and name == "v":
                x = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[1] % 32))
                L, R, kvd = x.shape
                x = x.view(L, R // 32, 2, 4, 4, kvd).permute(0, 1, 5, 3, 2, 4).reshape(L, R, kvd)   # tiles as they lie
            out[name] = x
        return out
    if case["kind"] == "store":
        def turn(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            f = freq_table(hd)
            ang = ((torch.arange(T, device="cuda") + pos).float()[:, None] * f[None]).double()
            j = torch.arange(hd // 2, device="cuda")
            i0, i1 = (j, j + hd // 2) if case["neox"] else (2 * j, 2 * j + 1)
            y = torch.empty_like(x)
            z = torch.complex(x[..., i0], x[..., i1]) * torch.polar(torch.ones_like(ang), ang)[:, None]
            y[..., i0], y[..., i1] = z.real, z.imag
            return y
        return {"q": turn(m["q"], m.get("qnorm")), "k": _held(case, turn(m["k"], m.get("knorm"))), "v": _held(case, m["v"])}
    # attention: a head at a time, the keys of a position before the window or after the query left out by their position
    k, v, q = _held(case, m["kc"][0]), _held(case, m["vc"][0]), m["q"].double()
    lo, hi = span(case)
    p = torch.arange(lo, hi, device="cuda")
    swa, G = case.get("swa", 0), case["nh"] // case["nkv"]
    if case["kind"] == "tree":
        par, see, depth = tree_parents(T, case["width"]), torch.zeros(T, hi - lo, dtype=torch.bool), []
        for t in range(T):
            depth.append(depth[par[t]] + 1 if par[t] >= 0 else 0)
            a = t
            while a >= 0:
                see[t, pos - lo + a] = True
                a = par[a]
        see = see.cuda()
        at = torch.tensor(depth, device="cuda") + pos
        see |= (p[None] < pos) & (p[None] > at[:, None] - swa if swa else True)
    else:
        at = torch.arange(T, device="cuda") + pos
        see = (p[None] <= at[:, None]) & (p[None] > at[:, None] - swa if swa else True)
    o = torch.zeros(T, case["nh"], hd, dtype=torch.float64, device="cuda")
    for h in range(case["nh"]):
        w = torch.softmax((q[:, h] @ k[:, h // G].T / math.sqrt(hd)).masked_fill(~see, -math.inf), -1)
        o[:, h] = w @ v[:, h // G]
    return o
