"""The cache operators' argument checks and launches on the CPU: the library built against hip_stub.cpp, where memory is the
host's and nothing runs."""
import ctypes as C
import math
import os
import subprocess

import pytest

from conftest import ROOT
from quipullm_amd import capi

CSRC = os.path.join(ROOT, "quipullm_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


class Stub:
    def __init__(self, path):
        self.L = L = C.CDLL(path)
        L.qp_op_id.argtypes = [C.c_char_p]
        for f in (L.qp_dispatch, L.qp_dispatch_noalloc):
            f.argtypes = [C.c_int, C.c_void_p, C.c_uint32, C.c_void_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32]
        L.qp_alloc.argtypes = [C.c_uint64, C.POINTER(C.c_uint64)]
        L.qp_graph_end.argtypes = [C.POINTER(C.c_uint64)]
        assert L.qp_init(0) == 0, self.error()
        self.graph = C.c_uint64()

    def error(self):
        b = C.create_string_buffer(512)
        self.L.qp_last_error(b, 512)
        return b.value.decode()

    def buf(self, n):
        p = C.c_uint64()
        assert self.L.qp_alloc(n, C.byref(p)) == 0
        return p.value

    def dispatch(self, op, u, bufs, grid, noalloc=False):
        """The error text ('' for none), and the launches."""
        i = self.L.qp_op_id(op.encode())
        assert i >= 0, op
        ub = capi.uniform([("f" if isinstance(x, float) else "u", x) for x in u])
        hs = (C.c_uint64 * len(bufs))(*bufs)
        g = tuple(grid) + (1,) * (3 - len(grid))
        f = self.L.qp_dispatch_noalloc if noalloc else self.L.qp_dispatch
        rc = f(i, C.create_string_buffer(ub, len(ub)), len(ub), hs, len(bufs), *g)
        log = C.create_string_buffer(1 << 16)
        assert self.L.stub_launches(log, 1 << 16) == 0
        return self.error() if rc else "", [l.split() for l in log.value.decode().splitlines()]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("stub") / "libquipu_stub.so")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-w", "-I%s/include" % ROCM, "-I" + CSRC,
                        "-o", out, os.path.join(CSRC, "quipu.cpp"), os.path.join(ROOT, "tests", "hip_stub.cpp"), "-Wl,-Bsymbolic",
                        "-Wl,--no-undefined"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    return Stub(out)


def cache_bytes(fmt, rows, nkv, hd):
    r32 = -(-rows // 32) * 32
    return r32 * nkv * (hd + hd // 32) if fmt == 2 else r32 * nkv * hd * 2 if fmt == 1 else rows * nkv * hd * 4


class Call:
    """A call of each operator that is right, to be changed in one place."""

    def __init__(self, lib, op, fmt=2, T=5, hd=128, nh=8, nkv=2, rows=100, cap=0, swa=0):
        self.lib, self.op = lib, op
        n = cache_bytes(fmt, rows, nkv, hd)
        kc, vc, paso = lib.buf(n), lib.buf(n), lib.buf(16)
        q, k, v, o = (lib.buf(4 * T * h * hd) for h in (nh, nkv, nkv, nh))
        self.grid = (nh, T)
        if op == "norm_rope_kv":
            self.names = "hd nh nkv neox eps nrot esc cap fmt rows"
            self.u = [hd, nh, nkv, 1, 1e-6, hd, 1.0, cap, fmt, rows]
            self.bnames = "paso q k v qo kc vc qnorm knorm freq pos"
            self.b = [paso, q, k, v, o, kc, vc, lib.buf(4 * hd), lib.buf(4 * hd), lib.buf(2 * hd), lib.buf(4 * T)]
        elif op == "kv_read":
            self.names, self.u = "hd nkv cap fmt rows p0 n out", [hd, nkv, cap, fmt, rows, 3, T, 0]
            self.bnames, self.b = "paso kc vc k v", [0, kc, vc, k, v]
        elif op == "kv_ramal":
            self.names, self.u = "hd nkv cap fmt rows n", [hd, nkv, cap, fmt, rows, T]
            self.bnames, self.b = "paso idx kc vc", [paso, lib.buf(4 * T), kc, vc]
        elif op == "atencion_mx8":
            self.names = "hd nh nkv swa scale cap bidir centred fmt rows ns"
            self.u = [hd, nh, nkv, swa, 0.1, cap, 0, 0, fmt, rows, 0]
            self.bnames, self.b = "paso q kc vc o parts", [paso, q, kc, vc, o, 0]
        else:
            self.names = "hd nh nkv swa scale cap fmt rows ns"
            self.u = [hd, nh, nkv, swa, 0.1, cap, fmt, rows, 0]
            self.bnames = "paso q kc vc o mask pos parts"
            self.b = [paso, q, kc, vc, o, lib.buf(4 * T * -(-T // 32)), lib.buf(4 * T), 0]
        self.names, self.bnames = self.names.split(), self.bnames.split()

    def run(self, noalloc=False, bufs=None, **change):
        u, b = list(self.u), list(self.b)
        for k, x in change.items():
            if k in self.names:
                u[self.names.index(k)] = x
            elif k != "grid":
                b[self.bnames.index(k)] = x
        return self.lib.dispatch(self.op, u, bufs(b) if bufs else b, change.get("grid", self.grid), noalloc)


OPS = ["norm_rope_kv", "kv_read", "kv_ramal", "atencion_mx8", "atencion_arbol"]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("hd", [64, 128])
def test_right_calls_launch(lib, op, fmt, hd):
    if op == "atencion_mx8" and fmt != 2:
        assert "cache type" in Call(lib, op, fmt, hd=hd).run()[0]
        return
    err, log = Call(lib, op, fmt, hd=hd).run()
    assert not err and len(log) == 1, (err, log)
    err, log = Call(lib, op, fmt, hd=hd, rows=40, cap=40, swa=36).run()
    assert not err and len(log) == 1, (err, log)


COMMON = [(dict(hd=96), "head_dim"), (dict(hd=0), "head_dim"), (dict(nkv=0), "nkv"), (dict(rows=0), "0"), (dict(fmt=3), "cache type"),
          (dict(cap=101), "ring"), (dict(kc=0), "no cache"), (dict(vc=0), "no cache"), (dict(rows=129), "the K cache")]
HEADS = [(dict(nh=0), "nh"), (dict(q=0), "null"), (dict(paso=0), "null")]
REFUSALS = {
    "norm_rope_kv": HEADS + [(dict(nh=65536), "nh"), (dict(nrot=130), "nrot"), (dict(nrot=63), "nrot"), (dict(k=0), "null"),
                             (dict(v=0), "null"), (dict(qo=0), "null"), (dict(freq=0), "frequency"), (dict(cap=4), "ring"),
                             (dict(grid=(8, 6)), "holds")],
    "kv_read": [(dict(out=2), "output type"), (dict(p0=96), "positions"), (dict(p0=0xffffffff), "positions"), (dict(k=0), "null"),
                (dict(v=0), "null"), (dict(n=6), "holds"), (dict(cap=4), "positions"), (dict(cap=90, p0=0xfffffffe), "positions")],
    "kv_ramal": [(dict(paso=0), "null"), (dict(idx=0), "null"), (dict(n=101), "rows in a cache"), (dict(n=6), "the path"),
                 (dict(cap=4), "rows in a cache")],
    "atencion_mx8": HEADS + [(dict(nh=7), "nh"), (dict(nh=66), "nh"), (dict(o=0), "null"), (dict(bidir=1), "not supported"),
                             (dict(centred=1), "not supported"), (dict(ns=65), "shares"), (dict(ns=2), "without a buffer"),
                             (dict(cap=50), "ring"), (dict(cap=50, swa=47), "ring"), (dict(swa=1 << 31), "window"),
                             (dict(grid=(8, 6)), "holds")],
    "atencion_arbol": HEADS + [(dict(nh=7), "nh"), (dict(nh=66), "nh"), (dict(o=0), "null"), (dict(mask=0), "mask"),
                               (dict(swa=9, pos=0), "positions"), (dict(ns=65), "shares"), (dict(ns=2), "without a buffer"),
                               (dict(cap=50), "ring"), (dict(swa=0xffffffff), "window"), (dict(grid=(8, 6)), "holds")],
}


@pytest.mark.parametrize("op,change,word", [(op, c, w) for op in OPS for c, w in COMMON + REFUSALS[op]])
def test_refusals(lib, op, change, word):
    err, log = Call(lib, op).run(**change)
    assert op in err and word in err and not log, (err, log)


@pytest.mark.parametrize("op", OPS)
def test_bindings_past_their_buffers(lib, op):
    """Every binding one element short of what the call needs."""
    c = Call(lib, op, T=5)
    for i, p in enumerate(c.b):
        name = c.bnames[i]
        if not p or name in ("paso", "idx", "pos", "mask", "freq", "qnorm", "knorm"):
            continue
        err, log = c.run(**{name: p + 32 * 4 * 4})
        assert op in err and "holds" in err and not log, (name, err)


def test_missing_bindings(lib):
    for op, least in (("norm_rope_kv", 7), ("kv_read", 5), ("kv_ramal", 4), ("atencion_mx8", 5), ("atencion_arbol", 6)):
        err, log = Call(lib, op).run(bufs=lambda b: b[:least - 1])
        assert err and not log, op
    c = Call(lib, "kv_ramal")
    assert "bindings" in c.run(bufs=lambda b: b + [b[2]])[0]
    assert "bindings" in c.run(bufs=lambda b: b[:2] + b[2:] * 65)[0]
    assert not c.run(bufs=lambda b: b[:2] + b[2:] * 64)[0]


def test_offsets_past_31_bits(lib):
    """A cache that a lane's 32-bit offsets do not reach (bindings that are not the library's: their room is not known)."""
    far = 1 << 40
    b = [far] * 8
    for op, u, rows in (("atencion_mx8", [128, 8, 8, 0, 0.1, 0, 0, 0, 2], 1 << 24), ("atencion_arbol", [128, 8, 8, 0, 0.1, 0, 1], 1 << 20),
                        ("atencion_arbol", [128, 8, 8, 0, 0.1, 0, 0], 1 << 19)):
        bufs = b[:5] + ([0] if op == "atencion_mx8" else [far, 0, 0])
        assert "31 bits" in lib.dispatch(op, u + [rows, 0], bufs, (8, 1))[0]
        assert not lib.dispatch(op, u + [rows - 32, 0], bufs, (8, 1))[0]


def test_shares_and_blocks(lib):
    """What the rules choose: one launch where the keys are few or the blocks fill the device, else shares and their joining;
    blocks of 128 rows where there are enough; none while a graph is captured without a buffer for the shares."""
    def shape(T, rows, nh=32, nkv=8, **kw):
        return Call(lib, "atencion_mx8", T=T, hd=128, nh=nh, nkv=nkv, rows=rows, **kw).run()[1]
    assert [l[0] for l in shape(1, 200)] == ["qp_attn_mx8_h128_causal"]
    a = shape(1, 4400)
    assert [l[0] for l in a] == ["qp_attn_mx8_h128_causal", "qp_attn_mx8_comb4"] and a[0][1:] == ["8", "1", "18", "256"]
    assert shape(1, 131072)[0][3] == "64"
    assert [l[0] for l in shape(2048, 2048)] == ["qp_attn_mx8_h128_causal_wide"]
    assert [l[0] for l in shape(256, 5556)] == ["qp_attn_mx8_h128_causal_wide", "qp_attn_mx8_comb"]
    assert shape(700, 1400)[0][0] == "qp_attn_mx8_h128_causal"
    assert shape(512, 512)[0][:4] == ["qp_attn_mx8_h128_causal", "8", "128", "1"]
    c = Call(lib, "atencion_mx8", T=1, nh=32, nkv=8, rows=4400)
    parts, short = (lib.buf(n * 32 * (4 * 128 + 8)) for n in (7, 6))
    assert lib.L.qp_graph_begin() == 0
    try:
        alone = c.run()[1]
        given = c.run(ns=7, parts=parts)[1]
    finally:
        assert lib.L.qp_graph_end(C.byref(lib.graph)) == 0
    assert [l[3] for l in alone] == ["1"]
    assert [l[0] for l in given] == ["qp_attn_mx8_h128_causal", "qp_attn_mx8_comb"] and given[0][3] == "7"
    assert "shares' buffer" in c.run(ns=7, parts=short)[0]
    # the fixed scratch: shares only as long as they fit it
    assert c.run(noalloc=True)[1][0][3] == "18"


def test_store_groups(lib):
    for T, hd, heads in ((1, 128, "1"), (256, 128, "1"), (512, 128, "4"), (512, 64, "1"), (1024, 64, "4")):
        log = Call(lib, "norm_rope_kv", T=T, hd=hd, nh=32, nkv=8, rows=2048).run()[1]
        assert [l[0] for l in log] == ["qp_norm_rope_kv_h%d_%s" % (hd, heads)], (T, hd, log)
        assert int(log[0][1]) == math.ceil(T * hd / 128)


def test_argmax_rows(lib):
    v, out = lib.buf(4 * 100 * 7), lib.buf(4 * 7)
    assert lib.dispatch("argmax", [100], [0, v, out], (1,)) == ("", [["qp_argmax", "1", "1", "1", "1024"]])
    assert lib.dispatch("argmax", [100, 7], [0, v, out], (1,)) == ("", [["qp_argmax", "7", "1", "1", "1024"]])
    for u in ([100, 8], [101, 7], [1, 8], [1, 65536]):
        err, log = lib.dispatch("argmax", u, [0, v, out], (1,))
        assert "argmax" in err and not log


def exact_calls():
    """(op, fmt, T, hd, given shares): each operator with every cache type and head size, a mask of one word a row and of two."""
    for op in OPS:
        for fmt in (0, 1, 2):
            if op == "atencion_mx8" and fmt != 2:
                continue
            for T, hd in ((5, 128), (33, 64)):
                yield op, fmt, T, hd, 0
                if op.startswith("atencion"):
                    yield op, fmt, T, hd, 3


@pytest.mark.parametrize("op,fmt,T,hd,ns", list(exact_calls()))
def test_bindings_of_exactly_what_is_needed(lib, op, fmt, T, hd, ns):
    """Buffers of exactly the bytes that the call reads or writes are taken; each binding one element (4 bytes) further on is
    refused, by a message that names it."""
    nh, nkv, rows = 8, 2, 101
    c = Call(lib, op, fmt, T=T, hd=hd, nh=nh, nkv=nkv, rows=rows, swa=40 if op.startswith("atencion") else 0)
    r32 = 128
    k = v = 4 * rows * nkv * hd
    if fmt == 1:
        k, v = 2 * rows * nkv * hd, 2 * r32 * nkv * hd
    elif fmt == 2:
        k = v = r32 * nkv * (hd + hd // 32)
    heads = lambda h: 4 * T * h * hd   # noqa: E731
    need = {"kc": (k, "the K cache"), "vc": (v, "the V cache")}
    if op == "norm_rope_kv":
        need.update(q=(heads(nh), "q"), qo=(heads(nh), "the output of q"), k=(heads(nkv), "k"), v=(heads(nkv), "v"),
                    qnorm=(4 * hd, "q's norm"), knorm=(4 * hd, "k's norm"), freq=(4 * (hd // 2), "the frequency table"),
                    pos=(4 * T, "the positions"))
    elif op == "kv_read":
        need.update(k=(heads(nkv), "the keys' rows"), v=(heads(nkv), "the values' rows"))
    elif op == "kv_ramal":
        need.update(idx=(4 * T, "the path"))
    else:
        need.update(q=(heads(nh), "q"), o=(heads(nh), "the output"))
        if op == "atencion_arbol":
            need.update(mask=(4 * T * ((T + 31) // 32), "the mask"), pos=(4 * T, "the positions"))
        if ns:
            need.update(parts=(ns * T * nh * (4 * hd + 8), "the shares' buffer"))
            c.u[c.names.index("ns")] = ns
    assert set(need) == set(n for n, p in zip(c.bnames, c.b) if p or n == "parts" and ns) - {"paso"}
    bufs = {n: lib.buf(size) for n, (size, _) in need.items()}
    err, log = c.run(**bufs)
    assert not err and log, err
    for n, (size, what) in need.items():
        err, log = c.run(**dict(bufs, **{n: bufs[n] + 4}))
        assert err.startswith("%s: %s holds %d bytes" % (op, what, size - 4)) and not log, (n, err)


def test_read_rows_of_16_bits_exactly(lib):
    c = Call(lib, "kv_read", 1, T=5, hd=64, nkv=2)
    k, v = (lib.buf(2 * 5 * 2 * 64) for _ in "kv")
    assert not c.run(out=1, k=k, v=v)[0]
    assert "the keys' rows holds" in c.run(out=1, k=k + 4, v=v)[0] and "the values' rows holds" in c.run(out=1, k=k, v=v + 4)[0]
    assert "holds" in c.run(out=0, k=k, v=v)[0]


def test_argmax_rows_exactly(lib):
    v, out = lib.buf(4 * 100 * 7), lib.buf(4 * 7)
    assert not lib.dispatch("argmax", [100, 7], [0, v, out], (1,))[0]
    assert "the rows holds" in lib.dispatch("argmax", [100, 7], [0, v + 4, out], (1,))[0]
    assert "the output holds" in lib.dispatch("argmax", [100, 7], [0, v, out + 4], (1,))[0]
