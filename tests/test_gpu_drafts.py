"""The engine on an 8-bit KV cache, and drafted trees (verificarArbol, aceptarRama, the greedy loop with looked-up drafts),
against the CPU oracle on the same seeded synthetic GGUF files.  With f16 and 8-bit caches the oracle is given the GPU's own
cache rows, as the values that they hold (each side rounds its own K and V, and a value near a rounding boundary would land a
step apart); with f32 caches it keeps its own.  Node is started through the spawner of conftest.py, never from this process.
"""
import json
import os

import numpy as np
import pytest

import mx8
import refs
from conftest import ROOT, run
from quipullm_amd import build, synth
from test_gpu_model import generate, oracle_run, rel

pytestmark = pytest.mark.gpu
ENG = os.path.join(ROOT, "quipullm_amd", "js", "engine.js")


@pytest.fixture(scope="module", autouse=True)
def native():
    if not build.built() or not os.path.exists(build.NAPI):
        pytest.fail("native parts not built: run __graft_entry__.build() first")


def slots_of(c, ctx, batch):
    """Slots of each layer's cache: windowed layers keep a ring of window + batch."""
    if c.arch != "gemma3":
        return [ctx] * c.n_layers
    return [24 + batch if i % 2 == 0 else ctx for i in range(c.n_layers)]


def held_rows(path, c, slots, npos, fmt):
    """The first npos rows of K and V of every layer, as the values that the cache holds: [layers][npos][nkv hd] float64, and
    the scales' steps (8 bits)."""
    raw, at = np.fromfile(path, np.uint8), 0
    nkv, hd = c.nkv, c.hd
    ks, vs, steps = [], [], []
    for S in slots:
        if fmt == mx8.MX8:
            R = mx8.slots32(S)
            qi, ei = np.arange(R * nkv * hd).reshape(R, nkv, hd), R * nkv * hd + np.arange(R * nkv * hd // 32).reshape(R, nkv, hd // 32)
            n = qi.size + ei.size
            step = []
            for lay, out in ((mx8.k_bytes, ks), (mx8.v_bytes, vs)):
                b = np.empty(n, np.uint8)
                b[lay(qi, ei)] = raw[at:at + n]
                at += n
                q, e = b[:qi.size].reshape(qi.shape)[:npos], b[qi.size:].reshape(ei.shape)[:npos]
                out.append(mx8.dequantise(q, e).reshape(npos, nkv * hd))
                step.append(np.repeat(2.0 ** (e.astype(np.float64) - 133), 32, -1).reshape(npos, nkv * hd))
            steps.append(step)
        else:
            kvd = nkv * hd
            n = S * kvd * 2
            ks.append(raw[at:at + n].view(np.float16).reshape(S, kvd)[:npos].astype(np.float64))
            at += n
            n = mx8.slots32(S) * kvd * 2
            vs.append(refs.v_rows(raw[at:at + n].view(np.float16), npos, kvd).astype(np.float64))
            at += n
    assert at == raw.size
    return np.array(ks), np.array(vs), steps


def as_reference(ks, vs):
    """As f16 bits: the blocks' values have 7 bits and fit f16 as they are."""
    out = []
    for x in (ks, vs):
        h = x.astype(np.float16)
        assert np.array_equal(h.astype(np.float64), x)
        out.append(h.view(np.uint16))
    return out


@pytest.mark.parametrize("name", ["mini_llama_q4km_c", "mini_llama_q8_c", "mini_qwen3_q4km_c", "mini_qwen3moe_q4k_c",
                                  "mini_gemma3_q4km_c"])
@pytest.mark.parametrize("plen,n,batch", [(40, 14, 32), (150, 8, 160)])
def test_8bit_cache_matches_oracle(oracle, models_dir, tmp_path, name, plen, n, batch):
    """Greedy ids identical and logits within 1e-3 relative, over chunks, one chunk, the reference's op sequence and the
    captured one-token step, given the cache's own values."""
    path = synth.ensure_model(name, models_dir)
    c = synth.CONFIGS[name]
    if c.arch == "gemma3" and plen + n > 24 + batch:
        pytest.skip("the ring wraps: earlier rows are gone")
    prompt = synth.random_prompt(c.vocab, plen, 1)
    kvf = os.path.join(str(tmp_path), "kv.bin")
    for mode in ("ref", "fast"):
        r, lg = generate(path, prompt, n, mode, "mx8", str(tmp_path), ["--batch", str(batch)], kv_out=kvf)
        lg = lg.reshape(-1, c.vocab)
        # (models without the captured step write the last token's logits too)
        ks, vs, _ = held_rows(kvf, c, slots_of(c, 256, batch), plen + n - 1, mx8.MX8)
        want_ids, want_lg = oracle_run(oracle, path, prompt, n, True, as_reference(ks, vs))
        errs = [rel(a, b) for a, b in zip(lg, want_lg)]
        assert r["ids"] == want_ids, (mode, r["ids"], want_ids, errs)
        assert max(errs) < 1e-3, (mode, errs)


def test_8bit_rows_of_the_first_layer_are_the_rounded_values(oracle, models_dir, tmp_path):
    """Layer 0's rows (from the embeddings alone) are within half a step of the oracle's float32 K and V (and their own
    float32 differences, 1e-4 of a block's largest)."""
    import ctypes
    name = "mini_qwen3_q4km_c"
    path = synth.ensure_model(name, models_dir)
    c = synth.CONFIGS[name]
    prompt = synth.random_prompt(c.vocab, 40, 1)
    kvf = os.path.join(str(tmp_path), "kv.bin")
    m = oracle.Model(path, ctx=256, kv_f16=False)
    m.generate(prompt, 4)
    mm = oracle._Model.from_address(m.ptr)
    kvd, npos = c.nkv * c.hd, 43
    for mode in ("ref", "fast"):
        generate(path, prompt, 4, mode, "mx8", str(tmp_path), kv_out=kvf)
        ks, vs, steps = held_rows(kvf, c, [256] * c.n_layers, npos, mx8.MX8)
        for got, step, ptr in ((ks[0], steps[0][0], mm.kc), (vs[0], steps[0][1], mm.vc)):
            want = np.ctypeslib.as_array((ctypes.c_float * (c.n_layers * 256 * kvd)).from_address(ptr)).reshape(
                c.n_layers, 256, kvd)[0, :npos].astype(np.float64)
            assert np.all(np.abs(got - want) <= step * (0.5 + 128e-4)), float(np.max(np.abs(got - want) / step))
    m.close()


TREE = r"""
const fs = require('fs');
const engine = require(%(eng)s);
(async () => {
  const m = await engine.cargarModelo(%(path)s, {ctx: 256, options: {kv_f16: %(kv)s === 'f16', kv_mx8: %(kv)s === 'mx8', batch: 32}});
  const prompt = %(prompt)s, ids = %(ids)s, padres = %(padres)s, camino = %(camino)s, despues = %(despues)s;
  const fd = fs.openSync(%(out)s, 'w'), escribe = (f) => fs.writeSync(fd, Buffer.from(f.buffer, f.byteOffset, f.byteLength));
  await engine.prefill(m, prompt);
  const mal = [];
  const falla = (f) => { try { f(); mal.push(''); } catch (e) { mal.push(e.message); } };
  falla(() => m.aceptarRama([0]));
  falla(() => m.verificarArbol([], []));
  falla(() => m.verificarArbol([1, 2], [-1]));
  falla(() => m.verificarArbol([1, 2], [-1, 1]));
  falla(() => m.verificarArbol([1, 2], [-1, -2]));
  falla(() => m.verificarArbol([1, 1e9], [-1, 0]));
  falla(() => m.verificarArbol(new Array(33).fill(1), new Array(33).fill(-1)));
  const sig1 = Array.from(m.verificarArbol(ids, padres));
  const sig2 = Array.from(m.verificarArbol(ids, padres, {logits: (i, f) => escribe(f)}));
  falla(() => m.aceptarRama([camino[1]]));
  falla(() => m.aceptarRama([0, 3, 1]));
  m.aceptarRama(camino);
  falla(() => m.aceptarRama([0]));
  for (const t of despues) escribe(await m.forward([t], true));
  fs.closeSync(fd);
  m.volcarKV(%(kvf)s);
  console.log(JSON.stringify({sig1: sig1, sig2: sig2, pos: m.pos, hist: m.hist, mal: mal}));
  m.free();
})().catch((e) => { console.error(e.stack); process.exit(1); });
"""
PADRES = [-1, 0, 0, 1, 2, 2, 4, -1, 7]


@pytest.mark.parametrize("name", ["mini_llama_q4km_c", "mini_qwen3moe_q4k_c", "mini_gemma3_q4km_c"])
@pytest.mark.parametrize("kv", ["f32", "f16", "mx8"])
@pytest.mark.parametrize("camino", [[0, 2, 4, 6], [7, 8], [0, 1]])
def test_tree_and_path_match_oracle(oracle, models_dir, tmp_path, name, kv, camino):
    """Every drafted token's logits are those of the oracle behind the prompt and the token's path (f32; f16 and 8 bits: the
    accepted path's, given the cache's values), within 1e-3 relative, and so are those of the tokens after the accepted path."""
    path = synth.ensure_model(name, models_dir)
    c = synth.CONFIGS[name]
    prompt = [int(t) for t in synth.random_prompt(c.vocab, 38, 4)]
    ids = [int(t) for t in synth.random_prompt(c.vocab, len(PADRES), 5)]
    despues = [int(t) for t in synth.random_prompt(c.vocab, 3, 6)]
    out, kvf = str(tmp_path / "lg.f32"), str(tmp_path / "kv.bin")
    print("node tree", name, kv, camino, flush=True)
    script = TREE % {k: json.dumps(v) for k, v in dict(eng=ENG, path=path, kv=kv, prompt=prompt, ids=ids, padres=PADRES,
                                                       camino=camino, despues=despues, out=out, kvf=kvf).items()}
    rc, o, err = run(["timeout", "-k", "5", "110", "node", "-e", script], timeout=120)
    assert rc == 0, err[-3000:]
    r = json.loads(o.strip().splitlines()[-1])
    assert all(r["mal"]) and len(r["mal"]) == 10, r["mal"]
    lg = np.fromfile(out, np.float32).reshape(-1, c.vocab)
    T = len(PADRES)
    assert len(lg) == T + len(despues)
    taken = prompt + [ids[i] for i in camino] + despues
    assert r["hist"] == taken and r["pos"] == len(taken)
    assert r["sig1"] == r["sig2"] == [int(np.argmax(f)) for f in lg[:T]]
    m = oracle.Model(path, ctx=256, kv_f16=kv != "f32")
    nodes = range(T)
    if kv != "f32":
        ks, vs, _ = held_rows(kvf, c, slots_of(c, 256, 32), len(taken), mx8.MX8 if kv == "mx8" else mx8.F16)
        m.set_kv_reference(*as_reference(ks, vs))
        nodes = camino
    errs = {}
    for i in nodes:
        way, j = [], i
        while j >= 0:
            way.insert(0, ids[j])
            j = PADRES[j]
        m.reset()
        m.forward(prompt[:32], False)
        m.forward(prompt[32:], False)
        errs[i] = rel(lg[i], m.forward(way))
    m.reset()
    m.forward(prompt[:32], False)
    m.forward(prompt[32:], False)
    m.forward([ids[i] for i in camino], False)
    for k, t in enumerate(despues):
        errs["after %d" % k] = rel(lg[T + k], m.forward([t]))
    m.close()
    assert max(errs.values()) < 1e-3, errs


@pytest.mark.parametrize("name", ["mini_llama_q4km_c", "mini_qwen3moe_q4k_c", "mini_gemma3_q4km_c"])
@pytest.mark.parametrize("kv", ["f32", "mx8"])
def test_looked_up_drafts_give_the_greedy_ids(models_dir, tmp_path, name, kv):
    """engine.generar with drafts returns the ids of the plain greedy loop, in fewer passes where drafts were accepted."""
    path = synth.ensure_model(name, models_dir)
    block = [int(t) for t in synth.random_prompt(1000, 9, 31)]
    prompt = block * 4
    a, _ = generate(path, prompt, 40, "engine", kv, str(tmp_path))
    b, _ = generate(path, prompt, 40, "engine", kv, str(tmp_path), ["--drafts", "12"])
    print(name, kv, b["drafts"], flush=True)
    assert a["ids"] == b["ids"]
    assert a["pos"] == b["pos"] == len(prompt) + 39
    assert b["drafts"]["pasos"] + b["drafts"]["aceptados"] == 39


RINGS = r"""
const engine = require(%(eng)s);
(async () => {
  const p = %(p)s, x = %(x)s, path = %(path)s, op = {ctx: 256, options: {batch: 32}};
  const gen = (m, ids, n) => engine.generar(m, ids, {temperature: 0, max_tokens: n});
  const m = await engine.cargarModelo(path, op);
  await gen(m, p, 10);                                     // positions 0 .. 68 written
  const b = await gen(m, p.slice(0, 45).concat(x), 1);     // 45 of them stay
  const c = await gen(m, p.slice(0, 20).concat(x), 10);    // position 0's slot has held position 56
  await gen(m, p.slice(0, 30), 1);
  const antes = m.alto;
  m.verificarArbol(x.concat(x, x, x).slice(0, 28), new Array(28).fill(-1));   // positions 30 .. 57 written
  const despues = m.alto;
  const d = await gen(m, p.slice(0, 20).concat(x), 10);
  m.free();
  const f = await engine.cargarModelo(path, {ctx: 256, options: {batch: 32, prompt_cache: false}});
  const c2 = await gen(f, p.slice(0, 20).concat(x), 10);
  f.free();
  console.log(JSON.stringify({b: b.reutilizados, c: c.reutilizados, d: d.reutilizados, cids: c.ids, dids: d.ids, want: c2.ids,
    antes: antes, despues: despues}));
})().catch((e) => { console.error(e.stack); process.exit(1); });
"""


def test_rings_remember_what_was_overwritten(models_dir):
    """Ring caches (windows of 24, rings of 56 slots): a prefix is not reused where a position written since then, by ids that
    were dropped or by drafted tokens, took the slot of a key that its window needs, though the ids processed now are few."""
    path = synth.ensure_model("mini_gemma3_q4km_c", models_dir)
    p, x = ([int(t) for t in synth.random_prompt(1000, n, s)] for n, s in ((60, 41), (7, 42)))
    print("node rings", flush=True)
    rc, o, err = run(["timeout", "-k", "5", "110", "node", "-e", RINGS % {k: json.dumps(v) for k, v in
                                                                        dict(eng=ENG, p=p, x=x, path=path).items()}], timeout=120)
    assert rc == 0, err[-3000:]
    r = json.loads(o.strip().splitlines()[-1])
    assert r["b"] == 45 and r["c"] == 0 and r["d"] == 0
    assert r["cids"] == r["dids"] == r["want"]
    assert r["despues"] == 58 and r["antes"] < 56


DEEP = r"""
const fs = require('fs');
const engine = require(%(eng)s);
(async () => {
  const m = await engine.cargarModelo(%(path)s, {ctx: 256, options: {kv_f16: %(kv)s === 'f16', kv_mx8: %(kv)s === 'mx8', batch: 32}});
  const fd = fs.openSync(%(out)s, 'w'), escribe = (f) => fs.writeSync(fd, Buffer.from(f.buffer, f.byteOffset, f.byteLength));
  await engine.prefill(m, %(prompt)s);
  const sig = Array.from(m.verificarArbol(%(ids)s, %(padres)s, {logits: (i, f) => escribe(f)}));
  m.aceptarRama(%(camino)s);
  for (const t of %(despues)s) escribe(await m.forward([t], true));
  fs.closeSync(fd);
  m.volcarKV(%(kvf)s);
  console.log(JSON.stringify({sig: sig, pos: m.pos, ventana: m.ventana}));
  m.free();
})().catch((e) => { console.error(e.stack); process.exit(1); });
"""


@pytest.mark.parametrize("kv,plen", [("f32", 38), ("f32", 20), ("f16", 20), ("mx8", 20)])
@pytest.mark.parametrize("fork", [False, True])
def test_trees_deeper_than_the_window(oracle, models_dir, tmp_path, kv, plen, fork):
    """Trees of 32 tokens on windows of 24: a chain, and one of 29 that forks behind its 26th token.  A token sees of its
    ancestors what one-token decoding sees: logits within 1e-3 relative of the oracle's, along the path and behind it (f32: along
    both forks, the ring of 56 slots wrapping; f16 and 8 bits: given the cache's values)."""
    name = "mini_gemma3_q4km_c"
    path = synth.ensure_model(name, models_dir)
    c = synth.CONFIGS[name]
    prompt = [int(t) for t in synth.random_prompt(c.vocab, plen, 4)]
    ids = [int(t) for t in synth.random_prompt(c.vocab, 32, 51)]
    padres = [i - 1 for i in range(29)] + ([25, 29, 30] if fork else [28, 29, 30])
    camino = [i for i in range(32) if not fork or i < 26 or i >= 29]
    despues = [int(t) for t in synth.random_prompt(c.vocab, 3, 6)]
    out, kvf = str(tmp_path / "lg.f32"), str(tmp_path / "kv.bin")
    print("node deep tree", kv, plen, fork, flush=True)
    script = DEEP % {k: json.dumps(x) for k, x in dict(eng=ENG, path=path, kv=kv, prompt=prompt, ids=ids, padres=padres,
                                                       camino=camino, despues=despues, out=out, kvf=kvf).items()}
    rc, o, err = run(["timeout", "-k", "5", "110", "node", "-e", script], timeout=120)
    assert rc == 0, err[-3000:]
    r = json.loads(o.strip().splitlines()[-1])
    taken = plen + len(camino) + len(despues)
    assert r["ventana"] == 24 and r["pos"] == taken
    lg = np.fromfile(out, np.float32).reshape(-1, c.vocab)
    assert r["sig"] == [int(np.argmax(f)) for f in lg[:32]]
    m = oracle.Model(path, ctx=256, kv_f16=kv != "f32")
    if kv != "f32":
        ks, vs, _ = held_rows(kvf, c, slots_of(c, 256, 32), taken, mx8.MX8 if kv == "mx8" else mx8.F16)
        m.set_kv_reference(*as_reference(ks, vs))
    errs = {}
    for way in [list(range(29)), camino] if fork and kv == "f32" else [camino]:
        m.reset()
        m.forward(prompt[:32], False)
        if plen > 32:
            m.forward(prompt[32:], False)
        for i in way:
            errs[i] = rel(lg[i], m.forward([ids[i]]))
    for k, t in enumerate(despues):
        errs["after %d" % k] = rel(lg[32 + k], m.forward([t]))
    m.close()
    print({k: float("%.2g" % x) for k, x in errs.items()}, flush=True)
    assert max(errs.values()) < 1e-3, errs


@pytest.mark.parametrize("kv", ["f32", "mx8"])
def test_looked_up_drafts_deeper_than_the_window(models_dir, tmp_path, kv):
    """As test_looked_up_drafts_give_the_greedy_ids, with chains of 31 drafted tokens on windows of 24."""
    path = synth.ensure_model("mini_gemma3_q4km_c", models_dir)
    prompt = [int(t) for t in synth.random_prompt(1000, 40, 31)] * 2
    a, _ = generate(path, prompt, 60, "engine", kv, str(tmp_path))
    b, _ = generate(path, prompt, 60, "engine", kv, str(tmp_path), ["--drafts", "31"])
    print(kv, b["drafts"], flush=True)
    assert a["ids"] == b["ids"]
