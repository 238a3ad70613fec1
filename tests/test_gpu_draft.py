"""Models with 8-bit caches, drafted trees in one pass, scored texts (llm_set_kv, llm_verify, llm_keep, llm_score).

Bars.  Two paths of the fast mode (batched and step by step) add in other orders, and an int8 code of an activation, or here of
a cache row, that lies next to a border may land on its other side: logits within 2e-2 of their scale, 1e-3 at most of the
positions, as for the batched prefill (test_gpu_prefill.py).  The first layer's cache rows depend on no attention: they are
the fp32 model's, quantized by the definition, exactly.  A wiring mistake moves logits by their own size: the distance to the
fp32 cache is held to a quarter of it.  Log probabilities: those of the logits in float64, within 1e-5 (sums of at most a few
hundred terms in fp32)."""
import os
import subprocess

import numpy as np
import pytest

from helpers import GOLDEN, PKG_DIR, pkg, rel_err, synth
from test_gpu_operators import quantized

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TINY = [f"{GOLDEN}/tiny.qwb", f"{GOLDEN}/tiny.bin"]
PROMPT = [5, 77, 300, 12, 9, 41, 7, 130, 222, 3]


def prompt(m, n, seed=0):
    return np.random.default_rng(seed).integers(3, m.info.vocab_size, n).astype(np.int32)


def flip_bar(a, b):
    e = [rel_err(x, y) for x, y in zip(a, b)]
    assert max(e) < 2e-2 and np.median(e) < 1e-3, e


def steps(m, ids, pos0=0):
    return np.stack([m.forward(t, pos0 + i) for i, t in enumerate(ids)])


@pytest.mark.parametrize("path", TINY)
@pytest.mark.parametrize("kind", ["bf16", "int8", "e4m3"])
def test_cache_rows_and_paths(path, kind):
    """the first layer's rows, written by steps and by the batched prefill; both paths' logits; generations from graphs"""
    a, b = pkg().Model(path, 64), pkg().Model(path, 64)
    ids = prompt(a, 24)
    b.set_kv(kind)
    assert b.kv == kind and a.kv == "fp32"
    kvh, ctx = a.info.n_kv_heads, a.info.ctx
    hs = a.info.dim // a.info.n_heads
    want, rows = {}, {}
    for how in ("steps", "prefill"):
        for m, out in ((a, want), (b, rows)):
            lg = steps(m, ids)[-1] if how == "steps" else m.prefill(ids)
            out[how] = [m.read_state(w, 0).reshape(ctx, kvh, hs)[:24] for w in (1, 2)] + [lg]
        for x, y in zip(want[how][:2], rows[how][:2]):
            v, _, _ = quantized(torch.from_numpy(x).double(), kind)
            assert np.array_equal(v.float().numpy(), y), how
        assert rel_err(rows[how][2], want[how][2]) < 0.25
    flip_bar([rows["steps"][2]], [rows["prefill"][2]])
    b.set_prefill(False)
    g = b.generate(ids[:9], 12, logits=True)
    seq = list(ids[:9]) + list(g["ids"])
    lg = steps(b, seq[:len(g["logits"])])
    assert np.array_equal(lg, g["logits"])  # the captured steps are the eager ones
    b.set_prefill(True)
    flip_bar(b.generate(ids[:9], 1, logits=True)["logits"], lg[:9])
    b.set_kv("fp32")
    assert np.array_equal(b.prefill(ids), want["prefill"][2])
    a.close(), b.close()


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_long_context_steps_over_a_quantized_cache(tmp_path, kind):
    """positions across many slices: a prompt of 700 tokens in one pass, then steps; the same by steps alone"""
    p = synth("qwb", str(tmp_path / "m.qwb"), "tiny", 3, "max_seq=1024")
    m = pkg().Model(p, 1024)
    m.set_kv(kind)
    ids = prompt(m, 710, 1)
    m.prefill(ids[:700])
    a = steps(m, ids[700:], 700)
    b = steps(m, ids)[700:]
    flip_bar(a, b)
    m.close()


TREE = ([11, 22, 33, 44, 55, 66, 77], [-1, 0, 0, 1, 2, 2, 5])


@pytest.mark.parametrize("path", TINY)
@pytest.mark.parametrize("kind", ["fp32", "bf16", "int8", "e4m3"])
def test_a_tree_is_its_paths(path, kind):
    """every node's logits are those of its path step by step; its parent's give its log probability; the accepted path's
    rows moved together continue as the path itself would"""
    m = pkg().Model(path, 64)
    m.set_kv(kind)
    ids, (tokens, parents) = prompt(m, 17, 2), TREE
    m.prefill(ids)
    nxt, lp, lg = m.verify(17, tokens, parents, logits=True)
    state = [m.read_state(w, 1).copy() for w in (1, 2)]
    want = np.empty_like(lg)
    for i in range(len(tokens)):
        path_i, j = [], i
        while j >= 0:
            path_i.insert(0, j)
            j = parents[j]
        want[i] = steps(m, [tokens[k] for k in path_i], 17)[-1]
    flip_bar(lg, want)
    row = {int(t): r for r, t in reversed(list(enumerate(m.head_ids)))}
    for i in range(len(tokens)):
        assert nxt[i] == m.head_ids[int(np.argmax(lg[i]))]
        if parents[i] < 0:
            assert lp[i] == 0.0
        elif tokens[i] not in row:
            assert lp[i] == -np.inf
        else:
            x = lg[parents[i]].astype(np.float64)
            assert abs(lp[i] - (x[row[tokens[i]]] - x.max() - np.log(np.exp(x - x.max()).sum()))) < 1e-5
    # the same tree again, then its path 0, 2, 5, 6 kept
    again = m.verify(17, tokens, parents)
    assert np.array_equal(again[0], nxt) and np.array_equal(again[1], lp)
    m.keep(17, [0, 2, 5, 6])
    kvd = state[0].size // m.info.ctx
    for w, old in zip((1, 2), state):
        new, old = m.read_state(w, 1).reshape(m.info.ctx, kvd), old.reshape(m.info.ctx, kvd)
        assert np.array_equal(new[:17], old[:17])
        assert np.array_equal(new[17:21], old[17:][[0, 2, 5, 6]])
    a = steps(m, [99, 98], 21)
    m.prefill(ids)
    b = steps(m, [11, 33, 66, 77, 99, 98], 17)[4:]
    flip_bar(a, b)
    m.close()


@pytest.mark.parametrize("n", [1, 2, 40, 64])
def test_chains_of_drafted_tokens(tmp_path, n):
    """no parents: a chain, as the same tokens forced step by step; from an empty cache too"""
    m = pkg().Model(synth("qwb", str(tmp_path / "m.qwb"), "tiny", 4, "max_seq=128"), 128)
    for kind, pos0 in (("fp32", 0), ("int8", 0), ("int8", 50)):
        m.set_kv(kind)
        ids = prompt(m, pos0 + n, 5)
        if pos0:
            m.prefill(ids[:pos0])
        _, lp, lg = m.verify(pos0, ids[pos0:], logits=True)
        flip_bar(lg, steps(m, ids[pos0:], pos0))
        assert (lp[1:] < 0).all()
    m.close()


def test_drafts_at_the_end_of_the_context_and_refusals(capfd):
    m = pkg().Model(TINY[0], 32)
    ids = prompt(m, 32, 6)
    m.prefill(ids[:28])
    _, _, lg = m.verify(28, ids[28:], logits=True)
    flip_bar(lg, steps(m, ids[28:], 28))
    for call in (lambda: m.verify(29, ids[28:]), lambda: m.verify(-1, [1]), lambda: m.verify(0, [m.info.vocab_size]),
                 lambda: m.verify(0, [1, 2], [-1, 1]), lambda: m.verify(0, [1, 2], [-2, 0]), lambda: m.verify(0, []),
                 lambda: m.keep(0, [1, 1]), lambda: m.keep(0, [2, 1]), lambda: m.keep(31, [1]), lambda: m.keep(0, [64]),
                 lambda: m.score([]), lambda: m.score(ids, top=33), lambda: m.score(ids, temperature=0.0),
                 lambda: m.score([-1])):
        with pytest.raises(RuntimeError):
            call()
    m.set_strict(True)
    for call in (lambda: m.verify(0, [1]), lambda: m.set_kv("int8")):
        with pytest.raises(RuntimeError):
            call()
    assert m.kv == "fp32"
    m.set_strict(False)
    m.set_kv("int8")
    with pytest.raises(RuntimeError):
        m.set_strict(True)
    assert not m.strict and m.kv == "int8"
    m.prefill(ids[:28])
    m.close()


def test_positions_far_outside_are_refused():
    m = pkg().Model(TINY[0], 64)
    far = 2 ** 31 - 1
    for pos0, ids in ((far, [5, 6]), (far - 1, [5]), (64, [5]), (63, [5, 6])):
        with pytest.raises(RuntimeError):
            m.verify(pos0, ids)
    for pos0, path in ((far, [0, 1]), (0, [0, far]), (64, [0]), (63, [0, 1]), (60, [0, 4]), (far - 2, [5, 63])):
        with pytest.raises(RuntimeError):
            m.keep(pos0, path)
    m.verify(62, [5, 6])
    m.keep(62, [1])
    m.close()


def test_first_scores_of_a_model():
    """a model's first call allocates the buffers (zeroed, on another stream than the tokens come by): it scores as the next"""
    for _ in range(60):
        m = pkg().Model(TINY[0], 64)
        ids = prompt(m, 31, 8)
        for a, b in zip(m.score(ids, top=32), m.score(ids, top=32)):
            assert np.array_equal(a, b)
        v = [m.verify(len(ids), ids[:8], [-1, 0, 0, 1, 2, 3, 4, 5], logits=True) for _ in range(2)]
        for a, b in zip(*v):
            assert np.array_equal(a, b, equal_nan=a.dtype == np.float32)
        m.close()


@pytest.mark.parametrize("path", TINY)
@pytest.mark.parametrize("strict", [False, True])
@pytest.mark.parametrize("n", [1, 2, 31])
def test_scores_are_those_of_the_logits(path, strict, n):
    m = pkg().Model(path, 64)
    m.set_strict(strict)
    ids = prompt(m, n, 8)
    lg = m.generate(ids, 1, logits=True)["logits"][:n].astype(np.float64)
    for temperature in (1.0, 0.6):
        lp, ent, ti, tl = m.score(ids, top=5, temperature=temperature)
        y = lg / temperature
        z = y - y.max(1, keepdims=True)
        z = z - np.log(np.exp(z).sum(1, keepdims=True))
        row = {int(t): r for r, t in reversed(list(enumerate(m.head_ids)))}
        for i in range(n - 1):
            want = z[i, row[int(ids[i + 1])]] if int(ids[i + 1]) in row else -np.inf
            assert lp[i] == want or abs(lp[i] - want) < 1e-5
        assert np.abs(ent + (np.exp(z) * z).sum(1)).max() < 1e-5
        order = np.argsort(-lg, 1, kind="stable")[:, :5]
        assert np.array_equal(ti, m.head_ids[order])
        assert np.abs(tl - np.take_along_axis(z, order, 1)).max() < 1e-5
    a = m.score(ids, top=2)
    m.set_prefill(False)  # position by position
    b = m.score(ids, top=2)
    if strict:
        for x, y in zip(a, b):
            assert np.array_equal(x, y)
    m.close()


def test_speculative_greedy_decoding_is_greedy_decoding():
    """a draft of right and wrong tokens at every turn: the accepted tokens are the model's own greedy ones"""
    m = pkg().Model(TINY[0], 128)
    ids = list(prompt(m, 9, 11))
    want = list(m.generate(ids, 24)["ids"])
    m.prefill(ids)
    first = int(m.head_ids[int(np.argmax(m.forward(ids[-1], len(ids) - 1)))])
    out, pos, turns = [first], len(ids), 0
    rng = np.random.default_rng(0)
    while len(out) < len(want):
        # node 0: the last token; its children: a wrong guess, and the right continuation up to two deep, then a wrong one
        right = want[len(out):len(out) + 2]
        wrong = int(rng.integers(3, 400))
        tokens = [out[-1], wrong] + right + [wrong]
        parents = [-1, 0] + [0, 2][:len(right)] + [1 + len(right) if right else 0]
        nxt, _ = m.verify(pos, tokens, parents)
        path, node = [0], 0
        while True:
            out.append(int(nxt[node]))
            kids = [i for i in range(len(tokens)) if parents[i] == node and tokens[i] == nxt[node]]
            if not kids or len(out) >= len(want):
                break
            node = kids[0]
            path.append(node)
        m.keep(pos, path)
        pos += len(path)
        turns += 1
    assert out[:len(want)] == want and turns < len(want)
    m.close()


@pytest.mark.parametrize("exe,name", [("qwen_hip", "tiny.qwb"), ("runq_hip", "tiny.bin")])
def test_the_hosts_take_the_caches_type(exe, name):
    path = os.path.join(GOLDEN, name)
    m = pkg().Model(path, 64)
    m.set_kv("int8")
    ids = [1, 5, 77, 30]
    n = 12 if name.endswith("qwb") else m.info.ctx
    want = list(m.generate(ids, 12 if name.endswith("qwb") else n - len(ids) + 1)["ids"])
    m.close()
    run = [os.path.join(PKG_DIR, "host", exe), path, "--ids", ",".join(map(str, ids)), "-t", "0", "-n", str(n), "--kv", "int8"]
    r = subprocess.run(run + (["-c", "64"] if exe == "qwen_hip" else []), capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert [int(x) for x in r.stdout.strip().split(",") if x] == want
    bad = subprocess.run(run[:-1] + ["int4"], capture_output=True, text=True, timeout=60)
    assert bad.returncode != 0 and "--kv int4" in bad.stderr


def test_scores_of_a_text_hold_no_logits_of_the_whole_context(tmp_path):
    """ten tokens scored in a context of 65536: the memory of their own rows (those of every position: 67 MB)"""
    m = pkg().Model(synth("qwb", str(tmp_path / "m.qwb"), "tiny", 3, "max_seq=65536"), 65536)
    assert m.info.n_logits * 65536 * 4 > 60 << 20
    ids = prompt(m, 10, 4)
    m.prefill(ids)
    before = torch.cuda.mem_get_info()[0]
    a = m.score(ids, top=3)
    assert before - torch.cuda.mem_get_info()[0] < 16 << 20
    lg = m.generate(ids, 1, logits=True)["logits"][:10].astype(np.float64)
    z = lg - lg.max(1, keepdims=True)
    z -= np.log(np.exp(z).sum(1, keepdims=True))
    assert np.abs(a[3] - np.take_along_axis(z, np.argsort(-lg, 1, kind="stable")[:, :3], 1)).max() < 1e-5
    m.close()


def test_scores_over_several_chunks(tmp_path):
    """a text longer than a chunk of 2048, its scores those of the logits that a generation keeps"""
    m = pkg().Model(synth("qwb", str(tmp_path / "m.qwb"), "tiny", 3, "max_seq=4600"), 4600)
    ids = prompt(m, 4500, 4)
    lp, ent, ti, tl = m.score(ids, top=2)
    lg = m.generate(ids, 1, logits=True)["logits"][:4500].astype(np.float64)
    z = lg - lg.max(1, keepdims=True)
    z -= np.log(np.exp(z).sum(1, keepdims=True))
    row = {int(t): r for r, t in reversed(list(enumerate(m.head_ids)))}
    want = np.array([z[i, row[int(t)]] if int(t) in row else -np.inf for i, t in enumerate(ids[1:])])
    there = np.isfinite(want)
    assert (lp[~there] == -np.inf).all() and np.abs(lp[there] - want[there]).max() < 1e-5
    assert np.abs(ent + (np.exp(z) * z).sum(1)).max() < 1e-5
    order = np.argsort(-lg, 1, kind="stable")[:, :2]
    assert np.array_equal(ti, m.head_ids[order])
    assert np.abs(tl - np.take_along_axis(z, order, 1)).max() < 1e-5
    b = m.score(ids[:7], top=2)  # fewer rows than the memory held
    assert np.array_equal(b[2], ti[:7]) and np.abs(b[0][there[:6]] - lp[:6][there[:6]]).max() < 1e-2
    m.close()
