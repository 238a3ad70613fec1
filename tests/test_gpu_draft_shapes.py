"""Drafted trees and quantized caches in models with the heads of the supported ones: 14 query heads over 2 of 64, 28 over 4 of
128, 12 over 12 of 64 (two layers each, small heads).

Bars.  The batched pass and the steps add in other orders.  A sum of dim / 32 group products in fp32 is off by at most that many
half steps, through eight products in a row and the attention: 8 (3584 / 32) 2^-24 < 1e-4 of the logits.  But an int8 code of an
activation, or a code of a cache row, that lies next to a border may land on its other side, and then all that follows
moves by up to a step of that code (one e4m3 code of one K row: a hundred values of the next layer's rows, 1e-2 of the logits).  So
a node whose path's rows have the same codes both ways, which leaves its own activations, is held to 1e-4 at the median of
such nodes, and every node to a quarter of the logits' scale, which a wiring mistake moves by their own size.  The first layer's
rows of a prompt are exact."""
import numpy as np
import pytest

from helpers import pkg, rel_err, synth
from test_gpu_draft import prompt, steps
from test_gpu_operators import quantized

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
SHAPES = [("qwb", "dim=896", "heads=14", "kv_heads=2", "hidden=1024"), ("qwb", "dim=3584", "heads=28", "kv_heads=4", "hidden=1024"),
          ("bin", "dim=768", "heads=12", "kv_heads=12", "hidden=768")]


@pytest.fixture(scope="module", params=SHAPES, ids=lambda s: "-".join(s[:3]))
def model(request, tmp_path_factory):
    fmt, *shape = request.param
    path = synth(fmt, str(tmp_path_factory.mktemp("m") / f"m.{'qwb' if fmt == 'qwb' else 'bin'}"), "tiny", 3, "layers=2",
                 "max_seq=1024", *shape)
    m = pkg().Model(path, 1024)
    yield m
    m.close()


def paths(parents):
    out = []
    for i in range(len(parents)):
        p, j = [], i
        while j >= 0:
            p.insert(0, j)
            j = parents[j]
        out.append(p)
    return out


@pytest.mark.parametrize("kind", ["fp32", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("length", [0, 61, 700])
def test_trees_and_steps(model, kind, length):
    """a tree of 21 tokens behind a prompt is its paths step by step; the accepted one, moved together, goes on as the path does"""
    m = model
    m.set_kv("fp32")
    ids = prompt(m, length + 23, length + 1)
    kvh, ctx = m.info.n_kv_heads, m.info.ctx
    hs = m.info.dim // m.info.n_heads
    if length:
        m.prefill(ids[:length])
        want = [m.read_state(w, 0).reshape(ctx, kvh, hs)[:length].copy() for w in (1, 2)]
    m.set_kv(kind)
    if length:
        m.prefill(ids[:length])
        for w, x in zip((1, 2), want):
            v, _, _ = quantized(torch.from_numpy(x).double(), kind)
            assert np.array_equal(v.float().numpy(), m.read_state(w, 0).reshape(ctx, kvh, hs)[:length])
    rng = np.random.default_rng(length)
    parents = [-1] + [i - 1 if rng.random() < 0.5 else int(rng.integers(0, i)) for i in range(1, 21)]
    tokens = ids[length:length + 21]

    def rows():
        return np.stack([m.read_state(w, layer).reshape(ctx, -1)[length:length + 21] for layer in range(2) for w in (1, 2)])

    nxt, lp, lg = m.verify(length, tokens, parents, logits=True)
    tree = rows()
    kept = max(paths(parents), key=len)
    m.keep(length, kept)
    assert np.array_equal(rows()[:, :len(kept)], tree[:, kept])
    more = steps(m, ids[-2:], length + len(kept))
    err, alike = [], []
    for i, p in enumerate(paths(parents)):
        want = steps(m, tokens[p], length)[-1]
        err.append(rel_err(lg[i], want))
        r = rows()[:, :len(p)]
        alike.append(bool((np.abs(tree[:, p] - r) <= 1e-4 * np.abs(r).max((1, 2), keepdims=True)).all()))
    err, alike = np.array(err), np.array(alike)
    assert err.max() < 0.25 and (not alike.any() or np.median(err[alike]) < 1e-4), (err, alike)
    x = lg.astype(np.float64)
    x -= x.max(1, keepdims=True)
    x -= np.log(np.exp(x).sum(1, keepdims=True))
    row = {int(t): r for r, t in reversed(list(enumerate(m.head_ids)))}
    for i, p in enumerate(parents):
        assert nxt[i] == m.head_ids[int(np.argmax(lg[i]))]
        want = 0.0 if p < 0 else x[p, row[int(tokens[i])]] if int(tokens[i]) in row else -np.inf
        assert lp[i] == want or abs(lp[i] - want) < 1e-5
    want = steps(m, list(tokens[kept]) + list(ids[-2:]), length)[-2:]
    assert max(rel_err(a, b) for a, b in zip(more, want)) < 0.25
