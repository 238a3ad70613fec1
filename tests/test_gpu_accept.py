"""llm_draft_accept against its definition: the residual distributions one after another in float64.  Kept nodes, paths and drawn
tokens have to be equal; a log probability is off by at most the rounding of its result.  Without draft probabilities by its row's
sum too, in 32 bits: an exponent y = (x - m) log2(e) / T is off by three roundings, 3 2^-24 |y|, which over the row is 3 2^-24 ln 2
sum p |y| <= 3 2^-24 ln 2 log2(vocab) <= 2.2e-6; the instruction by 2^-22; eight chains of eight additions by 2^-21: 2.9e-6 <
2^-18."""
import math
import random

import pytest

import pages_ref as ref
from helpers import pkg
from pages_ref import ROWS
from test_gpu_pages import DEV, gen, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def inputs(g, b, t, v, kind, draft, tree, hot=3.0, noise=0.5):
    """logits, draft probabilities (or None), tokens drawn from them, parents (or None), coins"""
    x = (torch.randn(b, t, v, generator=g) * hot).to(ROWS[kind])
    q = torch.softmax(x.float() + noise * torch.randn(b, t, v, generator=g), -1)
    q = q.to(ROWS[draft]) if draft else None
    parents = [[-1] + [r if not tree else max(0, r - int(torch.randint(0, 4, (), generator=g))) for r in range(t - 1)]
               for _ in range(b)]
    p = q.float() if draft else torch.softmax(x.float(), -1)
    tokens = torch.zeros(b, t, dtype=torch.int32)
    for i in range(b):
        for j in range(1, t):
            tokens[i, j] = int(torch.multinomial(p[i, parents[i][j]], 1, generator=g))
    coins = torch.rand(b, t, generator=g)
    return x, q, tokens, parents if tree else None, coins


def run(x, q, tokens, parents, coins, n, temperature):
    on = lambda y: None if y is None else y.to(DEV)  # noqa: E731
    return pkg().draft_accept(on(x), on(tokens), on(coins), None if parents is None else ints(parents), None if n is None else ints(n),
                              on(q), temperature)


def check(x, q, tokens, parents, coins, n, temperature, got):
    b, t, v = x.shape
    kept, path, drawn, logp = (y.cpu() for y in got)
    f32 = float(torch.tensor(temperature, dtype=torch.float32))
    for i in range(b):
        want = ref.accept(x[i].double(), tokens[i].tolist(), coins[i].double().tolist(), None if parents is None else parents[i],
                          t if n is None else min(max(n[i], 0), t), None if q is None else q[i].double(), f32)
        assert int(kept[i]) == want[0], i
        assert path[i].tolist() == want[1], i
        assert int(drawn[i]) == want[2], i
        for a, w in zip(logp[i].tolist(), want[3]):
            assert a == w or (math.isnan(a) and math.isnan(w)) or abs(a - w) <= 2.0 ** -24 * abs(w) + (2.0 ** -18 if q is None else 1e-12), (i, a, w)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 0.0])
@pytest.mark.parametrize("kind,draft", [("fp32", None), ("bf16", None), ("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("b,t,v,tree", [(1, 1, 1, False), (3, 2, 2, False), (5, 6, 63, True), (4, 9, 1000, False), (9, 17, 4096, True),
                                        (2, 64, 4097, True), (3, 5, 10007, True), (2, 4, 70001, False)])
def test_chains_and_trees(b, t, v, tree, kind, draft, temperature):
    g = gen(b * t + v)
    args = inputs(g, b, t, v, kind, draft, tree)
    n = [t - i % max(1, t // 2) for i in range(b)]
    check(*args, n, temperature, run(*args, n, temperature))
    check(*args, None, temperature, run(*args, None, temperature))


@pytest.mark.parametrize("draft", [None, "fp32"])
def test_drafts_that_are_far_off(draft):
    """most are turned down: long rows of siblings, twice the same token among them"""
    g = gen(5)
    x, q, tokens, _, coins = inputs(g, 6, 33, 300, "fp32", draft, False, hot=1.0, noise=3.0)
    parents = [[-1] + [0] * 20 + [1 + r // 4 for r in range(12)] for _ in range(6)]
    tokens[:, 5:9] = tokens[:, 4:5]
    coins[0] = 0.999999
    coins[1] = 0.0
    check(x, q, tokens, parents, coins, None, 1.0, run(x, q, tokens, parents, coins, None, 1.0))


def test_the_draft_is_the_target():
    """q = p: everything is kept but for rounding, and where nothing is left the target's row is drawn from"""
    g = gen(6)
    x = torch.log(torch.tensor([0.5, 0.25, 0.125, 0.125])).repeat(4, 5, 1)
    q = torch.softmax(x, -1) * torch.tensor([1.0, 1.0, 2.0, 4.0])[:, None, None]  # (of the last two all is turned down at times)
    tokens = torch.randint(0, 4, (4, 5), generator=g).int()
    coins = torch.rand(4, 5, generator=g)
    check(x, q, tokens, None, coins, None, 1.0, run(x, q, tokens, None, coins, None, 1.0))


def test_trees_that_are_none():
    """parents at or behind their node, below zero, tokens outside the vocabulary, sequences of no node"""
    g = gen(7)
    for draft in (None, "bf16"):
        x, q, tokens, parents, coins = inputs(g, 5, 12, 50, "fp32", draft, True)
        parents[0][3], parents[0][4], parents[1][2], parents[1][1] = 3, 7, -1, 1 << 30
        tokens[2, 1], tokens[2, 5], tokens[3, 1] = -1, 50, 1 << 30
        tokens[:, 0] = -5
        n = [12, 12, 12, 0, -3]
        check(x, q, tokens, parents, coins, n, 1.0, run(x, q, tokens, parents, coins, n, 1.0))


@pytest.mark.parametrize("temperature", [1.0, 0.0])
@pytest.mark.parametrize("draft", [None, "fp32"])
def test_rows_without_probabilities(draft, temperature):
    """NaN, infinities, masked logits, rows of nothing but -infinity; the row may be the first, a middle or an unvisited one"""
    g = gen(8)
    for v in (40, 5000):
        x, q, tokens, _, coins = inputs(g, 8, 5, v, "fp32", draft, False, noise=0.0)
        coins[:, 1:] = 0.0
        x[0, 0, 3] = math.nan
        x[1, 2, v - 1] = math.inf
        x[2, 1] = -math.inf
        x[3, :, : v // 2] = -math.inf
        x[4, 4, 0] = math.nan
        x[5, 3, 7] = -math.inf
        x[6, 2, 5], x[6, 2, 6] = math.nan, math.inf
        x[7] = torch.where(torch.arange(v) == v - 2, x[7], torch.tensor(-math.inf))
        check(x, q, tokens, None, coins, None, temperature, run(x, q, tokens, None, coins, None, temperature))


def test_equal_logits_and_the_ends_of_the_row():
    """temperature 0 takes the first of equal ones; coins 0 and just below 1 draw the first and the last that has weight"""
    x = torch.zeros(2, 3, 9000)
    x[:, :, 4100] = x[:, :, 8200] = 5.0
    tokens = torch.tensor([[0, 4100, 8200]] * 2, dtype=torch.int32)
    coins = torch.full((2, 3), 0.5)
    check(x, None, tokens, None, coins, None, 0.0, run(x, None, tokens, None, coins, None, 0.0))
    x = torch.full((2, 1, 9000), -math.inf)
    x[:, 0, 17], x[:, 0, 8191] = 0.0, 0.0
    coins = torch.tensor([[0.0], [1.0 - 2.0 ** -24]])
    got = run(x, None, torch.zeros(2, 1, dtype=torch.int32), None, coins, None, 1.0)
    assert got[2].tolist() == [17, 8191]


def test_rows_of_other_strides():
    """logits in a slice of wider rows, the same draft row for all sequences (stride 0)"""
    g = gen(9)
    x, q, tokens, parents, coins = inputs(g, 3, 7, 501, "bf16", "fp32", True)
    wide = torch.randn(7, 3, 1003, generator=g).to(torch.bfloat16).to(DEV)
    wide[..., 1:502] = x.transpose(0, 1).to(DEV)
    q[1:] = q[:1].clone()
    got = pkg().draft_accept(wide.transpose(0, 1)[..., 1:502], tokens.to(DEV), coins.to(DEV), ints(parents),
                             probs=q[:1].to(DEV).expand(3, 7, 501))
    check(x, q, tokens, parents, coins, None, 1.0, got)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("shape", ["chain", "siblings"])
def test_what_comes_out_is_distributed_as_the_target(shape, draft):
    """20000 sequences with the same rows and their own drafts and coins: the token behind node 0, kept or drawn, falls to each of
    the vocabulary's tokens as often as the target says, within six standard deviations of a count"""
    g, b, v = gen(10 + draft), 20000, 12
    x = torch.randn(1, 3, v, generator=g) * 1.5
    q = torch.softmax(torch.randn(1, 3, v, generator=g), -1)
    p = torch.softmax(x[0, 0].double(), 0)
    parents = [[-1, 0, 1 if shape == "chain" else 0]] * b
    if draft:
        tokens = torch.zeros(b, 3, dtype=torch.int32)
        tokens[:, 1] = torch.multinomial(q[0, 0], b, replacement=True, generator=g).int()
        tokens[:, 2] = torch.multinomial(q[0, 1 if shape == "chain" else 0], b, replacement=True, generator=g).int()
    else:
        tokens = torch.tensor([[0, int(p.argmax()), 3]], dtype=torch.int32).repeat(b, 1)
    coins = torch.rand(b, 3, generator=g)
    kept, path, drawn, _ = (y.cpu() for y in run(x.expand(b, 3, v), q.expand(b, 3, v) if draft else None, tokens, parents, coins,
                                                 None, 1.0))
    first = torch.where(kept > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long()).squeeze(1), drawn)
    count = torch.bincount(first.long(), minlength=v).double()
    assert ((count - b * p).abs() <= 6 * (b * p * (1 - p)).sqrt() + 1).all()


def test_random_trees():
    r = random.Random(3)
    for seed in range(12):
        g = gen(100 + seed)
        b, t, v = r.randint(1, 6), r.randint(1, 40), r.randint(1, 6000)
        args = inputs(g, b, t, v, r.choice(["fp32", "bf16"]), r.choice([None, "fp32", "bf16"]), r.random() < 0.7,
                      hot=r.choice([0.3, 2.0, 8.0]), noise=r.choice([0.1, 1.0]))
        temperature = r.choice([1.0, 0.3, 2.0, 0.0, 1e-30, 1e30])
        check(*args, None, temperature, run(*args, None, temperature))


@pytest.mark.parametrize("kind,draft", [("fp32", "fp32"), ("bf16", "fp32"), ("fp32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("v", [5003, 16383, 16384, 20485])
@pytest.mark.parametrize("t,wide", [(3, 2), (4, 3), (20, 3), (64, 7)])
def test_many_children(kind, draft, v, t, wide):
    """up to seven children of a node, most of them turned down, some without a token or twice the same one"""
    g, b = gen(v + t + wide), 6
    x = (torch.randn(b, t, v, generator=g) * 2.0).to(ROWS[kind])
    q = torch.softmax(x.float() * torch.linspace(0.0, 1.0, b)[:, None, None] + 2.0 * torch.randn(b, t, v, generator=g), -1).to(ROWS[draft])
    parents = [[-1] + [i // wide for i in range(t - 1)] for _ in range(b)]
    tokens = torch.zeros(b, t, dtype=torch.int32)
    for i in range(b):
        for j in range(1, t):
            tokens[i, j] = int(torch.multinomial(q[i, parents[i][j]].float(), 1, generator=g))
    tokens[2, 1], tokens[3, 2] = -1, tokens[3, 1]
    parents[4][t - 1] = -1
    coins = torch.rand(b, t, generator=g)
    n = [t, t, t, t, t, t - 1]
    for temperature in (1.0, 0.6, 0.0):
        check(x, q, tokens, parents, coins, n, temperature, run(x, q, tokens, parents, coins, n, temperature))
