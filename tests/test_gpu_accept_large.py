"""llm_draft_accept where a likely token was turned down, for large batches and vocabularies, against its definition in float64."""
import pytest

from helpers import pkg
from test_gpu_accept import check, inputs, run
from test_gpu_pages import DEV, gen

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1.0, 0.5])
@pytest.mark.parametrize("v", [100, 5003, 33000])
@pytest.mark.parametrize("shares", [[0.3, 0.2, 0.1], [0.999, 0.6], [0.9] * 5, [0.2, 0.9, 0.99, 0.05]])
@pytest.mark.parametrize("tail", [0.3, 1e-3, 1e-5, 1.2e-7])
def test_children_behind_a_likely_one(tail, shares, v, temperature):
    """Drafts that were not drawn, most of the row's probability in the first child, which is turned down.  Each later child has a share
    of what is then left, and a coin 1/512 of itself below it (it is kept) or above (it is turned down): a child's probability is off
    by 2^-16 of itself at most."""
    g, t = gen(len(shares) + v), len(shares) + 2
    x = torch.randn(v, generator=g, dtype=torch.float64)
    likely = torch.randperm(v, generator=g)[:len(shares) + 1].tolist()
    p = torch.exp(x)
    p[likely] = 0.0
    left, sizes = tail, [1.0 - tail]
    for share in shares:
        sizes.append(left * share)
        left -= left * share
    p *= left / p.sum()
    p[likely] = torch.tensor(sizes, dtype=torch.float64)
    row = (torch.log(p) * temperature).float()
    true = torch.softmax(row.double() / temperature, 0)
    cond = []
    for token in likely:
        keep = torch.ones(v, dtype=torch.bool)
        keep[likely[:len(cond)]] = False
        cond.append(float(true[token] / true[keep].sum()))
    b = 2 * len(shares)
    coins = torch.zeros(b, t)
    for i in range(b):  # sequence i keeps child 1 + i / 2, just so, or turns it down, just so, and keeps the next
        last = 1 + i // 2
        for c in range(len(likely)):
            near = cond[c] * (1.0 + 2.0 ** -9) if c < last or (c == last and i % 2) else cond[c] * (1.0 - 2.0 ** -9) if c == last else 0.0
            coins[i, c + 1] = min(near, 1.0 - 2.0 ** -24)
        assert coins[i, 1] >= cond[0]
        coins[i, 0] = float(torch.rand((), generator=g))
    tokens = torch.tensor([[0] + likely], dtype=torch.int32).repeat(b, 1)
    parents = [[-1] + [0] * (t - 1)] * b
    args = (row.expand(b, t, v).contiguous(), None, tokens, parents, coins, None, temperature)
    got = run(*args)
    check(*args, got)
    for i in range(b):
        if i % 2 == 0:
            assert got[1][i, 1] == 2 + i // 2
        elif cond[1 + i // 2] * (1.0 + 2.0 ** -9) < 1.0 - 2.0 ** -24:
            assert got[1][i, 1] != 2 + i // 2


@pytest.mark.parametrize("temperature", [0.8, 0.0])
@pytest.mark.parametrize("kind,draft", [("fp32", None), ("bf16", None), ("fp32", "fp32"), ("bf16", "fp32"), ("fp32", "bf16"), ("bf16", "bf16")])
def test_a_batch_whose_workgroups_take_four_segments(kind, draft, temperature):
    """16 trees of up to 37 nodes over 32771 logits: nine segments of 4096, two workgroups of four and one of the rest"""
    g, b, t, v = gen(3), 16, 37, 32771
    args = inputs(g, b, t, v, kind, draft, True)
    args[0][3, 0, :], args[0][3, 0, v - 2] = args[0][3, 0, :] - 60.0, 9.0  # (all of a row's weight in its last segment)
    n = [t - i % 7 for i in range(b)]
    check(*args, n, temperature, run(*args, n, temperature))


@pytest.mark.parametrize("temperature", [1.0, 0.0])
@pytest.mark.parametrize("kind,draft", [("fp32", None), ("bf16", None), ("fp32", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("v", [64 * 4096, 64 * 4096 + 1, 290001, 129 * 4096 - 5])
def test_vocabularies_of_more_than_64_segments(v, kind, draft, temperature):
    """the drawn token before, in and behind the 64th segment, and at the row's ends"""
    g, b, t = gen(v % 1000), 6, 3
    x, q, tokens, parents, coins = inputs(g, b, t, v, kind, draft, False, hot=1.0)
    at = [5, 63 * 4096 + 17, min(64 * 4096, v - 1), v - 1, v // 2, v - 30]
    for i in range(b):
        if temperature == 0.0:
            x[i, :, at[i]] = 30.0
        coins[i, 0] = (at[i] + 0.5) / v
    coins[3, 0], coins[0, 0] = 1.0 - 2.0 ** -24, 0.0
    check(x, q, tokens, parents, coins, None, temperature, run(x, q, tokens, parents, coins, None, temperature))


def test_results_do_not_hold_the_work_memory():
    """a program that keeps what a call returned keeps a few KB of it"""
    b, t, v = 3, 5, 70001
    x, q, tokens, parents, coins = inputs(gen(4), b, t, v, "fp32", "fp32", False)
    got = run(x, q, tokens, parents, coins, None, 1.0)
    assert pkg().lib().llm_draft_accept_work(b, t, v) > 65536
    assert all(y.untyped_storage().nbytes() <= 4096 and y.device.type == DEV for y in got)
