"""The operators over a cache in pages together, as a program that serves drafted tokens uses them: attention of the drafted trees
over the pages, tokens kept, room for them, their rows written, batches that change, pages moved.  Every step against the
definitions in float64 (tolerances: those of the attention's test; codes, tables, counts and tokens are equal); captured, on other
streams and again: the same bits."""
import random

import pytest

import pages_ref as ref
import test_gpu_accept
import test_gpu_page_attention
from helpers import pkg
from pages_ref import ROWS, Pool, same
from test_gpu_pages import DEV, gen, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def parents_of(r, b, t):
    return [[-1] + [max(0, i - r.randint(1, 4)) for i in range(1, t)] for _ in range(b)]


def masks_of(parents, t):
    out = []
    for row in parents:
        m = []
        for i, p in enumerate(row):
            m.append(1 << i | (m[p] if p >= 0 else 0))
        out.append([x - (1 << 64) if x >> 63 else x for x in m])
    return torch.tensor(out, dtype=torch.int64)


@pytest.mark.parametrize("cache,rows,heads,h,hs,page,t,draft", [("int8", "fp32", 4, 2, 64, 64, 7, None), ("e4m3", "bf16", 6, 1, 48, 128, 13, "bf16"),
                                                                ("int8", "bf16", 4, 4, 128, 64, 33, "fp32")])
def test_drafted_steps(cache, rows, heads, h, hs, page, t, draft):
    """seven steps of five sequences: trees whose likely tokens are the target's, two sequences that end or are shared at a time"""
    g, r = gen(t), random.Random(t)
    b, layers, vocab = 5, 2, 97
    per = -(-(4 * page + 70) // page)
    pages = b * per - 3
    pool = Pool(layers, pages, h, page, hs, cache, g)
    lens, table, refs = [0, 1, page - 3, page, 2 * page + 63], [[-1] * per for _ in range(b)], [0] * pages
    ref.reserve(pool, table, refs, [0] * b, lens, per * page)
    tensors = pool.tensors()
    d_table, d_lens, d_refs = ints(table), ints(lens), ints(refs)
    head = torch.randn(heads * hs, vocab, generator=g).to(DEV)
    for step in range(7):
        n = [t, 1, t, 0, r.randint(1, t)] if step % 3 == 1 else [t] * b
        parents = parents_of(r, b, t)
        mask, scale, d_n = masks_of(parents, t), hs ** -0.5, ints(n)
        new = []
        for layer in range(layers):
            q, kn, vn = (torch.randn(b, t, x, hs, generator=g).to(ROWS[rows]) for x in (heads, h, h))
            new.append((kn, vn))
            out = pkg().page_attention(q.to(DEV), *[x[layer] for x in tensors], d_table, d_lens, kn.to(DEV), vn.to(DEV), d_n, mask.to(DEV))
            test_gpu_page_attention.check(pool, table, q, kn, vn, lens, n, mask.numpy().view("uint64"), scale, out, layer)
        x = (out.float().reshape(b, t, -1) @ head) * (3.0 / hs ** 0.5)
        probs = torch.softmax(x + 0.5 * torch.randn(b, t, vocab, generator=g).to(DEV), -1).to(ROWS[draft]) if draft else None
        like = (torch.softmax(x, -1) if probs is None else probs.float()).cpu()
        tokens = torch.tensor([[int(torch.multinomial(like[i, max(0, parents[i][j])], 1, generator=g)) for j in range(t)] for i in range(b)],
                              dtype=torch.int32)
        coins = torch.rand(b, t, generator=g)
        got = pkg().draft_accept(x, tokens.to(DEV), coins.to(DEV), ints(parents), d_n, probs, 1.0)
        test_gpu_accept.check(x.cpu(), None if probs is None else probs.cpu(), tokens, parents, coins, n, 1.0, got)
        d_kept, d_path = got[:2]
        kept, path = d_kept.tolist(), d_path.tolist()
        there = pkg().page_reserve(*tensors, d_table, d_refs, d_lens, d_kept, max_n=t)
        want = ref.reserve(pool, table, refs, lens, kept, t)
        assert tuple(there.tolist()) == want and want[0] == 1
        for layer, (kn, vn) in enumerate(new):
            pkg().page_write(kn.to(DEV), vn.to(DEV), *[x[layer] for x in tensors], d_table, d_lens, d_kept, d_path, d_refs)
            ref.write(pool, kn, vn, table, lens, kept, path, refs, layer)
        d_lens += d_kept
        lens = [a + k for a, k in zip(lens, kept)]
        if step % 2:
            to = r.sample(range(b), 2)
            source = [r.choice([-1, *range(b)]), -1 if max(lens) > 3 * page else r.randrange(b)]
            pkg().page_fork(d_table, d_lens, d_refs, ints(to), ints(source), page)
            ref.fork(table, lens, refs, to, source, page)
        if step % 3 == 2:
            moved = pkg().page_compact(*tensors, d_table, d_refs)
            assert tuple(moved.tolist()) == tuple(ref.compact(pool, table, refs))
        assert d_table.tolist() == table and d_lens.tolist() == lens and d_refs.tolist() == refs
        pool.compare(tensors, [i for i, x in enumerate(refs) if x > 0])


class Served:
    """The state of one batch on the GPU and the buffers that its steps read."""

    def __init__(self, seed, cache="int8", rows="bf16", draft=True):
        g, r = gen(seed), random.Random(seed)
        self.b, self.t, self.vocab, self.page, self.layers, h, hs, heads = 3, 9, 5001, 64, 2, 2, 64, 4
        per, pages = 6, 16
        pool = Pool(self.layers, pages, h, self.page, hs, cache, g)
        lens, table, refs = [70, 64, 3], [[-1] * per for _ in range(self.b)], [0] * pages
        ref.reserve(pool, table, refs, [0] * self.b, lens, per * self.page)
        self.pool, self.table, self.lens, self.refs = pool.tensors(), ints(table), ints(lens), ints(refs)
        kind = dict(dtype=ROWS[rows], device=DEV)
        self.q = torch.zeros(self.layers, self.b, self.t, heads, hs, **kind)
        self.kn, self.vn = (torch.zeros(self.layers, self.b, self.t, h, hs, **kind) for _ in range(2))
        self.parents = ints(parents_of(r, self.b, self.t))
        self.mask = masks_of(self.parents.tolist(), self.t).to(DEV)
        self.logits = torch.zeros(self.b, self.t, self.vocab, device=DEV)
        self.probs = torch.zeros(self.b, self.t, self.vocab, device=DEV) if draft else None
        self.tokens, self.coins = torch.zeros(self.b, self.t, dtype=torch.int32, device=DEV), torch.zeros(self.b, self.t, device=DEV)
        self.to, self.source = ints([0, 2]), ints([1, -1])

    def clone(self):
        out = object.__new__(Served)
        for k, x in vars(self).items():
            setattr(out, k, [y.clone() for y in x] if k == "pool" else x.clone() if torch.is_tensor(x) else x)
        return out

    def feed(self, seed):
        """the next step's inputs, into the same buffers"""
        g = gen(seed)
        for x in (self.q, self.kn, self.vn):
            x.copy_(torch.randn(x.shape, generator=g))
        logits = torch.randn(self.logits.shape, generator=g) * 3.0
        self.logits.copy_(logits)
        p = torch.softmax(logits + 0.3 * torch.randn(logits.shape, generator=g), -1)
        if self.probs is not None:
            self.probs.copy_(p)
        parents = self.parents.tolist()
        self.tokens.copy_(torch.tensor([[int(torch.multinomial(p[i, max(0, j)], 1, generator=g)) for j in row]
                                        for i, row in enumerate(parents)], dtype=torch.int32))
        self.coins.copy_(torch.rand(self.coins.shape, generator=g))

    def step(self):
        outs = [pkg().page_attention(self.q[i], *[x[i] for x in self.pool], self.table, self.lens, self.kn[i], self.vn[i], mask=self.mask)
                for i in range(self.layers)]
        kept, path, drawn, logp = pkg().draft_accept(self.logits, self.tokens, self.coins, self.parents, None, self.probs, 0.8)
        there = pkg().page_reserve(*self.pool, self.table, self.refs, self.lens, kept, max_n=self.t)
        for i in range(self.layers):
            pkg().page_write(self.kn[i], self.vn[i], *[x[i] for x in self.pool], self.table, self.lens, kept, path, self.refs)
        back = pkg().page_read(*[x[0] for x in self.pool], self.table, self.lens, self.t, kept)
        self.lens.add_(kept)
        pkg().page_fork(self.table, self.lens, self.refs, self.to, self.source, self.page)
        moved = pkg().page_compact(*self.pool, self.table, self.refs)
        return [*outs, kept, path, drawn, logp, there, *back, moved]

    def all(self):
        return [*self.pool, self.table, self.lens, self.refs]


def equal(a, b):
    for i, (x, y) in enumerate(zip(a, b, strict=True)):
        x, y = (z.view(torch.int8) if z.element_size() == 1 else z for z in (x, y))
        assert same(x, y), i


def same_books(a, b):
    """tables, lengths, references and what used pages hold (free ones hold what was left there: the same too)"""
    equal(a.all(), b.all())


@pytest.mark.parametrize("cache,rows,draft", [("int8", "bf16", True), ("e4m3", "fp32", False)])
def test_two_captured_steps_and_eager_ones(cache, rows, draft):
    """two graphs, each of a whole step of a state of its own; replayed in turn, with new inputs, other eager steps between"""
    begin = [Served(seed, cache, rows, draft) for seed in (1, 2)]
    eager = [s.clone() for s in begin]
    warm = begin[0].clone()
    warm.feed(99)
    warm.step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in begin:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.step())
        graphs.append(graph)
    for turn in range(5):
        for i in (0, 1) if turn % 2 == 0 else (1, 0):
            begin[i].feed(10 * turn + i)
            eager[i].feed(10 * turn + i)
            graphs[i].replay()
            want = eager[i].step()
            if turn == 2:
                torch.cuda.synchronize()
            equal(outs[i], want)
            same_books(begin[i], eager[i])


def test_streams_of_their_own():
    """two batches' steps on two streams at once: what each leaves is what it leaves alone on the default stream"""
    begin = [Served(seed) for seed in (3, 4)]
    alone = [s.clone() for s in begin]
    for i, s in enumerate(begin + alone):
        s.feed(i % 2)
    streams = [torch.cuda.Stream() for _ in begin]
    torch.cuda.synchronize()
    got = []
    for s, stream in zip(begin, streams):
        with torch.cuda.stream(stream):
            got.append([s.step(), s.step()])
    torch.cuda.synchronize()
    for s, one, g in zip(alone, begin, got):
        want = [s.step(), s.step()]
        for x, y in zip(g, want):
            equal(x, y)
        same_books(one, s)


def test_the_same_again():
    """one state's step ten times over: the same bits"""
    begin = Served(5)
    begin.feed(7)
    first = begin.clone()
    want = first.step()
    for _ in range(10):
        s = begin.clone()
        equal(s.step(), want)
        same_books(s, first)
