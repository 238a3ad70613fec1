"""Pages of a cache written and read, shared, taken, freed and moved (llm_page_write, llm_page_read, llm_page_fork,
llm_page_reserve, llm_page_compact) against their definitions in plain loops and float64.  No tolerances: codes, scales, tables
and counts are those of the definition, and a value read is code times scale, rounded once."""
import math
import random

import pytest

import pages_ref as ref
from helpers import pkg
from pages_ref import ROWS, Pool, same

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows_of(g, b, t, h, hs, kind, spread=1.0):
    return [(torch.randn(b, t, h, hs, generator=g) * torch.exp(spread * torch.randn(b, t, h, 1, generator=g))).to(ROWS[kind])
            for _ in range(2)]


# ---- rows ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("hs,h,page,layout", [(16, 1, 64, "plain"), (48, 6, 64, "heads"), (64, 2, 128, "wide"),
                                              (80, 3, 256, "plain"), (128, 4, 128, "heads"), (256, 1, 64, "wide"),
                                              (176, 2, 256, "plain")])
def test_rows_written_and_read(cache, rows, hs, h, page, layout):
    """ragged sequences over old rows, in the middle of blocks, across pages, past the table and before it, without a page"""
    g, t = gen(hs + page), 150
    b, per = 7, 3 * 256 // page
    pages = b * per + 2
    pool = Pool(2, pages, h, page, hs, cache, g)
    ids = torch.randperm(pages, generator=g).tolist()
    table = [[ids[i * per + j] for j in range(per)] for i in range(b)]
    table[3][1], table[2][1] = pages, -1  # (no page)
    pos, n = [0, 63, 64, page - 70, per * page - 20, -5, 1], [150, 1, 64, 149, 150, 150, 0]
    k, v = rows_of(g, b, t, h, hs, rows)
    tensors = pool.tensors(layout)
    layer = [x[1] for x in tensors]
    pkg().page_write(k.to(DEV), v.to(DEV), *layer, ints(table), ints(pos), ints(n))
    ref.write(pool, k, v, table, pos, n, layer=1)
    pool.compare(tensors)
    at, count = [0, 1, 60, page - 70, per * page - 40, -9, 0], [150, 70, 0, 150, 150, 20, 1]
    want = ref.read(pool, table, at, count, t, layer=1)
    got = pkg().page_read(*layer, ints(table), ints(at), t, ints(count))
    half = pkg().page_read(*layer, ints(table), ints(at), t, ints(count), dtype=torch.bfloat16)
    for side in range(2):
        assert same(got[side], want[side].float())
        assert same(half[side], want[side].float().to(torch.bfloat16))
    # into rows that are there already, those of all heads and tokens apart
    out = [torch.full((b, t, 2 * h, hs), 7.0, device=DEV)[:, :, ::2] for _ in range(2)]
    pkg().page_read(*layer, ints(table), ints(at), t, ints(count), out=out)
    for side in range(2):
        assert same(out[side], torch.where(want[2][..., None, None], want[side].float(), torch.tensor(7.0)))


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_rows_one_at_a_time(cache):
    """a block that grows by a token a call, its largest value rising and falling: the scale is doubled, never cut, and a value
    of int8 is off by at most one step of the last scale: half a step of every scale it has had, each at most half the next"""
    g, hs, h = gen(3), 32, 2
    pool = Pool(1, 2, h, 64, hs, cache)
    tensors = pool.tensors(layers=False)
    table, scales = [[1]], []
    size = [1.0, 0.5, 3.0, 3.0, 1e-3, 100.0, 90.0, 0.0, 1e4, 1.0, 1e30, 1e-30] + [1.0] * 52
    x = [torch.randn(1, 64, h, hs, generator=g) * torch.tensor(size)[:, None, None] for _ in range(2)]
    for i in range(64):
        k, v = x[0][:, i:i + 1], x[1][:, i:i + 1]
        pkg().page_write(k.to(DEV), v.to(DEV), *tensors, ints(table), ints([i]))
        ref.write(pool, k, v, table, [i], [1])
        scales.append(tensors[2][1].cpu().clone())
    pool.compare(tensors)
    assert all(bool((b >= a).all()) for a, b in zip(scales, scales[1:]))
    if cache == "int8":
        for side in range(2):
            step = pool.scale[side][0, 1].double()[:, 0, None, None]
            err = (pool.values(side)[1] - x[side][0].permute(1, 0, 2).double()).abs()
            assert bool((err <= step * (1 + 2.0 ** -20)).all())
    # begun again at its first position, a block forgets its scale
    k, v = x[0][:, :1], x[1][:, :1]
    pkg().page_write(k.to(DEV), v.to(DEV), *tensors, ints(table), ints([0]))
    ref.write(pool, k, v, table, [0], [1])
    pool.compare(tensors)
    assert float(tensors[2][1].max()) < 1.0


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_rows_at_the_borders(cache):
    """zeros, the smallest and the largest values, exact halves between codes, infinities and NaN; old scales of zero, below zero
    and NaN"""
    hs, top = 64, ref.TOP[cache]
    rows = torch.zeros(10, 1, 1, hs)
    rows[1, 0, 0, 3] = 1e-45
    rows[2, 0, 0] = torch.linspace(-3e38, 3e38, hs)
    rows[3, 0, 0] = torch.arange(hs) - 31.5
    rows[3, 0, 0, 0] = top
    rows[4, 0, 0, 5] = math.inf
    rows[5, 0, 0, 6] = math.nan
    rows[6, 0, 0] = 1e-39 * torch.linspace(-1, 1, hs)
    rows[7, 0, 0] = torch.linspace(-2, 2, hs)
    rows[8, 0, 0] = torch.linspace(-2, 2, hs)
    rows[9, 0, 0] = torch.linspace(-2, 2, hs)
    pool = Pool(1, 10, 1, 64, hs, cache, gen(1))
    table = [[i] for i in range(10)]
    for start in (0, 9):
        for old in (None, 0.0, -0.01, math.nan):
            if old is not None:
                for s in pool.scale:
                    s[0, 7:] = old
            tensors = pool.tensors(layers=False)
            pkg().page_write(rows.to(DEV), rows.to(DEV), *tensors, ints(table), ints([start] * 10))
            ref.write(pool, rows, rows, table, [start] * 10, [1] * 10)
            pool.compare(tensors)


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_rows_of_kept_paths(cache, rows):
    """the accepted tokens of a tree, some of them twice, one that is none; pages that are shared or free stay as they are"""
    g, b, t, h, hs = gen(9), 4, 21, 2, 64
    pool = Pool(1, 9, h, 64, hs, cache, g)
    table, pos, n = [[0, 1], [2, 3], [4, 5], [6, 7]], [60, 40, 62, 0], [9, 21, 5, 3]
    refs = [1, 1, 1, 0, 2, 1, 1, 1, 0]
    path = torch.randint(0, t, (b, t), generator=g).sort(1)[0]
    path[3, 1], path[0, 2] = -1, t
    k, v = rows_of(g, b, t, h, hs, rows)
    tensors = pool.tensors(layers=False)
    pkg().page_write(k.to(DEV), v.to(DEV), *tensors, ints(table), ints(pos), ints(n), path=path.int().to(DEV), refs=ints(refs))
    ref.write(pool, k, v, table, pos, n, path.tolist(), refs)
    pool.compare(tensors)


def test_rows_of_other_strides_and_long_prompts():
    """rows of all layers and heads together, read from a slice; a prompt of several pages at once, then its last part again"""
    g, b, t, h, hs = gen(4), 2, 700, 3, 96
    pool = Pool(1, 40, h, 128, hs, "int8", g)
    table = [list(range(8)), list(range(20, 28))]
    wide = torch.randn(b, t, 2, h, 2 * hs, generator=g)
    k, v = wide[:, :, 0, :, :hs], wide[:, :, 1, :, hs:]
    tensors = pool.tensors("heads", layers=False)
    on = wide.to(DEV)
    for pos, n in (([0, 100], [700, 613]), ([690, 690], [10, 7])):
        pkg().page_write(on[:, :, 0, :, :hs], on[:, :, 1, :, hs:], *tensors, ints(table), ints(pos), ints(n))
        ref.write(pool, k, v, table, pos, n)
        pool.compare(tensors)


def test_pages_far_apart():
    """pages and layers more than 4 GiB apart"""
    h, hs, page = 2, 64, 64
    big = torch.empty(2, 3, h, (1 << 31) // h // hs, hs, dtype=torch.int8, device=DEV)  # 2 GiB a page
    k = big[:, :, :, :page]
    far = torch.empty(2, 3, h, (1 << 31) // h // hs // 64, hs, 64, dtype=torch.int8, device=DEV)
    v = far[:, :, :, :1]
    ks, vs = (torch.zeros(2, 3, h, 1, device=DEV) for _ in range(2))
    pool = Pool(2, 3, h, page, hs, "int8")
    for x in (k, v):
        x.zero_()
    g = gen(2)
    rows = rows_of(g, 1, 64, h, hs, "fp32")
    table, refs, lens = ints([[2]]), ints([0, 0, 1]), ints([0])
    P = pkg()
    for layer in range(2):
        P.page_write(*(x.to(DEV) for x in rows), k[layer], v[layer], ks[layer], vs[layer], table, lens)
        ref.write(pool, *rows, [[2]], [0], [64], layer=layer)
    pool.compare([k, v, ks, vs])
    host, counts = [[2]], [0, 0, 1]
    assert P.page_compact(k, v, ks, vs, table, refs).tolist() == list(ref.compact(pool, host, counts))
    pool.compare([k, v, ks, vs])
    assert table.tolist() == host == [[0]] and refs.tolist() == counts


# ---- tables --------------------------------------------------------------------------------------------------------


class Both:
    """a pool, its tables and counts on the device and in plain lists, and the same calls on both"""

    def __init__(self, seqs, per, pages, page=64, layers=2, h=2, hs=16, cache="int8", layout="plain", seed=0):
        self.pool = Pool(layers, pages, h, page, hs, cache, gen(seed))
        self.dev = self.pool.tensors(layout)
        self.table, self.refs, self.lens = [[-1] * per for _ in range(seqs)], [0] * pages, [0] * seqs
        self.d_table, self.d_refs, self.d_lens = ints(self.table), ints(self.refs), ints(self.lens)

    def fork(self, to, source):
        pkg().page_fork(self.d_table, self.d_lens, self.d_refs, ints(to), ints(source), self.pool.page)
        ref.fork(self.table, self.lens, self.refs, to, source, self.pool.page)

    def reserve(self, n, most=None):
        got = pkg().page_reserve(*self.dev, self.d_table, self.d_refs, self.d_lens, ints(n), max_n=most)
        want = ref.reserve(self.pool, self.table, self.refs, self.lens, n, most or 1 << 30)
        assert tuple(got.tolist()) == want
        return want

    def grow(self, n):
        self.lens = [a + b for a, b in zip(self.lens, n)]
        self.d_lens.copy_(ints(self.lens))

    def compact(self):
        got = pkg().page_compact(*self.dev, self.d_table, self.d_refs)
        assert tuple(got.tolist()) == ref.compact(self.pool, self.table, self.refs)

    def check(self):
        assert self.d_table.tolist() == self.table
        assert self.d_refs.tolist() == self.refs
        assert self.d_lens.tolist() == self.lens
        self.pool.compare(self.dev)
        count = [0] * len(self.refs)
        for row in self.table:
            for e in row:
                if e >= 0:
                    count[e] += 1
        assert count == self.refs


@pytest.mark.parametrize("page,layout,cache,h,hs", [(64, "plain", "int8", 2, 16), (128, "heads", "e4m3", 3, 48),
                                                    (256, "wide", "int8", 1, 128)])
@pytest.mark.parametrize("seed", range(3))
def test_batches_that_come_and_go(page, layout, cache, h, hs, seed):
    """sequences that grow, are forked, end and are compacted, in random order"""
    r = random.Random(seed)
    seqs, per = 9, 5
    x = Both(seqs, per, 32, page, 2, h, hs, cache, layout, seed)
    for _ in range(30):
        what = r.choice(["grow", "grow", "grow", "fork", "end", "compact"])
        if what == "grow":
            n = [min(r.choice([0, 1, 1, r.randint(1, page), r.randint(1, 2 * page)]), per * page - a) for a in x.lens]
            if x.reserve(n, r.choice([None, max(max(n), 1)]))[0]:
                x.grow(n)
        elif what == "fork":
            k = r.randint(1, seqs)
            x.fork([r.randint(-1, seqs) for _ in range(k)], [r.randint(-1, seqs) for _ in range(k)])
        elif what == "end":
            x.fork([r.randrange(seqs)], [-1])
        else:
            x.compact()
        x.check()


def test_beams_follow_their_parents():
    """a permutation, beams that all come from one, the last owner's page kept in place"""
    x = Both(4, 3, 12)
    x.reserve([100, 0, 0, 0])
    x.grow([100, 0, 0, 0])
    x.fork([1, 2, 3], [0, 0, 0])
    x.check()
    assert x.refs[:2] == [4, 4]
    assert x.reserve([1, 1, 1, 1], 1) == (1, 3)  # three copies, the last keeps the shared one
    x.grow([1, 1, 1, 1])
    x.check()
    assert x.table[3][1] == 1 and x.refs[1] == 1
    x.fork([0, 1, 2, 3], [3, 2, 0, 0])
    x.check()
    assert x.reserve([0, 1, 1, 0], 1) == (1, 1)
    x.check()
    x.fork([0, 1, 2, 3, 0], [1, 0, 3, 2, 0])  # 0 is named again: its first entry does nothing
    x.check()


def test_room_that_is_not_there():
    """everything or nothing: too few pages, a sequence past its row; then less is asked for"""
    x = Both(3, 2, 4)
    assert x.reserve([65, 65, 1]) == (0, 5)
    x.check()
    assert x.reserve([129, 1, 1])[0] == 0
    x.check()
    assert x.reserve([65, 1, 1]) == (1, 4)
    x.grow([65, 1, 1])
    assert x.reserve([0, 0, 0], 1) == (1, 0)
    assert x.reserve([1, 64, 0]) == (0, 1)
    x.check()
    x.fork([2], [-1])
    assert x.reserve([1, 64, 0]) == (1, 1)
    x.check()
    x.fork([0, 1, 2], [-1, -1, -1])
    x.check()
    assert x.refs == [0] * 4
    x.compact()
    x.check()


@pytest.mark.parametrize("pages", [1, 2, 1023, 1024, 1025, 8191, 8192, 8193, 50000])
def test_pools_of_many_sizes(pages):
    """free pages found, and used ones moved, in pools around the sizes that a pass of the books takes"""
    r = random.Random(pages)
    per = min(pages, 300)
    x = Both(3, per, pages, layers=1, h=1, hs=16)
    n = [64 * (per // 3)] * 3 if per >= 3 else [64 * per, 0, 0]
    x.reserve(n)
    x.grow(n)
    x.check()
    # the pages anywhere in the pool
    where = r.sample(range(pages), sum(1 for c in x.refs if c))
    moved = dict(zip([i for i, c in enumerate(x.refs) if c], where))
    x.table = [[moved.get(e, -1) for e in row] for row in x.table]
    x.refs = [0] * pages
    for e in where:
        x.refs[e] = 1
    x.d_table.copy_(ints(x.table))
    x.d_refs.copy_(ints(x.refs))
    x.fork([1], [-1])
    x.reserve([0, 65 if pages > 2 else 0, 0])
    x.check()
    x.compact()
    x.check()


def test_wide_tables():
    """more entries, and more sequences, than a workgroup has threads"""
    x = Both(1100, 3, 4000, layers=1, h=1, hs=16)
    n = [1 + (i * 29) % 150 for i in range(1100)]
    x.reserve(n, 160)
    x.grow(n)
    x.check()
    x.fork(list(range(0, 1100, 2)), [(i * 7) % 1100 for i in range(0, 1100, 2)])
    x.check()
    x.reserve([1 if a % 64 else 0 for a in x.lens], 1)
    x.check()


def test_nothing_to_do():
    x = Both(2, 2, 4)
    x.fork([], [])
    got = pkg().page_reserve(*x.dev, x.d_table, x.d_refs, x.d_lens, ints([1, 1]), max_n=0)
    assert got.tolist() == [1, 0]
    x.compact()
    x.check()
    rows = torch.zeros(2, 0, 2, 16, device=DEV)
    layer = [y[0] for y in x.dev]
    pkg().page_write(rows, rows, *layer, x.d_table, x.d_lens)
    assert pkg().page_read(*layer, x.d_table, x.d_lens, 0)[0].shape == (2, 0, 2, 16)
    x.check()
