"""llm_page_attention against its definition in float64.

Tolerances.  u = 2^-24, half a step of fp32; L the positions a row sees, |q| its largest query value.
  A score is a sum of hs products and a scale: off by at most (hs + 8) u |scale| sum |q k|, the query's 22 bits (4 u) among
  the 8; a query value far below |q| is held to 2^-39 |q|: 2^-39 |scale| |q| sum |k| more.  With d their sum's largest over the
  row, a weight is off by a factor of e^(2 d), and everything else (exponentials, a weight's second fp16 piece (2 u), sums, scales,
  joins) by (L + 64) u: all relative to sum p |v|.
  A weight far below the block's largest is held to 2^-39 of that, at most 1: L 2^-39 max |v|.
  bf16 rows: the output's rounding, 2^-8 of the value; a weight over pages is one fp16 piece, off by 2^-11 at most, and so is its
  share of the sum: 2^-10 sum p |v|.  int8 codes count as code + 128 on the way, with 128 times the query's and the weights' sums
  taken off again: sums of up to 255 in the place of 127 |code|, (hs + 8) u |scale| 128 s sum |q| more for a score (s the block's
  scale) and (L + 64) u 128 s sum p for a value."""
import math
import random

import numpy as np
import pytest

import pages_ref as ref
from helpers import pkg
from pages_ref import ROWS, Pool, same
from test_gpu_pages import DEV, gen, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def tree_masks(r, b, t):
    """bits of ancestors and the node itself, random parents"""
    m = np.zeros((b, t), np.uint64)
    for i in range(b):
        for j in range(t):
            parent = r.randint(-1, j - 1) if r.random() < 0.5 else j - 1
            m[i, j] = np.uint64((1 << j) | (int(m[i, parent]) if parent >= 0 else 0))
    return m


def check(pool, table, q, kn, vn, lens, n, mask, scale, got, layer=0):
    half = got.dtype == torch.bfloat16
    biased = half and pool.cache == "int8"
    b, t, heads, hs = q.shape
    group, page = heads // pool.h, pool.page
    val = [pool.values(0, layer), pool.values(1, layer)]
    worst = 0.0
    for i in range(b):
        ln = min(max(lens[i], 0), len(table[i]) * page)
        there = torch.tensor([0 <= table[i][p // page] < pool.pages for p in range(ln)], dtype=torch.bool)
        pg = [table[i][p // page] for p in range(ln) if there[p]]
        off = [p % page for p in range(ln) if there[p]]
        live = min(max(n[i], 0), t)
        for h in range(pool.h):
            k, v = val[0][pg, h, off].reshape(-1, hs), val[1][pg, h, off].reshape(-1, hs)
            old = k.shape[0]
            size_k, size_v = ((pool.scale[side][layer][pg, h].abs().double()[range(old), [o // 64 for o in off]] if biased and old else
                               torch.zeros(old, dtype=torch.float64)) for side in range(2))
            if kn is not None:
                k, v = torch.cat((k, kn[i, :live, h].double())), torch.cat((v, vn[i, :live, h].double()))
            for j in range(live):
                sees = torch.ones(k.shape[0], dtype=torch.bool)
                if kn is not None:
                    bits = (1 << (j + 1)) - 1 if mask is None else int(mask[i, j])
                    sees[old:] = torch.tensor([bool((bits >> x) & 1) for x in range(live)], dtype=torch.bool)
                ks, vs = k[sees], v[sees]
                for x in range(h * group, (h + 1) * group):
                    y = got[i, j, x].double().cpu()
                    if not len(ks):
                        assert (y == 0).all()
                        continue
                    qd = q[i, j, x].double()
                    p = torch.softmax(ks @ qd * scale, 0)
                    want, size = p @ vs, p @ vs.abs()
                    if not torch.isfinite(vs).all():
                        assert y.isnan().all()
                        continue
                    d = abs(scale) * float(((hs + 8) * U * (ks.abs() @ qd.abs()) + 2.0 ** -39 * qd.abs().max() * ks.abs().sum(1)).max())
                    if biased and old:
                        d += abs(scale) * (hs + 8) * U * 128 * float(size_k.max()) * float(qd.abs().sum())
                    tol = (math.expm1(min(2 * d, 700.0)) + (len(ks) + 64) * U) * size + len(ks) * 2.0 ** -39 * float(vs.abs().max()) + 1e-37
                    if half:
                        tol = tol + 2.0 ** -8 * want.abs() + 2.0 ** -10 * size
                    if biased and old:
                        tol = tol + (len(ks) + 64) * U * 128 * float((p[:old] * size_v).sum())
                    worst = max(worst, float(((y - want).abs() / tol).max()))
                    assert ((y - want).abs() <= tol).all(), (i, j, x, worst)
        # rows behind the last token
        assert (got[i, live:] == 0).all()


def case(cache, rows, heads, h, hs, page, lens, t, n=None, masked=True, layout="plain", scale=None, own=True, seed=0, bad=False,
         spread=1.0, k_spread=None, max_len=None, spare=0, v_top=1.0):
    g, r = gen(seed + hs + t), random.Random(seed)
    b = len(lens)
    per = -(-max(max(lens), 1) // page) + spare
    pages = b * per + 2
    pool = Pool(2, pages, h, page, hs, cache, g)
    for s, by in zip(pool.scale, (spread if k_spread is None else k_spread, spread)):
        s *= torch.exp(by * torch.randn(s.shape, generator=g))
    pool.scale[1] *= v_top
    ids = torch.randperm(pages, generator=g).tolist()
    table = [[ids[i * per + j] if j * page < lens[i] else -1 for j in range(per)] for i in range(b)]
    q = torch.randn(b, t, heads, hs, generator=g).to(ROWS[rows])
    kn, vn = ((torch.randn(b, t, h, hs, generator=g) * torch.exp(torch.randn(b, t, h, 1, generator=g))).to(ROWS[rows])
              for _ in range(2))
    vn = (vn.float() * v_top).to(ROWS[rows])
    mask = tree_masks(r, b, t) if masked else None
    nn = [t] * b if n is None else n
    tensors = pool.tensors(layout)
    if bad:  # infinities and NaN wherever nothing is seen: behind lens in its block, in blocks and pages behind it
        nan = 0x7F if cache == "e4m3" else -128
        for i in range(b):
            for at in range(max(lens[i], 0), -(-max(lens[i], 0) // 64) * 64):
                pg, blk = table[i][at // page], at % page // 64
                tensors[0].view(torch.int8)[1, pg, :, at % page] = nan
                tensors[1].view(torch.int8)[1, pg, :, blk, :, at % 64] = nan
        seen = {(table[i][at // page], at % page // 64) for i in range(b) for at in range(0, lens[i], 64)}
        for pg in range(pages):
            for blk in range(page // 64):
                if (pg, blk) not in seen:
                    tensors[2][1, pg, :, blk] = math.nan
                    tensors[3][1, pg, :, blk] = math.inf
        for i in range(b):
            for j in range(t):
                if j >= nn[i]:
                    kn[i, j], vn[i, j], q[i, j] = math.nan, math.inf, math.nan
    m = None if mask is None else torch.from_numpy(mask.view(np.int64)).to(DEV)
    layer = [x[1] for x in tensors]
    kw = dict(k_rows=kn.to(DEV), v_rows=vn.to(DEV)) if own else {}
    sc = hs ** -0.5 if scale is None else scale
    got = pkg().page_attention(q.to(DEV), *layer, ints(table), ints(lens), n=None if n is None else ints(n), mask=m, scale=scale,
                               max_len=max_len, **kw)
    check(pool, table, q, kn if own else None, vn if own else None, lens, nn, mask, sc, got, layer=1)
    return got


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,h,hs,page,layout", [(2, 2, 16, 64, "plain"), (6, 6, 48, 128, "heads"), (14, 2, 64, 64, "wide"),
                                                    (28, 4, 128, 128, "plain"), (5, 1, 80, 256, "heads"),
                                                    (3, 1, 160, 64, "plain"), (8, 4, 256, 64, "wide"), (4, 2, 208, 256, "plain")])
def test_trees(cache, rows, heads, h, hs, page, layout):
    case(cache, rows, heads, h, hs, page, [0, 37, 131, 300], 5, [5, 3, 4, 0], layout=layout, bad=True, spare=2)


@pytest.mark.parametrize("cache,rows,hs", [("int8", "fp32", 64), ("int8", "bf16", 128), ("e4m3", "fp32", 48),
                                           ("e4m3", "bf16", 256)])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_one_token(cache, rows, hs, length):
    case(cache, rows, 4, 2, hs, 64, [length], 1, masked=False, bad=True)


@pytest.mark.parametrize("t", [2, 16, 17, 33, 63, 64])
@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("e4m3", "bf16")])
def test_long_trees(cache, rows, t):
    case(cache, rows, 3, 1, 64, 128, [600, 63, 0], t, [t, t - 1, t])
    case(cache, rows, 14, 2, 64, 64, [200], t, masked=False)


@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("e4m3", "bf16")])
def test_tokens_without_rows_of_their_own(cache, rows):
    """over the pages only, as over another's states: nothing at all for an empty sequence"""
    got = case(cache, rows, 6, 2, 64, 64, [100, 0, 1], 3, [3, 3, 2], own=False)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-6, 3.0, -2.0])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_scales(cache, scale):
    case(cache, "fp32", 4, 2, 64, 64, [130, 5], 3, scale=scale)
    case(cache, "bf16", 4, 2, 64, 64, [130, 5], 3, scale=scale)


@pytest.mark.parametrize("v_top", [2.0 ** 110, 2.0 ** -100])
@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("int8", "bf16"), ("e4m3", "fp32"), ("e4m3", "bf16")])
def test_values_near_the_ends_of_fp32(cache, rows, v_top):
    """values up to about 2^110 (their scale 2^110, 0.02 and the codes), whose sums with weights up to 1 stay below 2^127"""
    case(cache, rows, 4, 2, 64, 64, [700, 64, 3], 3, spread=0.0, v_top=v_top)
    if v_top > 1.0:
        case(cache, rows, 28, 4, 128, 64, [9000], 33, spread=0.0, v_top=v_top)


@pytest.mark.parametrize("spread", [6.0, 20.0])
@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("e4m3", "bf16")])
def test_blocks_of_very_different_scales(cache, rows, spread):
    case(cache, rows, 4, 2, 64, 64, [500, 64], 2, spread=spread)
    case(cache, rows, 4, 2, 64, 64, [500, 64], 2, spread=spread, k_spread=0.0)


@pytest.mark.parametrize("cache,heads,h,hs,page", [("int8", 28, 4, 128, 64), ("e4m3", 14, 2, 64, 256), ("int8", 6, 6, 48, 128)])
def test_long_contexts(cache, heads, h, hs, page):
    """several thousand positions, and a bound of the lengths that is too low"""
    a = case(cache, "fp32", heads, h, hs, page, [4990], 3)
    b = case(cache, "fp32", heads, h, hs, page, [4990], 3, max_len=10)
    assert float((a - b).abs().max()) < 1e-4 * float(a.abs().max())
    case(cache, "bf16", heads, h, hs, page, [2400, 77, 0, 1300], 1, masked=False, bad=True)


@pytest.mark.parametrize("b,h,longest", [(2, 1, 12000), (3, 2, 5000), (63, 1, 1500), (64, 3, 700), (65, 1, 1500), (130, 1, 900),
                                         (511, 1, 300), (512, 1, 300), (513, 1, 300)])
def test_uneven_batches(b, h, longest):
    """one long sequence, one of every other length down to none"""
    lens = [longest if i == b // 2 else (i * 37) % 301 for i in range(b)]
    case("int8", "fp32", 2 * h, h, 16, 64, lens, 2, [1 + i % 2 for i in range(b)])


@pytest.mark.parametrize("cache,rows,heads,h,hs,lens,t", [
    ("int8", "fp32", 28, 4, 128, [1500], 37), ("int8", "bf16", 28, 4, 128, [900, 64, 7], 64),
    ("e4m3", "fp32", 64, 1, 64, [700, 0], 33), ("e4m3", "bf16", 64, 1, 32, [65], 64), ("int8", "bf16", 20, 2, 112, [640, 320], 19),
    ("int8", "fp32", 12, 1, 256, [300], 64)])
def test_many_rows(cache, rows, heads, h, hs, lens, t):
    case(cache, rows, heads, h, hs, 64, lens, t, bad=True)


def test_masks_that_leave_nothing():
    """no bit, over an empty and a filled sequence; bits of tokens that are not there"""
    g, h, hs = gen(1), 2, 64
    pool = Pool(1, 4, h, 64, hs, "int8", g)
    tensors = pool.tensors(layers=False)
    table, lens = [[-1, -1], [2, 0]], [0, 70]
    q, kn, vn = (torch.randn(2, 4, x, hs, generator=g) for x in (4, h, h))
    mask = np.array([[0, 1, 0, 1 << 63 | 2], [0, 1, 0, 5]], np.uint64)
    got = pkg().page_attention(q.to(DEV), *tensors, ints(table), ints(lens), kn.to(DEV), vn.to(DEV),
                               mask=torch.from_numpy(mask.view(np.int64)).to(DEV))
    check(pool, table, q, kn, vn, lens, [4, 4], mask, hs ** -0.5, got)
    assert (got[0, 0] == 0).all() and (got[0, 2] == 0).all() and (got[1] != 0).all()


def test_pages_that_are_not_there():
    """entries outside the pool in the middle of a sequence: their positions are not seen"""
    g, h, hs = gen(2), 1, 48
    pool = Pool(1, 6, h, 128, hs, "e4m3", g)
    table, lens = [[3, -1, 5, 6], [-7, 1 << 30, -1, -1], [0, 1, 2, 4]], [500, 300, 1 << 30]
    q, kn, vn = (torch.randn(3, 2, x, hs, generator=g).to(torch.bfloat16) for x in (5, h, h))
    got = pkg().page_attention(q.to(DEV), *pool.tensors(layers=False), ints(table), ints(lens), kn.to(DEV), vn.to(DEV))
    check(pool, table, q, kn, vn, lens, [2, 2, 2], None, hs ** -0.5, got)
    none = pkg().page_attention(q.to(DEV), *pool.tensors(layers=False), ints(table), ints([-3, 300, 0]))
    assert (none == 0).all()


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_new_rows_that_are_not_finite(rows, what):
    """a token's K or V row with one such value: no bit changes for those that do not see it, those that see its V row are NaN"""
    g, b, t, heads, h, hs = gen(3), 1, 20, 4, 2, 64
    pool = Pool(1, 3, h, 64, hs, "int8", g)
    tensors, table, lens = pool.tensors(layers=False), ints([[2, 0]]), ints([90])
    q, kn, vn = (torch.randn(b, t, x, hs, generator=g).to(ROWS[rows]).to(DEV) for x in (heads, h, h))
    mask = tree_masks(random.Random(5), b, t)
    m = torch.from_numpy(mask.view(np.int64)).to(DEV)
    clean = pkg().page_attention(q, *tensors, table, lens, kn, vn, mask=m)
    for side in range(2):
        for tok in (0, 7, 19):
            rows_ = [kn.clone(), vn.clone()]
            rows_[side][0, tok, 1, 33] = what
            got = pkg().page_attention(q, *tensors, table, lens, *rows_, mask=m)
            for i in range(t):
                sees = (int(mask[0, i]) >> tok) & 1
                assert same(got[0, i, :2], clean[0, i, :2])  # (of the other kv head)
                if not sees:
                    assert same(got[0, i, 2:], clean[0, i, 2:])
                elif side:
                    assert got[0, i, 2:].isnan().all()


def test_unseen_places_change_no_bit():
    g, h, hs = gen(4), 2, 128
    for cache in ("int8", "e4m3"):
        pool = Pool(1, 4, h, 128, hs, cache, g)
        tensors = pool.tensors(layers=False)
        q, kn, vn = (torch.randn(1, 3, x, hs, generator=g).to(DEV) for x in (8, h, h))
        args = (ints([[1, 3]]), ints([150]), kn, vn)
        a = pkg().page_attention(q, *tensors, *args)
        for x in tensors[:2]:
            x.view(torch.int8)[0] = 0x7F
            x.view(torch.int8)[2] = -1
        tensors[0].view(torch.int8)[3, :, 22:] = 0x7F
        tensors[1].view(torch.int8)[3, :, 0, :, 22:] = 0x7F
        tensors[1].view(torch.int8)[3, :, 1] = 0x7F
        for x in tensors[2:]:
            x[0], x[2], x[3, :, 1] = math.nan, math.inf, -math.inf
        assert same(a, pkg().page_attention(q, *tensors, *args))
        tensors[3][3, 1, 0] = math.nan  # a block that is seen, of one head
        got = pkg().page_attention(q, *tensors, *args)
        assert same(got[:, :, :4], a[:, :, :4]) and got[:, :, 4:].isnan().all()


def test_out_and_rows_of_other_strides():
    """q, out and the new rows in slices of wider tensors; rows behind the last token of `out` left as they were"""
    g, b, t, heads, h, hs = gen(6), 2, 4, 6, 2, 80
    pool = Pool(1, 5, h, 64, hs, "int8", g)
    tensors, table = pool.tensors("wide", layers=False), [[4, 0], [1, 3]]
    wide = torch.randn(b, t, heads + 2 * h, 2 * hs, generator=g)
    on = wide.to(DEV)
    cut = [slice(0, heads), slice(heads, heads + h), slice(heads + h, None)]
    q, kn, vn = (wide[:, :, c, hs:] for c in cut)
    out = torch.full((t, b, heads, hs + 4), 9.0, device=DEV).transpose(0, 1)[..., :hs]
    r = pkg().page_attention(on[:, :, cut[0], hs:], *tensors, ints(table), ints([100, 128]), on[:, :, cut[1], hs:],
                             on[:, :, cut[2], hs:], n=ints([2, 4]), out=out)
    assert r is out
    assert (out[0, 2:] == 9.0).all()
    got = torch.where(torch.arange(t, device=DEV)[None, :, None, None] < ints([2, 4])[:, None, None, None], out, torch.zeros(()).to(DEV))
    check(pool, table, q, kn, vn, [100, 128], [2, 4], None, hs ** -0.5, got)


@pytest.mark.parametrize("slope", [-0.05, 0.002, 0.05, 0.4])
@pytest.mark.parametrize("t,heads,length", [(1, 2, 800), (40, 14, 3000)])
def test_scores_that_rise(slope, t, heads, length):
    """every position's score above (below) the one before: a new maximum in every block"""
    h, hs, g = 1, 64, gen(8)
    pages = -(-length // 64)
    pool = Pool(1, pages, h, 64, hs, "int8", g)
    # K's first dimension is 127, the block's scale carries the slope; the others are small
    pool.code[0][0, :, 0, 0, :, 0] = 127.0
    pool.code[0][0, :, 0, 0, :, 1:] = (pool.code[0][0, :, 0, 0, :, 1:] / 64).round()
    at = torch.arange(pages, dtype=torch.float64) * 64 * slope
    pool.scale[0][0, :, 0, 0] = ((at - at.min()) / 127 + 0.01).float()
    q = torch.randn(1, t, heads, hs, generator=g) * 0.05
    q[..., 0] = math.sqrt(hs)
    kn, vn = (torch.randn(1, t, h, hs, generator=g) for _ in range(2))
    got = pkg().page_attention(q.to(DEV), *pool.tensors(layers=False), ints([list(range(pages))]), ints([length]), kn.to(DEV),
                               vn.to(DEV))
    check(pool, [list(range(pages))], q, kn, vn, [length], [t], None, hs ** -0.5, got)
