"""llm_page_attention held between bounds that follow from its definition in float64, where scores or values are large, small, or so
many that the tile pairs and row waves take them.

Bounds.  u = 2^-24, half a step of fp32; L the positions a row sees, |q| its largest query value.
  A score is off by at most e = (hs + 8) u |scale| sum |q k| + 2^-39 |scale| |q| sum |k| (a sum of hs products, the scales, a query's
  pieces); d the largest over the row.
  2 d up to 1/2: each weight is off by a factor of e^(2 d) at most, all else by (L + 64) u, relative to sum p |v|; a weight far below the
  block's largest by 2^-39 of that: L 2^-39 max |v|; a V scale below 2^-103 loses bits to fp32's smallest numbers: 2^-118.
  2 d above: a position whose score is 2 d + 40 below the largest has a weight of e^-40 at most.  The others' values enclose the result
  but for (L + 64) u and L e^-40 of the largest value.
Rounding to the output's type is monotone: the output lies between the two bounds rounded, whatever its type."""
import math
import random

import numpy as np
import pytest

from helpers import pkg
from pages_ref import ROWS, Pool
from test_gpu_page_attention import tree_masks
from test_gpu_pages import DEV, gen, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def check(pool, table, q, kn, vn, lens, n, mask, scale, got, layer=0):
    """returns how many rows' results the bounds determine to 1% of their largest value, and all rows"""
    b, t, heads, hs = q.shape
    group, page = heads // pool.h, pool.page
    val = [pool.values(0, layer), pool.values(1, layer)]
    got, fine, rows = got.cpu(), 0, 0
    for i in range(b):
        at = torch.arange(min(max(lens[i], 0), len(table[i]) * page))
        pages = torch.tensor(table[i])[at // page]
        there = (pages >= 0) & (pages < pool.pages)
        pages, at = pages[there], at[there] % page
        live = min(max(n[i], 0), t)
        assert (got[i, live:] == 0).all()
        for h in range(pool.h):
            k, v = val[0][pages, h, at].reshape(-1, hs), val[1][pages, h, at].reshape(-1, hs)
            sees = torch.ones(live, k.shape[0] + (live if kn is not None else 0), dtype=torch.bool)
            if kn is not None:
                bits = [(1 << (j + 1)) - 1 if mask is None else int(mask[i, j]) for j in range(live)]
                sees[:, k.shape[0]:] = torch.tensor([[bool(x >> y & 1) for y in range(live)] for x in bits], dtype=torch.bool).reshape(live, live)
                k, v = torch.cat((k, kn[i, :live, h].double())), torch.cat((v, vn[i, :live, h].double()))
            x = q[i, :live, h * group:(h + 1) * group].double().reshape(-1, hs)
            y = got[i, :live, h * group:(h + 1) * group].reshape(-1, hs)
            sees = sees.repeat_interleave(group, 0)
            some = sees.any(1)
            assert (y[~some] == 0).all()
            x, y, sees = x[some], y[some], sees[some]
            if not len(x):
                continue
            count = sees.sum(1, keepdim=True).double()
            s = (x @ k.T * scale).masked_fill(~sees, -math.inf)
            e = abs(scale) * ((hs + 8) * U * (x.abs() @ k.abs().T) + 2.0 ** -39 * x.abs().amax(1, keepdim=True) * k.abs().sum(1))
            d = e.masked_fill(~sees, 0.0).amax(1, keepdim=True)
            p = torch.softmax(s, 1)
            want, size = p @ v, p @ v.abs()
            top = torch.where(sees, v.abs().amax(1), 0.0).amax(1, keepdim=True)
            tol = (torch.expm1((2 * d).clamp(max=1.0)) + (count + 64) * U) * size + count * 2.0 ** -39 * top + 2.0 ** -118
            lo, hi = want - tol, want + tol
            for j in torch.nonzero(d[:, 0] > 0.25)[:, 0].tolist():
                near = s[j] >= s[j].max() - 2 * d[j] - 40
                slack = ((count[j] + 64) * U + count[j] * math.exp(-40)) * top[j]
                lo[j], hi[j] = v[near].amin(0) - slack, v[near].amax(0) + slack
            fine += int(((hi - lo).amax(1) <= 0.01 * top[:, 0]).sum())
            rows += len(x)
            lo, hi = lo.to(got.dtype).double(), hi.to(got.dtype).double()
            off = ~((y.double() >= lo) & (y.double() <= hi))
            assert not off.any(), (i, h, int(off.sum()), off.numel(), torch.nonzero(off)[0].tolist(), y[off][0], lo[off][0], hi[off][0])
    return fine, rows


def run(pool, table, q, lens, kn=None, vn=None, n=None, mask=None, scale=None, max_len=None, layout="plain", tensors=None):
    tensors = pool.tensors(layout, layers=False) if tensors is None else tensors
    m = None if mask is None else torch.from_numpy(mask.view(np.int64)).to(DEV)
    on = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    got = pkg().page_attention(on(q), *tensors, ints(table), ints(lens), on(kn), on(vn), n=None if n is None else ints(n), mask=m,
                               scale=scale, max_len=max_len)
    return check(pool, table, q, kn, vn, lens, [q.shape[1]] * q.shape[0] if n is None else n, mask,
                 q.shape[3] ** -0.5 if scale is None else scale, got)


TYPES = [("int8", "fp32"), ("int8", "bf16"), ("e4m3", "fp32"), ("e4m3", "bf16")]


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("q_size,k_size", [(64.0, 400.0), (8.0, 3200.0), (1.0, 1e6), (0.5, 1.0)])
def test_queries_of_one_sign_under_large_scales(cache, rows, q_size, k_size, sign):
    """a query's sum is far larger than its products with the rows, whose codes have both signs: scores of up to 1e6, below and above
    where fp32 has steps of one"""
    g, h, hs = gen(1), 2, 128
    pool = Pool(1, 6, h, 64, hs, cache, g)
    most = 16 if cache == "e4m3" else 20
    pool.code[0] = torch.randint(-most, most + 1, pool.code[0].shape, generator=g).double()
    pool.scale[0] = torch.full_like(pool.scale[0], k_size * sign)
    for _ in range(4):
        q = (q_size * (1.0 + torch.rand(1, 8, 4, hs, generator=g) / 4)).to(ROWS[rows])
        run(pool, [[5, 0, 3, 1]], q, [250])


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("q_top,k_top,scale", [(2.0 ** 121, 2.0 ** -118, None), (2.0 ** 126, 2.0 ** -123, None), (2.0 ** 121, 2.0 ** -121, -1.0),
                                               (2.0 ** 60, 2.0 ** -120, 2.0 ** 60), (2.0 ** 100, 2.0 ** -136, 2.0 ** 36),
                                               (2.0 ** -100, 2.0 ** 100, 1.0), (2.0 ** -120, 2.0 ** 112, 2.0 ** 8),
                                               (2.0 ** -130, 2.0 ** 10, 2.0 ** 120), (2.0 ** 100, 2.0 ** 25, 2.0 ** -125),
                                               (2.0 ** 115, 2.0 ** -143, 2.0 ** 30), (2.0 ** -113, 2.0 ** 126, 2.0 ** -12)])
def test_scores_of_large_and_small_factors(cache, rows, q_top, k_top, scale):
    """a query, a block's scale and the softmax scale of which two multiplied would leave fp32's range, and all three do not"""
    g, h, hs = gen(2), 2, 64
    pool = Pool(1, 8, h, 64, hs, cache, g)
    pool.code[0] = (pool.code[0] / (32 if cache == "e4m3" else 8)).round().clamp(-15, 15)
    pool.scale[0] = (torch.exp(0.5 * torch.randn(pool.scale[0].shape, generator=g)) / 8 * k_top).float()
    q = (torch.randn(2, 3, 8, hs, generator=g).clamp(-3.5, 3.5) / 4 * q_top).to(ROWS[rows])
    fine, all_ = run(pool, [[5, 0, 3, 1], [7, 2, 4, 6]], q, [250, 64], scale=scale)
    assert fine == all_


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("top", [2.0 ** 119, 2.0 ** 121])
@pytest.mark.parametrize("slope", [0.0, 0.15, 0.3, 4.0, -4.0])
def test_values_whose_scale_is_near_the_largest(cache, rows, top, slope):
    """values up to 2^121 under scores that rise or fall from block to block; few enough that their sums stay below 2^127"""
    g, h, hs = gen(3), 1, 64
    pool = Pool(1, 8, h, 64, hs, cache, g)
    pool.code[1] = torch.randint(-3 if top < 2.0 ** 120 else -1, 2, pool.code[1].shape, generator=g).double()
    pool.scale[1] = torch.full_like(pool.scale[1], top)
    pool.code[0][..., 0] = 8.0
    pool.code[0][..., 1:] = 0.0
    pool.scale[0][0, :, 0, 0] = 0.5 + torch.arange(8) * slope
    pool.scale[0][0, :, 0, 0] -= pool.scale[0][0, :, 0, 0].min() - 0.5
    q = torch.ones(1, 2, 2, hs).to(ROWS[rows])
    for lens in ([20], [500]):
        run(pool, [list(range(8))], q, lens, scale=1.0)


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("hs", [64, 128, 192])
@pytest.mark.parametrize("lens", [[2, 3, 5], [64, 67, 200]])
def test_weights_hold_what_fp32_sums_need(cache, rows, hs, lens):
    """nearly equal weights, of few positions: the bounds are narrow, and an output may be the other neighbour only where the exact
    result is next to the border between two"""
    g, h, b, heads = gen(4 + hs), 2, len(lens), 16
    pool = Pool(1, 4 * b, h, 64, hs, cache, g)
    q = (torch.randn(b, 4, heads, hs, generator=g) * 0.05).to(ROWS[rows])
    table = [[4 * i + j for j in range(4)] for i in range(b)]
    fine, all_ = run(pool, table, q, lens)
    assert fine == all_


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("side", [0, 1])
def test_scales_that_are_not_finite(cache, rows, what, side):
    """a block with such a scale makes all those NaN that see its positions, of its head, and changes no bit of others"""
    g, h, hs = gen(5), 2, 64
    pool = Pool(1, 5, h, 64, hs, cache, g)
    tensors, table, lens = pool.tensors(layers=False), ints([[2, 0], [3, 1]]), ints([90, 70])
    q = torch.randn(2, 3, 6, hs, generator=g).to(ROWS[rows]).to(DEV)
    clean = pkg().page_attention(q, *tensors, table, lens)
    for page in (2, 0):
        old = tensors[2 + side][page, 1].clone()
        tensors[2 + side][page, 1] = what
        got = pkg().page_attention(q, *tensors, table, lens)
        tensors[2 + side][page, 1] = old
        assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :, :3], clean[0, :, :3])
        assert got[0, :, 3:].isnan().all()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("by", [6.0, 20.0])
def test_blocks_of_very_different_scales_choose_the_largest(cache, rows, by):
    """scales from 2^-80 to 2^80: of most rows one position has all the weight, or a few"""
    g, h, hs = gen(6), 2, 64
    fine = all_ = 0
    for t in (1, 5):
        pool = Pool(1, 12, h, 64, hs, cache, g)
        pool.scale[0] *= torch.exp(by * torch.randn(pool.scale[0].shape, generator=g))
        q, kn, vn = (torch.randn(1, t, x, hs, generator=g).to(ROWS[rows]) for x in (6, h, h))
        a, b = run(pool, [list(range(12))], q, [700], kn, vn)
        fine, all_ = fine + a, all_ + b
    assert fine >= 0.5 * all_


@pytest.mark.parametrize("cache,rows", [("int8", torch.float32), ("e4m3", torch.bfloat16)])
def test_new_rows_whose_tokens_lie_far_apart(cache, rows):
    """more than 16 MiB from token to token"""
    g, b, t, heads, h, hs = gen(2), 2, 18, 4, 2, 64
    pool = Pool(1, 4, h, 64, hs, cache, g)
    q, kn, vn = (torch.randn(b, t, x, hs, generator=g).to(rows) for x in (heads, h, h))
    far = torch.zeros(t, (20 << 20) // rows.itemsize, dtype=rows, device=DEV)
    on = []
    for i, x in enumerate((kn, vn)):
        y = far[:, i * 4096:i * 4096 + b * h * hs].view(t, b, h, hs).transpose(0, 1)
        y.copy_(x)
        on.append(y)
    tensors, table, lens = pool.tensors(layers=False), [[3, 1], [0, 2]], [100, 7]
    want = pkg().page_attention(q.to(DEV), *tensors, ints(table), ints(lens), kn.to(DEV), vn.to(DEV))
    assert torch.equal(want, pkg().page_attention(q.to(DEV), *tensors, ints(table), ints(lens), *on))
    run(pool, table, q, lens, kn, vn, tensors=tensors)


# ---- tile pairs and row waves: the host's bound of the lengths chooses them, so that short contexts reach them

def work_bytes(h, rows, hs, b, most, max_n, block_rows, least):
    """what a call's work memory has where its row blocks are of so many rows, from how positions are cut"""
    row_blocks = -(-rows // block_rows)
    one, both = max(32 // row_blocks, 1) * 8, max(64 // row_blocks, 1) * 8
    steps = -(-most // 64) + -(-max_n // 16)
    sizes = set()
    for cap in (one, both):
        if b == 1:
            cap = max(min(cap // h, -(-steps // least), 128), 1) * h
        whole = cap <= b * h or steps <= 3 * least or (b > 1 and cap == one)
        sizes.add(0 if whole else cap * rows * (hs + 2) * 4 + b * h * 8)
    return sizes - {0}


# (kv heads, heads, head size, positions' bound, lengths, tokens, live ones, whether waves take rows)
PAIRS = [
    (4, 28, 128, 16000, [300], 37, None, False),
    (4, 28, 128, 16000, [0], 37, None, False),
    (1, 5, 128, 170000, [130], 16, None, False),           # 80 rows: the last pair's second tile has none
    (1, 3, 64, 240000, [1000], 33, None, False),           # 99 rows: the last pair has three
    (2, 12, 48, 70000, [200, 0, 65], 11, [11, 5, 0], False),
    (1, 7, 112, 52000, [64, 700, 1, 0], 10, [10, 10, 3, 1], False),
    (4, 28, 128, 30000, [500], 64, None, True),
    (4, 28, 128, 8192, [300, 0, 64, 129], 64, [64, 64, 2, 0], True),
    (2, 14, 64, 54000, [128, 600], 64, [19, 64], True),    # 133 rows: of the last row block one wave has five, the others none
    (1, 9, 96, 90000, [900, 5, 64], 21, [15, 21, 1], True),
    (1, 64, 64, 510000, [200], 3, None, True),
]


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("h,heads,hs,most,lens,t,n,by_rows", PAIRS)
def test_tile_pairs(cache, rows, h, heads, hs, most, lens, t, n, by_rows):
    """with masks, own rows, unseen places that are not finite, in a pool that lies apart"""
    g, r, b = gen(7 + t), random.Random(t), len(lens)
    page = 256
    per, have = -(-most // page), [-(-x // page) for x in lens]
    pages = sum(have) + 2
    pool = Pool(1, pages, h, page, hs, cache, g)
    ids = iter(torch.randperm(pages, generator=g).tolist())
    table = [[next(ids) if j < have[i] else -1 for j in range(per)] for i in range(b)]
    q, kn, vn = (torch.randn(b, t, x, hs, generator=g).to(ROWS[rows]) for x in (heads, h, h))
    mask, live = tree_masks(r, b, t), [t] * b if n is None else n
    tensors = pool.tensors("wide", layers=False)
    nan = 0x7F if cache == "e4m3" else -128
    spare = list(ids)
    for pg in spare:
        tensors[2][pg], tensors[3][pg] = math.nan, math.inf
    for i in range(b):
        for at in range(lens[i], -(-lens[i] // 64) * 64):
            pg, blk = table[i][at // page], at % page // 64
            tensors[0].view(torch.int8)[pg, :, at % page] = nan
            tensors[1].view(torch.int8)[pg, :, blk, :, at % 64] = nan
        kn[i, live[i]:], vn[i, live[i]:], q[i, live[i]:] = math.nan, math.inf, math.nan
    # these sizes are of the kernels that this test is for, not of one tile a wave, nor of waves over positions
    c = pkg()._pages(*tensors)[0]
    need = pkg().lib().llm_page_attention_work(c, b, heads, t, most)
    size = lambda block, least: work_bytes(h, heads // h * t, hs, b, most, t, block, least)  # noqa: E731
    assert need in size(128 if by_rows else 32, 2 if by_rows else 4)
    assert need not in size(16, 4) and not (by_rows and need in size(32, 4))
    run(pool, table, q, lens, kn, vn, n, mask, max_len=most, tensors=tensors)


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("b,h,heads,hs,t", [(520, 2, 14, 64, 3), (160, 4, 8, 112, 20), (40, 4, 28, 64, 64)])
def test_tile_pairs_without_slices(cache, rows, b, h, heads, hs, t):
    """more than 512 sequences are not cut, nor those whose heads are as many as the slices; the last ones' waves take rows"""
    g = gen(8)
    lens = [(i * 37) % 90 for i in range(b)]
    pool = Pool(1, 40, h, 64, hs, cache, g)
    table = [[i % 40, (i + 7) % 40] + [-1] * 126 for i in range(b)]
    q, kn, vn = (torch.randn(b, t, x, hs, generator=g).to(ROWS[rows]) for x in (heads, h, h))
    n = [t - i % 3 for i in range(b)]
    tensors = pool.tensors(layers=False)
    c = pkg()._pages(*tensors)[0]
    most = 128 * 64
    assert pkg().lib().llm_page_attention_work(c, b, heads, t, most) == 0
    assert heads // h * t > 16 and -(-(heads // h * t) // 16) * b * h * 128 * (-(-hs // 64) * 64) > 6e6
    run(pool, table, q, lens, kn, vn, n, max_len=most, tensors=tensors)
