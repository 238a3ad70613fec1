"""What llm_tree_attention promises of scales, signs and unseen tokens, against the definition in float64.

Tolerances.  u = 2^-24, half a step of fp32; L the positions a row sees.
  A score, a sum of hs products with the query held to 22 bits at least (4 u), is off by at most d = (hs + 8) u |scale| max
  sum |q k|, a weight then by a factor of e^(2 d), everything else (exponential, scales, sums, joins) by (L + 64) u: all
  relative to sum p |v|.
  8-bit caches: a weight p sv is two fp16 pieces, the second a rounding of what the first leaves: 2^-12 2^-12 = u, and at most
  2^-25 where it is subnormal, with the largest |sv| that the row sees in [2^14, 2^15): L 2^-39 max |code| max |sv|.
  bf16 caches: a weight is three bf16 pieces for fp32 queries (2^-9 each: below u) and two for bf16 ones, 2^-16.
  bf16 outputs: 2^-8 of the value."""
import math

import numpy as np
import pytest

from helpers import pkg
from test_gpu_operators import CACHES, DEV, ROWS, U, cache_tensors, gen, quantized, same, tree_masks

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def put(x, cache, ctx=None, layout="heads"):
    """K or V rows (float64 [b, h, positions, hs]) as cache tensors on the device: codes, scales, the values they stand for"""
    b, h, n, hs = x.shape
    val, code, s = quantized(x, cache)
    store, _, sc, _ = cache_tensors(cache, b, h, ctx or n, hs, layout, 0.0)
    store[:, :, :n] = code.float().to(CACHES[cache]).to(DEV)
    if sc is not None:
        sc[:, :, :n] = s.to(DEV)
    return store, sc, val, code, s


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def bits(mask):
    return torch.from_numpy(np.array(mask, np.uint64).view(np.int64)).to(DEV)


def check(q, k, v, lens, mask, scale, got, cache):
    """got against float64; k and v are (values, codes, scales) of `put` on the CPU"""
    b, t, heads, hs = q.shape
    h, end = k[0].shape[1:3]
    group, at = heads // h, torch.arange(end)
    for i in range(b):
        node = at - lens[i]
        sees = torch.stack([(node < 0) | (torch.tensor([0 <= m < t and bool((int(mask[i][j]) >> m) & 1) for m in node.tolist()]))
                            for j in range(t)])
        sees = sees.unsqueeze(1).expand(t, group, end).reshape(t * group, end)
        count = sees.sum(-1, keepdim=True)
        for x in range(h):
            mine = slice(x * group, (x + 1) * group)
            qd, y = q[i, :, mine].double().cpu().reshape(t * group, hs), got[i, :, mine].double().cpu().reshape(t * group, hs)
            s = (qd @ k[0][i, x].T * scale).masked_fill(~sees, -math.inf)
            p = torch.softmax(s.masked_fill(count == 0, 0.0), -1) * (count > 0)
            want, size = p @ v[0][i, x], p @ v[0][i, x].abs()
            far = (qd.abs() @ k[0][i, x].abs().T).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
            tol = (2 * (hs + 8) * U * abs(scale) * far + (count + 64) * U) * size
            if v[2] is not None:
                big = v[1][i, x].abs().amax(-1) * v[2][i, x].double().abs()
                tol = tol + count * 2.0 ** -39 * big.expand_as(sees).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
            if cache == "bf16":
                tol = tol + (2.0 ** -16 if q.dtype == torch.bfloat16 else U) * size
            if q.dtype == torch.bfloat16:
                tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
            err = (y - want).abs()
            assert (err <= tol + 1e-37).all(), (i, x, float((err / (tol + 1e-37)).max()))


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("hs,heads,h,lens,t", [(64, 4, 2, [0, 30], 2), (128, 28, 4, [70, 6], 3), (128, 28, 4, [1800, 333], 1),
                                               (256, 2, 1, [40, 8], 5), (64, 14, 2, [90, 41], 37)])
def test_weights_of_16_bit_queries_keep_their_bits(cache, hs, heads, h, lens, t):
    """pairs of positions whose values nearly cancel: what is left of them holds a weight's low bits"""
    g = gen(hs + t)
    b, n = 2, max(lens) + t + 1
    n += n % 2
    x = [torch.randn(b, h, n, hs, generator=g).double() for _ in range(2)]
    # a pair: K alike within 2^-9, V the negative within 2^-10
    x[0][:, :, 1::2] = x[0][:, :, ::2] * (1 + 2.0 ** -9 * torch.rand(b, h, n // 2, 1, generator=g).double())
    x[1][:, :, 1::2] = -x[1][:, :, ::2] * (1 + 2.0 ** -10 * torch.rand(b, h, n // 2, 1, generator=g).double())
    q = (torch.randn(b, t, heads, hs, generator=g) * 0.1).to(torch.bfloat16)
    (k, ks, *kv), (v, vs, *vv) = (put(y, cache) for y in x)
    # every row sees both of a pair: the committed ones, and of the new tokens whole pairs (where lens is even)
    mask = [[sum(1 << m for m in range(j | 1) if m < t) | 1 << j for j in range(t)] for _ in range(b)]
    got = pkg().tree_attention(q.to(DEV), k, v, ints(lens), mask=bits(mask), k_scale=ks, v_scale=vs)
    check(q, kv, vv, lens, mask, hs ** -0.5, got, cache)


# many rows and positions enough for two row tiles a wave (8-bit caches; bf16), and few of one
SHAPES = [(64, 4, 2, 33, 6), (128, 28, 4, 70, 6), (128, 4, 2, 1500, 6), (128, 28, 4, 2000, 37), (48, 6, 6, 40, 20), (160, 3, 1, 61, 9),
          (256, 4, 2, 90, 7)]


def tree_case(cache, rows, hs, heads, h, length, t, seed=0):
    """a random tree over a filled cache with room behind it; node 1 has children, others do not see it"""
    g = gen(hs + length + t + seed)
    ctx = 40000 if t > 30 else length + t + 80
    x = [torch.randn(1, h, length + t, hs, generator=g).double() for _ in range(2)]
    q = torch.randn(1, t, heads, hs, generator=g).to(ROWS[rows])
    (k, ks, *kv), (v, vs, *vv) = (put(y, cache, ctx) for y in x)
    mask = tree_masks(g, 1, t)
    mask[0, 2] = 0b101  # (node 2 hangs on the root)
    mask[0, t - 1] &= ~np.uint64(2)
    return q, k, ks, kv, v, vs, vv, mask


def attend(q, k, ks, v, vs, length, mask, **kw):
    return pkg().tree_attention(q.to(DEV), k, v, ints([length]), mask=bits(mask), k_scale=ks, v_scale=vs, **kw)


def blind(mask, node):
    """the tokens that do not see the node"""
    return [i for i in range(mask.shape[1]) if not (int(mask[0, i]) >> node) & 1]


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("hs,heads,h,length,t", SHAPES)
def test_codes_that_are_nan_reach_their_descendants_only(rows, hs, heads, h, length, t):
    """e4m3 codes 0x7f and 0xff in the V row, or the K row, of one new token"""
    q, k, ks, kv, v, vs, vv, mask = tree_case("e4m3", rows, hs, heads, h, length, t)
    clean = attend(q, k, ks, v, vs, length, mask)
    check(q, kv, vv, [length], mask, hs ** -0.5, clean, "e4m3")
    for store in (v, k):
        for code, at in ((0x7f, hs - 1), (0xff, 5)):
            raw = store.view(torch.uint8)
            old = raw[0, :, length + 1, at].clone()
            raw[0, :, length + 1, at] = code
            dirty = attend(q, k, ks, v, vs, length, mask)
            raw[0, :, length + 1, at] = old
            for i in range(t):
                if i in blind(mask, 1):
                    assert torch.equal(dirty[0, i], clean[0, i])
                else:
                    assert dirty[0, i].isnan().all()


@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("e4m3", "fp32"), ("e4m3", "bf16"), ("bf16", "bf16"), ("fp32", "fp32")])
@pytest.mark.parametrize("t,pad", [(3, 8), (5, 64)])
def test_padded_trees_over_slots_that_were_never_written(cache, rows, t, pad):
    """a tree padded to a fixed number of nodes without masks: every byte of the slots behind it is 0xff, or 0x7f"""
    hs, heads, h, length = 128, 14, 2, 75
    q, k, ks, kv, v, vs, vv, mask = tree_case(cache, rows, hs, heads, h, length, t)
    wide = torch.zeros(1, pad, heads, hs, dtype=q.dtype)
    wide[:, :t] = q
    m = np.zeros((1, pad), np.uint64)
    m[:, :t] = mask
    clean = attend(wide, k, ks, v, vs, length, m)
    check(q, kv, vv, [length], mask, hs ** -0.5, clean[:, :t], cache)
    for byte in (0xff, 0x7f):
        for store in (k, v, ks, vs):
            if store is not None:
                store.view(torch.uint8).view(1, h, k.shape[2], -1)[:, :, length + t:] = byte
        assert torch.equal(attend(wide, k, ks, v, vs, length, m), clean)


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("hs,heads,h,length,t", SHAPES + [(64, 4, 2, 0, 1), (128, 28, 4, 9, 1)])
def test_scales_below_zero(cache, rows, hs, heads, h, length, t):
    """a value is its code times its scale, whatever the scale's sign: all below zero, and in turn"""
    q, k, ks, kv, v, vs, vv, mask = tree_case(cache, rows, hs, heads, h, length, max(t, 3))
    q, mask = q[:, :t], mask[:, :t]
    for every in (1, 2):
        signs = torch.ones(kv[2].shape[2])
        signs[::every] = -1.0
        sk, sv = kv[2] * signs, vv[2] * signs * 0.01
        ks[:, :, :sk.shape[2]], vs[:, :, :sv.shape[2]] = sk.to(DEV), sv.to(DEV)
        got = attend(q, k, ks, v, vs, length, mask)
        check(q, (kv[1] * sk.double().unsqueeze(-1), kv[1], sk), (vv[1] * sv.double().unsqueeze(-1), vv[1], sv), [length],
              mask, hs ** -0.5, got, cache)


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("hs,heads,h,length,t", SHAPES)
def test_scales_of_unseen_tokens_change_nothing(cache, rows, hs, heads, h, length, t):
    """one new token's V (and K) scale far above the others': the tokens that do not see it are the same bit for bit, those that
    do follow it"""
    q, k, ks, kv, v, vs, vv, mask = tree_case(cache, rows, hs, heads, h, length, t)
    clean = attend(q, k, ks, v, vs, length, mask)
    check(q, kv, vv, [length], mask, hs ** -0.5, clean, cache)
    for far in (2.0 ** 20, 2.0 ** 30, -2.0 ** 40, 2.0 ** 100, math.inf):
        s = vv[2].clone()
        s[:, :, length + 1] *= far
        vs[:, :, :length + t] = s.to(DEV)
        got = attend(q, k, ks, v, vs, length, mask)
        for i in blind(mask, 1):
            assert torch.equal(got[0, i], clean[0, i]), (far, i)
        if math.isfinite(far):
            check(q, kv, (vv[1] * s.double().unsqueeze(-1), vv[1], s), [length], mask, hs ** -0.5, got, cache)
    vs[:, :, :length + t] = vv[2].to(DEV)
    ks[:, :, length + 1] *= 2.0 ** 40
    got = attend(q, k, ks, v, vs, length, mask)
    for i in blind(mask, 1):
        assert torch.equal(got[0, i], clean[0, i])


@pytest.mark.parametrize("cache,rows", [("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "fp32"), ("bf16", "bf16"), ("int8", "fp32"),
                                        ("e4m3", "bf16")])
@pytest.mark.parametrize("hs,heads,h,length,t", SHAPES + [(128, 28, 4, 2500, 64)])
def test_rows_of_unseen_tokens_change_nothing(cache, rows, hs, heads, h, length, t):
    """other K and V rows of one new token, whose scores lie little or much above the others': the tokens that do not see it are
    the same bit for bit"""
    q, k, ks, kv, v, vs, vv, mask = tree_case(cache, rows, hs, heads, h, length, t)
    clean = attend(q, k, ks, v, vs, length, mask)
    for size in (0.1, 2.0, 9.0):
        # (along the first query of its own: its score, and those of its descendants', are far from the rest)
        row = q[0, 1, ::heads // h].double().view(1, h, 1, hs) * size
        code, s = quantized(row, cache)[1:]
        k[:, :, length + 1:length + 2] = code.float().to(CACHES[cache]).to(DEV)
        v[:, :, length + 1:length + 2] = (-code).float().to(CACHES[cache]).to(DEV)
        if s is not None:
            ks[:, :, length + 1:length + 2] = s.to(DEV)
        got = attend(q, k, ks, v, vs, length, mask)
        for i in blind(mask, 1):
            assert torch.equal(got[0, i], clean[0, i]), (size, i)


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", list(CACHES))
@pytest.mark.parametrize("hs,heads,h,length,t", [(64, 4, 2, 50, 5), (128, 28, 4, 3000, 2), (128, 28, 4, 2500, 37)])
@pytest.mark.parametrize("scale", [0.03, 0.5, -0.2, 0.0])
def test_scales_of_the_softmax(cache, rows, hs, heads, h, length, t, scale):
    """other scales than hs ** -0.5, below zero, and zero (the mean of what is seen), whole and in slices"""
    q, k, ks, kv, v, vs, vv, mask = tree_case(cache, rows, hs, heads, h, length, max(t, 3), 1)
    q, mask = q[:, :t], mask[:, :t]
    got = attend(q, k, ks, v, vs, length, mask, scale=scale)
    check(q, kv, vv, [length], mask, scale, got, cache)


@pytest.mark.parametrize("cache", list(CACHES))
def test_a_scale_of_zero_over_large_scores(cache):
    """0 times any score is 0: the mean, however large the products"""
    g = gen(12)
    b, h, hs, length, t, heads = 1, 2, 64, 45, 3, 4
    x = [torch.randn(b, h, length + t, hs, generator=g).double() * f for f in (2.0 ** 55, 1.0)]
    q = torch.randn(b, t, heads, hs, generator=g) * 2.0 ** 55
    (k, ks, *kv), (v, vs, *vv) = (put(y, cache) for y in x)
    mask = tree_masks(g, b, t)
    got = pkg().tree_attention(q.to(DEV), k, v, ints([length]), mask=bits(mask), k_scale=ks, v_scale=vs, scale=0.0)
    check(q, kv, vv, [length], mask, 0.0, got, cache)


@pytest.mark.parametrize("hs", [64, 128, 256])
def test_scores_over_fp32_caches_are_sums_of_short_chains(hs):
    """two positions of about one score and values of +1 and -1 show a score difference as tanh(difference / 2).  A chain of n
    additions is off by about u sqrt(n^2 / 2) of a term's size, four of n / 4 by half of that: the rms error is held to 3/4 of a
    chain's"""
    g = gen(hs)
    b, h = 256, 4
    k = torch.randn(b, h, 2, hs, generator=g) * 4
    q = torch.randn(b, 1, h, hs, generator=g) * 4
    qd = q[:, 0].double()  # [b, h, hs]
    # the largest element of each query evens the scores out
    at = qd.abs().argmax(-1, keepdim=True)
    diff = ((k[:, :, 0] - k[:, :, 1]).double() * qd).sum(-1, keepdim=True) / qd.gather(-1, at)
    k[:, :, 1] = k[:, :, 1].scatter_add(-1, at, diff.float())
    v = torch.ones(b, h, 2, hs)
    v[:, :, 1] = -1
    want = ((k[:, :, 0].double() - k[:, :, 1].double()) * qd).sum(-1)
    assert float(want.abs().max()) < 1e-3
    lens = torch.ones(b, dtype=torch.int32, device=DEV)
    got = pkg().tree_attention(q.to(DEV), k.to(DEV), v.to(DEV), lens, scale=1.0)[:, 0, :, 0].double().cpu()
    own = 2 * torch.atanh(got) - want
    chain = torch.zeros(b, h, 2, dtype=torch.float64)
    for i in range(hs):
        chain = (chain + k[..., i].double() * qd[:, :, None, i]).float().double()
    one = chain[..., 0] - chain[..., 1] - want
    assert float(own.square().mean().sqrt()) < 0.75 * float(one.square().mean().sqrt())
