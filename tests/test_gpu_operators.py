"""The operators on device memory (llm_kv_write, llm_kv_read, llm_tree_attention, llm_logprobs) against their definitions
in float64.

Tolerances.  u = 2^-24, half a step of fp32.
  cache rows: none; scales and codes are those of the definition.
  attention: a score is a sum of hs products, the query held to 22 bits at least (4 u): off by at most (hs + 8) u scale
    sum |q k|.  A
    weight is then off by a factor of e^(2 d), d the largest such error of the row, a sum over L positions by L u, and
    everything else (exponential, scales, joins) by 64 u; so is the output, relative to sum p |v|.  bf16: the weights'
    half step in fp16 (8-bit caches, 2^-11) or in two bf16 pieces (2^-16), and the output's, 2^-8 of its value.
    8-bit caches: the weights p sv are fp16 pieces, scaled so that the largest V scale lands in [2^14, 2^15).  The last
    piece has steps of 2^-24, so it is off by at most 2^-25 and a term code * w by |code| 2^-25 / (2^14 / max sv) <=
    2^-39 max |v|: L of those.  (It is all there is in a dimension where the tokens that count have the code 0.)
  log probabilities: exponents off by 4 u |x - max| / T, the sum's terms by their number in a thread's chain and 64 joins
    and roundings, the result by its own rounding."""
import math

import numpy as np
import pytest

from helpers import pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEV = "cuda"
CACHES = {"fp32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ROWS = {"fp32": torch.float32, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def quantized(x, cache):
    """(values, codes as float64, scales) of rows x (float64, on the CPU) by the definition"""
    if cache in ("fp32", "bf16"):
        v = x.float() if cache == "fp32" else x.float().to(torch.bfloat16)
        return v.double(), v.double(), None
    top = 127.0 if cache == "int8" else 448.0
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad.unsqueeze(-1), torch.zeros_like(x), x)
    s = (x.abs().amax(-1) / top).float()
    sd = torch.where(s > 0, s, torch.ones_like(s)).double().unsqueeze(-1)
    q = torch.where(s.unsqueeze(-1) > 0, x / sd, torch.zeros_like(x)).clamp(-top, top)
    if cache == "int8":
        q = torch.round(q)
    else:
        mid = (E4M3[1:] + E4M3[:-1]) / 2
        i = torch.bucketize(q.abs().contiguous(), mid)
        tie = (q.abs() == mid[i.clamp(max=125)]) & (i < 126) & (i % 2 == 1)
        q = torch.sign(q) * E4M3[i + tie.long()]
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    return q * s.double().unsqueeze(-1), q, s


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def cache_tensors(cache, b, h, ctx, hs, layout, fill):
    """empty K and V (and scales) in one of three layouts: heads apart, positions of all heads together, a slice of more"""
    def make(inner, dtype):
        if layout == "heads":
            return torch.full((b, h, ctx) + inner, fill, dtype=torch.float32).to(dtype).to(DEV)
        if layout == "positions":
            return torch.full((b, ctx, h) + inner, fill, dtype=torch.float32).to(dtype).to(DEV).transpose(1, 2)
        wide = torch.full((b, h, ctx + 3) + tuple(2 * d for d in inner), fill, dtype=torch.float32).to(dtype).to(DEV)
        return wide[:, :, 2:2 + ctx, :hs] if inner else wide[:, :, 2:2 + ctx]
    k, v = make((hs,), CACHES[cache]), make((hs,), CACHES[cache])
    if cache in ("fp32", "bf16"):
        return k, v, None, None
    return k, v, make((), torch.float32), make((), torch.float32)


# ---- the cache ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", list(CACHES))
@pytest.mark.parametrize("hs,h,layout", [(16, 1, "heads"), (48, 6, "positions"), (64, 2, "heads"), (80, 3, "slice"),
                                         (128, 4, "positions"), (256, 1, "heads")])
def test_rows_written_and_read(cache, rows, hs, h, layout):
    b, t, ctx = 3, 7, 19
    g = gen(hs + h)
    x = [torch.randn(b, t, h, hs, generator=g) * torch.exp(3 * torch.randn(b, t, h, 1, generator=g)) for _ in range(2)]
    x = [y.to(ROWS[rows]) for y in x]
    pos, n = torch.tensor([0, 15, -3], dtype=torch.int32), torch.tensor([7, 6, 5], dtype=torch.int32)
    k, v, ks, vs = cache_tensors(cache, b, h, ctx, hs, layout, 1.0)
    pkg().kv_write(x[0].to(DEV), x[1].to(DEV), k, v, pos.to(DEV), n.to(DEV), k_scale=ks, v_scale=vs)
    back = pkg().kv_read(k, v, pos.to(DEV), t, n.to(DEV), k_scale=ks, v_scale=vs)
    half = pkg().kv_read(k, v, pos.to(DEV), t, n.to(DEV), k_scale=ks, v_scale=vs, dtype=torch.bfloat16)
    for store, sc, y, got, got16 in ((k, ks, x[0], back[0], half[0]), (v, vs, x[1], back[1], half[1])):
        val, code, s = quantized(y.double(), cache)
        want_codes = torch.ones(b, h, ctx, hs, dtype=torch.float64)
        want_s, want = torch.ones(b, h, ctx), torch.zeros(b, t, h, hs, dtype=torch.float64)
        for i in range(b):
            for j in range(int(n[i])):
                p = int(pos[i]) + j
                if 0 <= p < ctx:
                    want_codes[i, :, p] = code[i, j]
                    want[i, j] = val[i, j].float().double()
                    if s is not None:
                        want_s[i, :, p] = s[i, j]
        assert same(store.float(), want_codes)
        if s is not None:
            assert same(sc, want_s)
        assert same(got, want)
        assert same(got16, want.float().to(torch.bfloat16))


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_rows_at_the_borders(cache):
    """rows of zeros, of the smallest and the largest values, exact halves between codes, infinities and NaN"""
    hs, top = 64, 127.0 if cache == "int8" else 448.0
    rows = [torch.zeros(hs), torch.full((hs,), 2.0 ** -149), torch.full((hs,), -(2.0 ** -140)),
            torch.linspace(-3e38, 3e38, hs), torch.full((hs,), torch.finfo(torch.float32).max)]
    half = torch.arange(hs).float() + 0.5  # scale 1: halves
    half[0] = top
    rows += [half, -half, half * 2.0 ** -100, half * 3.0 * 2.0 ** -130, half * 2.0 ** 100]
    g = gen(3)
    for _ in range(40):  # quotients next to a border: code + 1/2 times a scale that is no power of two, rounded
        s = float(torch.rand(1, generator=g)) + 0.5
        r = (torch.randint(-126, 126, (hs,), generator=g).double() + 0.5) * (s if cache == "int8" else s * 2)
        r[7] = top * s
        rows.append(r.float())
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.randn(hs, generator=g)
        r[11] = bad
        rows.append(r)
    x = torch.stack(rows).view(1, -1, 1, hs)
    t = x.shape[1]
    k, v, ks, vs = cache_tensors(cache, 1, 1, t, hs, "heads", 0.0)
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    pkg().kv_write(x.to(DEV), (-x).to(DEV), k, v, pos, k_scale=ks, v_scale=vs)
    back = pkg().kv_read(k, v, pos, t, k_scale=ks, v_scale=vs)
    for store, sc, y, got in ((k, ks, x, back[0]), (v, vs, -x, back[1])):
        val, code, s = quantized(y.double(), cache)
        assert same(sc[0, 0], s[0, :, 0])
        assert same(store[0, 0].float(), code[0, :, 0])
        assert same(got, val.float())


# ---- attention ---------------------------------------------------------------------------------------------------


def tree_masks(g, b, t):
    mask = np.zeros((b, t), np.uint64)
    for i in range(b):
        for j in range(t):
            p = int(torch.randint(0, j, (1,), generator=g)) if j else -1
            mask[i, j] = (mask[i, p] if p >= 0 else np.uint64(0)) | np.uint64(1 << j)
    return mask


def attention_check(q, kval, vval, lens, n, mask, scale, got, cache_len, cache):
    """got against float64 over the values kval, vval [b][h][ctx][hs] (float64, CPU)"""
    b, t, heads, hs = q.shape
    h = kval.shape[1]
    qd = q.double().cpu()
    for i in range(b):
        for j in range(t):
            if j >= n[i]:
                assert (got[i, j] == 0).all()
                continue
            seen = [p for p in range(min(int(lens[i]), cache_len))]
            seen += [int(lens[i]) + m for m in range(int(n[i])) if (int(mask[i][j]) >> m) & 1 and lens[i] + m < cache_len]
            if not seen:
                assert (got[i, j] == 0).all()
                continue
            idx = torch.tensor(seen)
            for hd in range(heads):
                kk, vv = kval[i, hd // (heads // h)][idx], vval[i, hd // (heads // h)][idx]
                s = (kk @ qd[i, j, hd]) * scale
                p = torch.softmax(s, 0)
                want = p @ vv
                d = (hs + 8) * U * scale * float((kk.abs() @ qd[i, j, hd].abs()).max())
                rel = 2 * d + (len(seen) + 64) * U
                tol = rel * (p @ vv.abs())
                if q.dtype == torch.bfloat16:
                    tol = tol + (2.0 ** -11 if cache in ("int8", "e4m3") else 2.0 ** -16) * (p @ vv.abs()) + 2.0 ** -8 * want.abs()
                if cache in ("int8", "e4m3"):
                    tol = tol + len(seen) * 2.0 ** -39 * float(vval[i, hd // (heads // h)].abs().max())
                err = (got[i, j, hd].double().cpu() - want).abs()
                assert (err <= tol + 1e-37).all(), (i, j, hd, float((err / (tol + 1e-37)).max()))


def attention_case(cache, rows, b, heads, h, hs, ctx, lens, t, n=None, layout="heads", seed=0, mask=None, poison=True,
                   max_len=None):
    g = gen(1000 * hs + 10 * t + seed)
    vals, tensors = [], []
    k, v, ks, vs = cache_tensors(cache, b, h, ctx, hs, layout, 0.0)
    for store, sc in ((k, ks), (v, vs)):
        x = torch.randn(b, h, ctx, hs, generator=g) * torch.exp(torch.randn(b, h, ctx, 1, generator=g))
        val, code, s = quantized(x.double(), cache)
        store.copy_(code.float().to(CACHES[cache]).to(DEV))
        if s is not None:
            sc.copy_(s.to(DEV))
        vals.append(val)
    q = torch.randn(b, t, heads, hs, generator=g).to(ROWS[rows])
    nn = [t] * b if n is None else n
    if mask is None:
        mask = tree_masks(g, b, t)
    if poison:  # what no token sees holds infinities and NaN
        for i in range(b):
            seen = 0
            for j in range(nn[i]):
                seen |= int(mask[i][j])
            for p in range(lens[i], ctx):
                if p - lens[i] >= nn[i] or not (seen >> (p - lens[i])) & 1:
                    for store, sc in ((k, ks), (v, vs)):
                        if sc is None:
                            store[i, :, p] = math.nan if p % 2 else math.inf
                        else:
                            sc[i, :, p] = math.nan if p % 2 else math.inf
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    m = torch.from_numpy(np.array(mask, np.uint64).view(np.int64)).to(DEV)
    got = pkg().tree_attention(q.to(DEV), k, v, it(lens), None if n is None else it(n), m, k_scale=ks, v_scale=vs,
                               max_len=max_len)
    attention_check(q, vals[0], vals[1], lens, nn, mask, hs ** -0.5, got, ctx, cache)
    return got


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", list(CACHES))
@pytest.mark.parametrize("heads,h,hs,layout", [(2, 2, 16, "heads"), (6, 6, 48, "positions"), (14, 2, 64, "heads"),
                                               (28, 4, 128, "slice"), (5, 1, 80, "positions"), (3, 1, 160, "heads"),
                                               (8, 4, 256, "positions")])
def test_attention_of_trees(cache, rows, heads, h, hs, layout):
    attention_case(cache, rows, 3, heads, h, hs, 150, [0, 37, 131], 5, [5, 3, 4], layout)


@pytest.mark.parametrize("cache,hs", [("int8", 64), ("int8", 128), ("fp32", 64), ("bf16", 128), ("e4m3", 256)])
@pytest.mark.parametrize("length", [0, 1, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 255, 256, 257, 1000])
def test_attention_of_one_token(cache, hs, length):
    attention_case(cache, "fp32", 1, 4, 2, hs, length + 3, [length], 1)


@pytest.mark.parametrize("t", [2, 16, 17, 33, 63, 64])
@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("bf16", "bf16"), ("fp32", "fp32"), ("e4m3", "bf16")])
def test_attention_of_long_trees(cache, rows, t):
    attention_case(cache, rows, 2, 3, 1, 64, 700, [600, 63], t)


@pytest.mark.parametrize("cache", list(CACHES))
def test_attention_masks_that_leave_nothing(cache):
    """no bit at all, not even the token itself; over an empty and over a filled cache"""
    mask = np.array([[0, 1, 0, 2], [0, 1, 0, 5]], np.uint64)
    got = attention_case(cache, "fp32", 2, 4, 2, 64, 80, [0, 70], 4, mask=mask)
    assert (got[0, 0] == 0).all() and (got[0, 2] == 0).all() and (got[1] != 0).all()


def test_attention_past_the_cache():
    """new tokens whose rows lie past the last position are not seen; lengths beyond it and below zero are cut"""
    attention_case("int8", "fp32", 1, 4, 2, 64, 70, [68], 4, mask=np.array([[1, 3, 7, 15]], np.uint64))
    q = torch.randn(2, 1, 4, 64, device=DEV)
    k, v = (torch.randn(2, 2, 70, 64, device=DEV) for _ in range(2))
    pk = pkg()
    far = pk.tree_attention(q, k, v, torch.tensor([1 << 30, -5], dtype=torch.int32, device=DEV))
    cut = pk.tree_attention(q, k, v, torch.tensor([70, 0], dtype=torch.int32, device=DEV))
    assert same(far, cut)


@pytest.mark.parametrize("cache,heads,h,hs", [("int8", 28, 4, 128), ("fp32", 14, 2, 64), ("bf16", 28, 4, 128)])
def test_attention_over_many_slices(cache, heads, h, hs):
    """contexts of several thousand positions, cut into slices that are joined; a bound of the lengths that is too low"""
    a = attention_case(cache, "fp32", 1, heads, h, hs, 5003, [4990], 3)
    attention_case(cache, "fp32", 2, heads, h, hs, 2500, [2400, 77], 2)
    b = attention_case(cache, "fp32", 1, heads, h, hs, 5003, [4990], 3, max_len=10)
    assert float((a - b).abs().max()) < 1e-4


def roomy_case(cache, rows, b, heads, h, hs, ctx, lens, t, n=None, max_len=None, seed=0):
    """a cache of ctx positions whose bound the lengths stay far below (max_len None: the cache's): rows as of a long
    context, checked over the positions that hold something; all others hold infinities and NaN"""
    g = gen(hs + t + seed)
    top = max(lens) + t
    k, v, ks, vs = cache_tensors(cache, b, h, ctx, hs, "heads", math.nan)
    vals = []
    for store, sc in ((k, ks), (v, vs)):
        x = torch.randn(b, h, top, hs, generator=g) * torch.exp(torch.randn(b, h, top, 1, generator=g))
        val, code, s = quantized(x.double(), cache)
        nn = [t] * b if n is None else n
        for i in range(b):
            end = lens[i] + nn[i]
            store[i, :, :end] = code[i, :, :end].float().to(CACHES[cache]).to(DEV)
            if s is not None:
                sc[i, :, :end] = s[i, :, :end].to(DEV)
        vals.append(val)
    q = torch.randn(b, t, heads, hs, generator=g).to(ROWS[rows])
    mask = tree_masks(g, b, t)
    it = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = pkg().tree_attention(q.to(DEV), k, v, it(lens), None if n is None else it(n),
                               torch.from_numpy(mask.view(np.int64)).to(DEV), k_scale=ks, v_scale=vs, max_len=max_len)
    attention_check(q, vals[0], vals[1], lens, nn, mask, hs ** -0.5, got, ctx, cache)


@pytest.mark.parametrize("cache,rows,b,heads,h,hs,ctx,t", [
    ("bf16", "bf16", 1, 28, 4, 128, 30000, 37), ("bf16", "fp32", 1, 28, 4, 128, 12000, 37),
    ("bf16", "bf16", 2, 12, 1, 96, 21000, 64), ("bf16", "fp32", 3, 20, 2, 112, 7000, 19),
    ("bf16", "fp32", 1, 28, 4, 128, 23000, 20), ("bf16", "bf16", 1, 28, 4, 128, 60000, 20),
    ("bf16", "bf16", 1, 28, 4, 128, 16000, 8), ("bf16", "bf16", 1, 14, 2, 64, 32000, 7),
    ("int8", "fp32", 1, 28, 4, 128, 12000, 37), ("int8", "bf16", 2, 28, 4, 128, 9000, 15),
    ("e4m3", "fp32", 3, 28, 4, 112, 4500, 37), ("e4m3", "bf16", 1, 28, 4, 128, 12000, 64),
    ("int8", "fp32", 3, 14, 2, 64, 16000, 37), ("fp32", "fp32", 1, 28, 4, 128, 9000, 37)])
@pytest.mark.parametrize("length", [0, 95, 1500])
def test_attention_of_many_rows(cache, rows, b, heads, h, hs, ctx, t, length):
    """the cuts of calls with many rows and a large bound, over empty, short and sliced contexts"""
    roomy_case(cache, rows, b, heads, h, hs, ctx, [length, 64, 7][:b], t, None if b == 1 else [t, t - 3, 1][:b])


@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("e4m3", "bf16"), ("bf16", "bf16"), ("fp32", "fp32")])
@pytest.mark.parametrize("b,h,longest", [(2, 1, 40000), (3, 2, 9000), (63, 1, 2500), (64, 3, 1700), (65, 1, 2500),
                                         (130, 1, 900), (300, 1, 700), (511, 1, 300), (512, 1, 300), (513, 1, 300)])
def test_attention_of_uneven_batches(cache, rows, b, h, longest):
    """one long sequence, one of every other length down to none: slices of equal steps over all of them"""
    lens = [longest if i == b // 2 else (i * 37) % 301 for i in range(b)]
    roomy_case(cache, rows, b, 2 * h, h, 16, longest + 70, lens, 2, [1 + i % 2 for i in range(b)])


@pytest.mark.parametrize("cache,rows", [("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16"), ("int8", "fp32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("slope", [-0.05, 0.002, 0.05, 0.4])
@pytest.mark.parametrize("t,heads,ctx", [(1, 2, 800), (40, 28, 30000)])
def test_attention_of_scores_that_rise(cache, rows, slope, t, heads, ctx):
    """every position's score above (below) the one before: a new maximum at every step, by little or by much"""
    g = gen(9)
    h, hs, length = 1, 128, 700
    top = length + t
    p = torch.arange(top).double() * slope
    x = [torch.randn(1, h, top, hs, generator=g).double() * 0.1 for _ in range(2)]
    u = torch.randn(hs, generator=g).double()
    x[0] += p.view(1, 1, top, 1) * u * hs ** 0.5 / (u @ u)  # score slope * position, and noise
    q = (u + 0.02 * torch.randn(1, t, heads, hs, generator=g).double()).float().to(ROWS[rows])
    k, v, ks, vs = cache_tensors(cache, 1, h, ctx, hs, "heads", math.nan)
    vals = []
    for y, store, sc in ((x[0], k, ks), (x[1], v, vs)):
        val, code, s = quantized(y, cache)
        store[:, :, :top] = code.float().to(CACHES[cache]).to(DEV)
        if s is not None:
            sc[:, :, :top] = s.to(DEV)
        vals.append(val)
    mask = tree_masks(g, 1, t)
    got = pkg().tree_attention(q.to(DEV), k, v, torch.tensor([length], dtype=torch.int32, device=DEV), None,
                               torch.from_numpy(mask.view(np.int64)).to(DEV), k_scale=ks, v_scale=vs)
    attention_check(q, vals[0], vals[1], [length], [t], mask, hs ** -0.5, got, ctx, cache)


@pytest.mark.parametrize("cache,rows", [("int8", "fp32"), ("fp32", "bf16")])
def test_attention_of_the_most_rows(cache, rows):
    roomy_case(cache, rows, 2, 64, 1, 16, 700, [130, 3], 64, [64, 2])


@pytest.mark.parametrize("seq,head,pos", [(1 << 32, 64 * 300, 64), (64 * 400, 1 << 32, 64), (64, 128, 1 << 24)])
def test_offsets_past_32_bits(seq, head, pos):
    """sequences, heads or positions more than 4 GiB apart: the same as a small cache"""
    P, g = pkg(), gen(8)
    b, h, ctx, hs, t = (2, 2, 300, 64, 3) if pos == 64 else (1, 2, 300, 64, 3)
    big = torch.zeros(((b - 1) * seq + (h - 1) * head + ctx * pos) + (1 << 20), dtype=torch.int8, device=DEV)
    far = [big[o:].as_strided((b, h, ctx, hs), (seq, head, pos, 1)) for o in (0, 1 << 19)]
    near = [torch.zeros(b, h, ctx, hs, dtype=torch.int8, device=DEV) for _ in range(2)]
    rows = [torch.randn(b, 290, h, hs, generator=g).to(DEV) for _ in range(2)]
    q = torch.randn(b, t, 4 * h, hs, generator=g).to(DEV)
    at = torch.tensor([5, 10][:b], dtype=torch.int32, device=DEV)
    lens = torch.tensor([292, 100][:b], dtype=torch.int32, device=DEV)
    got = []
    for k, v in (far, near):
        ks, vs = (torch.zeros(b, h, ctx, device=DEV) for _ in range(2))
        P.kv_write(rows[0], rows[1], k, v, at, k_scale=ks, v_scale=vs)
        got.append((k.clone(), v.clone(), ks, vs) + P.kv_read(k, v, at, 280, k_scale=ks, v_scale=vs) +
                   (P.tree_attention(q, k, v, lens, k_scale=ks, v_scale=vs),))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert bool((got[0][0] != 0).any()) and bool((got[0][6] != 0).any())


def test_attention_of_a_batch_above_its_bound():
    """a bound of the lengths that is too low costs time, not results"""
    for b, longest in ((3, 9000), (70, 3000)):
        lens = [longest if i == 1 else 11 * (i % 9) for i in range(b)]
        for max_len in (0, 13, 900):
            roomy_case("int8", "fp32", b, 2, 1, 32, longest + 5, lens, 2, max_len=max_len)


def test_attention_chain_is_the_default_mask():
    g = gen(5)
    b, t, heads, h, hs, ctx = 2, 9, 4, 2, 64, 100
    q, k, v = (torch.randn(s, generator=g).to(DEV) for s in ((b, t, heads, hs), (b, h, ctx, hs), (b, h, ctx, hs)))
    lens = torch.tensor([50, 0], dtype=torch.int32, device=DEV)
    chain = torch.tensor([[(2 << j) - 1 for j in range(t)]] * b, dtype=torch.int64, device=DEV)
    assert torch.equal(pkg().tree_attention(q, k, v, lens), pkg().tree_attention(q, k, v, lens, mask=chain))


@pytest.mark.parametrize("cache", ["fp32", "bf16"])
def test_attention_new_rows_that_are_not_finite_reach_their_descendants_only(cache):
    g = gen(6)
    b, t, heads, h, hs, ctx = 1, 6, 4, 2, 64, 90
    q, k, v = (torch.randn(s, generator=g) for s in ((b, t, heads, hs), (b, h, ctx, hs), (b, h, ctx, hs)))
    mask = [1, 3, 5, 11, 21, 33]  # node 1's descendants: 1, 3
    lens = torch.tensor([60], dtype=torch.int32, device=DEV)
    m = torch.tensor([mask], dtype=torch.int64, device=DEV)
    dt = CACHES[cache]
    clean = pkg().tree_attention(q.to(DEV), k.to(dt).to(DEV), v.to(dt).to(DEV), lens, mask=m)
    v[0, :, 61, 5] = math.inf
    dirty = pkg().tree_attention(q.to(DEV), k.to(dt).to(DEV), v.to(dt).to(DEV), lens, mask=m)
    for i in range(t):
        if (mask[i] >> 1) & 1:
            assert dirty[0, i].isnan().all()
        else:
            assert torch.equal(dirty[0, i], clean[0, i])


def test_attention_of_strided_queries_and_outputs():
    g = gen(7)
    b, t, heads, h, hs, ctx = 2, 3, 4, 2, 64, 60
    wide = torch.randn(t, b, heads + 2 * h, hs + 16, generator=g).to(DEV)
    q = wide.transpose(0, 1)[:, :, :heads, 8:8 + hs]
    k, v = (torch.randn(b, h, ctx, hs, generator=g).to(DEV) for _ in range(2))
    lens = torch.tensor([50, 20], dtype=torch.int32, device=DEV)
    out = torch.full((t, heads, b, hs), 7.0, device=DEV)
    view = out.permute(2, 0, 1, 3)
    n = torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    pkg().tree_attention(q, k, v, lens, n, out=view)
    want = pkg().tree_attention(q.contiguous(), k, v, lens, n)
    assert torch.equal(view[0], want[0]) and torch.equal(view[1, 0], want[1, 0])
    assert (view[1, 1:] == 7.0).all()  # rows behind the last token stay


# ---- log probabilities -------------------------------------------------------------------------------------------


def order(x):
    """indices in descending order: NaN first, the lowest index first among equals"""
    x = np.array(x, np.float64)
    return sorted(range(x.size), key=lambda i: (0 if np.isnan(x[i]) else 1, 0.0 if np.isnan(x[i]) else -x[i], i))


def logprobs_check(x, tokens, top, T, got):
    logp, entropy, ids, top_logp, lse = (y.cpu() for y in got)
    rows, vocab = x.shape
    y = x.double().cpu() / T
    for r in range(rows):
        m, z = float(y[r].max()), torch.logsumexp(y[r], 0)
        lp = y[r] - z
        p = torch.exp(lp)
        far = U * (4 * (m - y[r][torch.isfinite(y[r])]).abs() * p[torch.isfinite(y[r])]).sum() + (vocab / 256 + 64) * U
        tol = lambda v: float(far) + 4 * U * (abs(m) + abs(float(v)) + abs(float(v) + float(z) - m))  # noqa: E731
        assert abs(float(lse[r]) - float(z)) <= tol(0)
        h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum()
        spread = (p * torch.where(p > 0, (m - y[r]).abs(), torch.zeros_like(p))).sum()
        assert abs(float(entropy[r] - h)) <= 4 * (float(far) + (vocab / 256 + 64) * U * (1 + float(spread)))
        want = order(x[r].double().cpu().numpy())[:top]
        assert list(ids[r]) == want
        for a, i in zip(top_logp[r], want):
            assert float(a) == float(lp[i]) or abs(float(a) - float(lp[i])) <= tol(lp[i])
        for a, tk in zip(logp[r], tokens[r].tolist() if tokens is not None else []):
            if 0 <= tk < vocab:
                assert float(a) == float(lp[tk]) or abs(float(a) - float(lp[tk])) <= tol(lp[tk])
            else:
                assert float(a) == -math.inf


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,top,T", [(1, 1, 1, 1.0), (3, 2, 2, 0.5), (2, 5, 5, 1.0), (5, 63, 7, 1.0),
                                              (4, 64, 32, 2.0), (2, 257, 20, 1.0), (3, 4095, 20, 1.0), (3, 4097, 1, 0.7),
                                              (7, 8191, 32, 1.0), (2, 32000, 20, 1.3), (1, 65536, 20, 1.0),
                                              (2, 151937, 5, 1.0), (600, 1000, 3, 1.0)])
def test_logprobs(dtype, rows, vocab, top, T):
    g = gen(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 4).to(ROWS[dtype])
    tokens = torch.randint(-1, vocab + 1, (rows, 3), generator=g, dtype=torch.int32)
    logprobs_check(x, tokens, top, T, pkg().logprobs(x.to(DEV), tokens.to(DEV), top, T))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_logprobs_ties_masks_and_orders(dtype):
    """equal values (the lowest index first), masked ones, rising and falling rows, zeros of both signs"""
    vocab = 9001
    a = torch.zeros(8, vocab)
    a[1, ::2] = -0.0
    a[2] = torch.arange(vocab) / 64.0
    a[3] = -torch.arange(vocab) / 64.0
    a[4] = (torch.arange(vocab) % 7).float()
    a[5] = -math.inf
    a[5, [3, 4500, 9000]] = torch.tensor([1.0, 2.0, 1.0])
    a[6] = torch.finfo(torch.float32).min if dtype == "fp32" else -3e38
    a[6, 77] = 0.0
    a[7] = torch.randn(vocab, generator=gen(1)).round()
    x = a.to(ROWS[dtype])
    tokens = torch.tensor([[0, 4500, 9000]] * 8, dtype=torch.int32)
    for top in (1, 5, 32):
        logprobs_check(x, tokens, top, 1.0, pkg().logprobs(x.to(DEV), tokens.to(DEV), top))


def test_logprobs_of_rows_that_are_not_finite():
    vocab = 5000
    x = torch.randn(4, vocab, generator=gen(2))
    x[0, 4097], x[1, 17], x[2] = math.nan, math.inf, -math.inf
    tokens = torch.tensor([[1], [1], [1], [-7]], dtype=torch.int32)
    logp, entropy, ids, top_logp, lse = pkg().logprobs(x.to(DEV), tokens.to(DEV), 4)
    assert logp[:3].isnan().all() and float(logp[3]) == -math.inf
    assert entropy[:3].isnan().all() and lse[:2].isnan().all() and float(lse[2]) == -math.inf
    assert top_logp[:3].isnan().all() and not top_logp[3].isnan().any()
    for r in range(4):
        assert ids[r].tolist() == order(x[r].numpy())[:4]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lead", [0, 1, 2, 3, 5, 7])
def test_logprobs_of_strided_rows(dtype, lead):
    """rows that start anywhere within 16 bytes, infinities right before and behind them"""
    wide = torch.full((3, 4103 + 11), math.inf).to(ROWS[dtype])
    x = (torch.randn(3, 4103, generator=gen(lead)) * 3).to(ROWS[dtype])
    wide[:, lead:lead + 4103] = x
    logprobs_check(x, None, 6, 1.0, pkg().logprobs(wide.to(DEV)[:, lead:lead + 4103], None, 6))


# ---- as they are used --------------------------------------------------------------------------------------------


def step(P, st):
    """a drafted tree: its rows into the cache, its attention, its log probabilities"""
    P.kv_write(st["kr"], st["vr"], st["k"], st["v"], st["lens"], st["n"], k_scale=st["ks"], v_scale=st["vs"])
    o = P.tree_attention(st["q"], st["k"], st["v"], st["lens"], st["n"], st["mask"], k_scale=st["ks"], v_scale=st["vs"])
    return (o,) + P.logprobs(st["logits"], st["tokens"], 5)


def step_state(seed):
    g = gen(seed)
    b, t, heads, h, hs, ctx = 2, 6, 14, 2, 64, 900
    st = dict(kr=torch.randn(b, t, h, hs, generator=g), vr=torch.randn(b, t, h, hs, generator=g),
              q=torch.randn(b, t, heads, hs, generator=g), lens=torch.tensor([840, 13], dtype=torch.int32),
              n=torch.tensor([6, 4], dtype=torch.int32), logits=torch.randn(12, 20011, generator=g),
              tokens=torch.randint(0, 20011, (12, 2), generator=g, dtype=torch.int32),
              mask=torch.from_numpy(tree_masks(g, b, t).view(np.int64)))
    st = {k: v.to(DEV) for k, v in st.items()}
    st["k"], st["v"], st["ks"], st["vs"] = cache_tensors("int8", b, h, ctx, hs, "heads", 0.0)
    x = [torch.randn(b, 840, h, hs, generator=g).to(DEV) for _ in range(2)]
    pkg().kv_write(x[0], x[1], st["k"], st["v"], torch.zeros(2, dtype=torch.int32, device=DEV), k_scale=st["ks"], v_scale=st["vs"])
    return st


def test_a_drafted_step_on_another_stream():
    a, b = step_state(1), step_state(1)
    want = step(pkg(), a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(pkg(), b)
    s.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_two_drafted_steps_captured_and_replayed():
    """two graphs of their own states, replayed in turn with eager work between, inputs changed in place"""
    P = pkg()
    states, graphs, outs = [step_state(2), step_state(3)], [], []
    for st in states:
        step(P, st)
    torch.cuda.synchronize()
    for st in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(P, st))
        graphs.append(gr)
    for turn in range(4):
        for st in states:
            st["q"].mul_(1.1)
            st["kr"].add_(0.25)
            st["lens"].add_(1)
            st["logits"].mul_(0.9)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for st, got in zip(states, outs):
            for x, y in zip(got, step(P, st)):
                assert torch.equal(x, y), turn


def test_results_are_the_same_every_time():
    st = step_state(4)
    want = step(pkg(), st)
    for _ in range(5):
        for x, y in zip(step(pkg(), st), want):
            assert torch.equal(x, y)
