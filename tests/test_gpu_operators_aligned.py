"""Cache rows that start at any multiple of 4 bytes, which is all that the operators ask of them, and memory that lies on itself."""
import pytest

from helpers import pkg
from test_gpu_operators import CACHES, DEV, ROWS, attention_check, gen, quantized, same, tree_masks

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", list(CACHES))
@pytest.mark.parametrize("hs,off,pad", [(64, 1, 1), (64, 3, 2), (128, 1, 3), (48, 2, 1), (256, 1, 0)])
def test_rows_at_multiples_of_4_bytes(cache, rows, hs, off, pad):
    """off and pad: 4-byte words before the first row, and between a row and the next"""
    g, b, h, ctx, t, heads = gen(hs + off), 2, 2, 70, 5, 4
    dt = CACHES[cache]
    word = 4 // torch.empty(0, dtype=dt).element_size()
    step = hs + pad * word
    mem = [torch.zeros(off * word + b * h * ctx * step, dtype=torch.float32).to(dt).to(DEV) for _ in range(2)]
    k, v = (m[off * word:].as_strided((b, h, ctx, hs), (h * ctx * step, ctx * step, step, 1)) for m in mem)
    assert k.data_ptr() % 16 == 4 * off % 16
    ks, vs = (torch.zeros(b, h, ctx, device=DEV) for _ in range(2)) if cache in ("int8", "e4m3") else (None, None)
    x = [torch.randn(b, ctx, h, hs, generator=g).to(ROWS[rows]) for _ in range(2)]
    zero = torch.zeros(b, dtype=torch.int32, device=DEV)
    pkg().kv_write(x[0].to(DEV), x[1].to(DEV), k, v, zero, k_scale=ks, v_scale=vs)
    back = pkg().kv_read(k, v, zero, ctx, k_scale=ks, v_scale=vs)
    vals = []
    for y, store, s, got in zip(x, (k, v), (ks, vs), back):
        val, code, scale = quantized(y.double(), cache)
        assert same(store.float(), code.transpose(1, 2)) and same(got, val.float())
        assert s is None or same(s, scale.transpose(1, 2))
        vals.append(val.transpose(1, 2))
    for m, n in zip(mem, (step, step)):  # what lies between the rows stays
        rest = m[off * word:].view(-1, n)[:, hs:]
        assert (m[:off * word].float() == 0).all() and (rest.float() == 0).all()
    q = torch.randn(b, t, heads, hs, generator=g).to(ROWS[rows])
    mask, lens = tree_masks(g, b, t), [64, 7]
    got = pkg().tree_attention(q.to(DEV), k, v, torch.tensor(lens, dtype=torch.int32, device=DEV),
                               mask=torch.from_numpy(mask.view("int64")).to(DEV), k_scale=ks, v_scale=vs)
    attention_check(q, vals[0], vals[1], lens, [t] * b, mask, hs ** -0.5, got, ctx, cache)


def test_shared_memory_is_read_and_not_written(capfd):
    """sequences that share one cache (a stride of zero), and K and V in one tensor: attention and reads take them, writes do not"""
    g, b, h, ctx, hs = gen(3), 3, 2, 40, 64
    one = torch.randn(1, h, ctx, hs, generator=g).to(DEV)
    shared, apart = one.expand(b, h, ctx, hs), one.expand(b, h, ctx, hs).contiguous()
    lens = torch.tensor([30, 7, 0], dtype=torch.int32, device=DEV)
    q = torch.randn(b, 2, 4, hs, generator=g).to(DEV)
    assert torch.equal(pkg().tree_attention(q, shared, shared, lens), pkg().tree_attention(q, apart, apart.clone(), lens))
    for x, y in zip(pkg().kv_read(shared, shared, lens, 5), pkg().kv_read(apart, apart, lens, 5)):
        assert torch.equal(x, y)
    rows = torch.randn(b, 2, h, hs, generator=g).to(DEV)
    for k, v, says in ((shared, one.clone().expand(b, h, ctx, hs), "a stride of zero"), (apart, apart, "the same memory")):
        old = k.clone()
        with pytest.raises(RuntimeError):
            pkg().kv_write(rows, rows, k, v, lens)
        assert says in capfd.readouterr().err
        assert torch.equal(k, old)
    for out in (torch.zeros(1, 2, 4, hs, device=DEV).expand(b, 2, 4, hs), torch.zeros(b, 1, 4, hs, device=DEV).expand(b, 2, 4, hs)):
        with pytest.raises(RuntimeError):
            pkg().tree_attention(q, apart, apart, lens, out=out)
        assert "a stride of zero" in capfd.readouterr().err


def test_rows_read_into_one_tensor():
    """`out` as a tensor of two, K's rows and V's"""
    g = gen(4)
    k, v = (torch.randn(2, 2, 20, 64, generator=g).to(DEV) for _ in range(2))
    pos = torch.tensor([3, 11], dtype=torch.int32, device=DEV)
    out = torch.zeros(2, 2, 6, 2, 64, device=DEV)
    got = pkg().kv_read(k, v, pos, 6, out=out)
    for x, y, z in zip(got, pkg().kv_read(k, v, pos, 6), out):
        assert torch.equal(x, y) and torch.equal(z, y)
