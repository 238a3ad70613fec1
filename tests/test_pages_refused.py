"""What the operators over a cache in pages refuse (no GPU: nothing here reaches one)."""
import ctypes as C

import pytest

from helpers import pkg
from test_operators import BF16, E4M3, F32, I8, rows

AT = 0x10000


def pages(type=I8, n_layers=1, n_pages=8, n_kv=2, hs=64, page=64, **kw):
    n = page * hs
    d = dict(k=AT, v=2 * AT, k_scale=AT, v_scale=2 * AT, type=type, n_layers=n_layers, n_pages=n_pages, n_kv=n_kv, hs=hs, page=page,
             layer=n_pages * n_kv * n, id=n_kv * n, head=n, s_layer=n_pages * n_kv * page // 64, s_id=n_kv * page // 64,
             s_head=page // 64)
    d.update(kw)
    return pkg().LlmPages(**d)


def write(c, k=None, v=None, seqs=1, per=4, n=1, table=AT):
    k = k or rows()
    return pkg().lib().llm_page_write(C.byref(c), C.byref(k), C.byref(v or k), seqs, table, per, None, AT, None, None, n, None)


def read(c, k=None, v=None, seqs=1, per=4, n=1):
    k = k or rows()
    return pkg().lib().llm_page_read(C.byref(c), C.byref(k), C.byref(v or k), seqs, AT, per, AT, None, n, 0, None)


def attend(c, q=None, k=None, v=None, out=None, heads=4, seqs=1, per=4, n=1, scale=0.1, work=0):
    q = q or rows()
    ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
    return pkg().lib().llm_page_attention(C.byref(c), C.byref(q), ref(k), ref(v), C.byref(out or q), heads, seqs, AT, per, AT, None,
                                          None, n, 100, scale, 0, None, work, None)


def reserve(c, seqs=1, per=4, n=1, work=0):
    return pkg().lib().llm_page_reserve(C.byref(c), seqs, AT, per, AT, AT, AT, n, AT, AT, work, None)


def compact(c, seqs=1, per=4, work=0):
    return pkg().lib().llm_page_compact(C.byref(c), seqs, AT, per, AT, AT, AT, work, None)


def fork(n_pages=8, page=64, seqs=2, per=4, count=1, table=AT):
    return pkg().lib().llm_page_fork(n_pages, page, seqs, table, per, AT, AT, AT, AT, count, AT, 1 << 20, None)


def accept(type=F32, seqs=1, n=3, vocab=100, seq=300, row=100, t=1.0, probs=None, p_type=F32, p_seq=0, p_row=0, x=AT):
    return pkg().lib().llm_draft_accept(x, type, seqs, n, vocab, seq, row, t, probs, p_type, p_seq, p_row, AT, None, None, AT, AT, AT,
                                        AT, AT, AT, 1 << 20, None)


@pytest.mark.parametrize("kw,says", [
    (dict(type=F32), "type 0"), (dict(type=BF16), "type 1"), (dict(type=4), "type 4"), (dict(hs=8), "8 values"),
    (dict(hs=72), "72 values"), (dict(hs=272), "272 values"), (dict(page=32), "32 positions"), (dict(page=192), "192 positions"),
    (dict(page=512), "512 positions"), (dict(n_pages=0), "0 pages"), (dict(n_layers=0), "0 layers"), (dict(n_kv=0), "0 heads"),
    (dict(head=0), "lie on themselves"), (dict(id=64 * 64 - 16), "lie on themselves"), (dict(s_id=0), "lie on themselves"),
    (dict(n_layers=2, layer=0), "lie on themselves"), (dict(head=-8192), "lie on themselves"), (dict(id=64 * 64 * 2 + 8), "multiples of 16"),
    (dict(k=AT + 8), "multiples of 16"), (dict(v=AT + 4), "multiples of 16"), (dict(k_scale=AT + 2), "multiples of 16"),
    (dict(v=AT), "the same memory"), (dict(v_scale=AT), "the same memory"), (dict(), "not device memory"),
    (dict(type=E4M3), "not device memory"), (dict(k=0), "not device memory")])
def test_pools_refused(kw, says, capfd):
    for call in (write, read, attend, reserve, compact):
        assert call(pages(**kw)) == -1
        assert says in capfd.readouterr().err, call


def test_tables_refused(capfd):
    for call in (write, read, attend, reserve, compact):
        for kw in (dict(seqs=-1), dict(per=0), dict(per=(1 << 22) + 1)):
            assert call(pages(), **kw) == -1
            err = capfd.readouterr().err
            assert "a table of" in err or "pages for a sequence" in err
    assert write(pages(), table=AT + 2) == -1 and fork(table=AT + 1) == -1
    for kw in (dict(seqs=-1), dict(per=0)):
        assert fork(**kw) == -1
    assert capfd.readouterr().err.count("a table of") == 4


def test_arguments_refused(capfd):
    c = pages()
    for call in (lambda: write(c, n=-1), lambda: read(c, n=-1), lambda: attend(c, heads=3), lambda: attend(c, heads=0),
                 lambda: attend(c, heads=2 * 65), lambda: attend(c, n=65), lambda: attend(c, n=-1), lambda: attend(c, k=rows()),
                 lambda: attend(c, v=rows()), lambda: reserve(c, n=-1), lambda: fork(n_pages=0), lambda: fork(page=100),
                 lambda: fork(count=-1), lambda: fork(count=65536)):
        assert call() == -1
        assert "bad arguments" in capfd.readouterr().err
    for scale in (float("nan"), float("inf"), 3e38):
        assert attend(c, scale=scale) == -1
        assert "scale" in capfd.readouterr().err
    for call in (lambda: read(c, rows(tok=0), n=2), lambda: read(c, rows(head=0)), lambda: read(c, rows(seq=0), seqs=2),
                 lambda: attend(c, out=rows(tok=0), n=2), lambda: attend(c, out=rows(head=0)), lambda: attend(c, out=rows(seq=0), seqs=2)):
        assert call() == -1
        assert "a stride of zero" in capfd.readouterr().err
    for kw in (dict(type=I8), dict(seqs=-1), dict(seqs=65536), dict(n=65), dict(n=-1), dict(vocab=0), dict(vocab=(1 << 28) + 1),
               dict(t=-1.0), dict(t=1e-31), dict(t=float("nan")), dict(t=float("inf")), dict(seq=-1), dict(row=-1), dict(x=AT + 2),
               dict(probs=AT, p_type=I8), dict(probs=AT, p_seq=-1), dict(probs=AT, p_row=-1), dict(probs=AT + 1)):
        assert accept(**kw) == -1
        assert "bad arguments" in capfd.readouterr().err, kw
    assert accept() == -1 and fork() == -1
    assert capfd.readouterr().err.count("not device memory") == 2


def test_more_rows_than_there_are_positions_refused(capfd):
    """counts whose rounding up to blocks would pass an int"""
    for n in ((1 << 30) + 1, 0x7fffffff):
        assert write(pages(), n=n) == -1 and read(pages(), n=n) == -1
        assert capfd.readouterr().err.count("bad arguments") == 2
    assert write(pages(), n=1 << 30) == -1
    assert "not device memory" in capfd.readouterr().err


@pytest.mark.parametrize("layer,id,head,fine", [
    (64 * 4096, 2 * 4096, 4096, True),           # [layers][pages][heads]
    (4096, 2 * 3 * 4096, 3 * 4096, True),        # [pages][heads][layers]
    (16 * 4096, 4096, 8 * 4096, True),           # heads before pages
    (2 * 4096, 6 * 4096, 4096, True),            # layers between
    (4096, 2 * 4096, 4096, False),               # layers on heads
    (64 * 4096, 4096, 4096, False),              # pages on heads
    (7 * 2 * 4096, 2 * 4096, 4096, False),       # the last page on the next layer's first
    (64 * 4096, 4096, 7 * 4096, False),          # the last page of a head on the next head's first
    (1 << 62, 1 << 61, 1 << 60, False)])         # eight pages 2^61 apart reach past 2^62; their sum passes 64 bits
def test_pools_that_lie_on_themselves_refused(layer, id, head, fine, capfd):
    """three layers of eight pages of two heads"""
    c = pages(n_layers=3, layer=layer, id=id, head=head, s_layer=100, s_id=4, s_head=1)
    assert write(c) == -1
    assert ("not device memory" if fine else "lie on themselves") in capfd.readouterr().err


def test_nothing_to_do():
    assert fork(count=0) == 0 and fork(seqs=0) == 0 and accept(seqs=0) == 0 and accept(n=0) == 0


def test_work_sizes():
    L = pkg().lib()
    c = pages()
    assert L.llm_page_fork_work(10, 3) >= 4 * 30 and L.llm_page_fork_work(0, 3) == 0
    assert L.llm_page_reserve_work(C.byref(c), 3, 10, 100) >= 4 * 8
    assert L.llm_page_reserve_work(C.byref(c), 0, 10, 100) == 0
    assert L.llm_page_compact_work(C.byref(c)) >= 4 * 8
    assert L.llm_draft_accept_work(1, 65, 100) == 0 and L.llm_draft_accept_work(2, 3, 10000) > 0
    assert L.llm_page_attention_work(C.byref(c), 1, 3, 1, 100) == 0


def test_tensors_refused():
    torch = pytest.importorskip("torch")
    P = pkg()
    i = torch.zeros(2, dtype=torch.int32)
    table, refs = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    r = torch.zeros(2, 1, 2, 64)
    k, v = torch.zeros(4, 2, 64, 64, dtype=torch.int8), torch.zeros(4, 2, 1, 64, 64, dtype=torch.int8)
    s = torch.zeros(4, 2, 1)
    good = (k, v, s, s.clone())
    calls = lambda p: (lambda: P.page_write(r, r, *p, table, i), lambda: P.page_read(*p, table, i, 1),  # noqa: E731
                       lambda: P.page_attention(r, *p, table, i), lambda: P.page_reserve(*p, table, refs, i, i),
                       lambda: P.page_compact(*p, table, refs))
    for call in calls(good):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    for bad in ((k.float(), v, s, s), (k, v[:3], s, s), (k, v.transpose(3, 4), s, s), (k, v, s[:3], s), (k, v, s, s.double()),
                (k[:, :, :63], v, s, s), (k.transpose(2, 3), v, s, s), (k[:, :1], v[:, :1].clone(), s[:, :1], s[:, :1]),
                (k[0], v[0], s[0], s[0])):
        for call in calls(bad):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: P.page_write(r, r[:1], *good, table, i), lambda: P.page_write(r, r, *good, table[0], i),
                 lambda: P.page_write(r, r, *good, table.long(), i), lambda: P.page_write(r, r, *good, table, i, path=i),
                 lambda: P.page_write(r, r, *good, table, i, refs=i), lambda: P.page_attention(r, *good, table, i, k_rows=r),
                 lambda: P.page_attention(r, *good, table, i, mask=torch.zeros(1, 2, dtype=torch.int64)),
                 lambda: P.page_reserve(*good, table, i, i, i), lambda: P.page_fork(table, i, refs, i, i[:1], 64),
                 lambda: P.page_fork(table, i, refs, i, i, 64)):
        with pytest.raises(ValueError):
            call()
    x, t, u = torch.zeros(2, 3, 9), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    for call in (lambda: P.draft_accept(x, t, u), lambda: P.draft_accept(x.int(), t, u), lambda: P.draft_accept(x, t[:1], u),
                 lambda: P.draft_accept(x, t, u, parents=t[:, :2]), lambda: P.draft_accept(x, t, u, probs=x[:, :2]),
                 lambda: P.draft_accept(x.transpose(1, 2), t, u), lambda: P.draft_accept(x, t.long(), u)):
        with pytest.raises(ValueError):
            call()


def test_tensors_that_require_a_gradient_are_refused():
    torch = pytest.importorskip("torch")
    P = pkg()
    i, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    k, v = torch.zeros(4, 2, 64, 64, dtype=torch.int8), torch.zeros(4, 2, 1, 64, 64, dtype=torch.int8)
    for which in range(4):
        r, q, s, x = torch.zeros(2, 1, 2, 64), torch.zeros(2, 1, 2, 64), torch.zeros(4, 2, 1), torch.zeros(2, 3, 9)
        (r, q, s, x)[which].requires_grad_(True)
        pool = (k, v, s, torch.zeros(4, 2, 1))
        calls = {0: lambda: P.page_write(r, r, *pool, table, i), 1: lambda: P.page_attention(q, *pool, table, i),
                 2: lambda: P.page_compact(*pool, table, i), 3: lambda: P.draft_accept(x, i, i)}
        with pytest.raises(ValueError, match="no gradient"):
            calls[which]()


def test_sizes_that_no_grid_holds_are_refused_before_anything_is_launched(capfd):
    """tables and pools whose second launch would fail after the first has changed the books"""
    assert compact(pages(), seqs=1 << 10, per=1 << 22) == -1
    assert "a table of" in capfd.readouterr().err
    assert compact(pages(), seqs=1 << 9, per=(1 << 22) - 1) == -1
    assert "not device memory" in capfd.readouterr().err
    for layers, says in ((1 << 12, "layers of"), ((1 << 11), "not device memory")):
        c = pages(n_layers=layers, n_pages=2, n_kv=1 << 13, hs=16, layer=1 << 24, id=1 << 23, head=1 << 10, s_layer=1 << 14,
                  s_id=1 << 13, s_head=1)
        for call in (compact, reserve):
            assert call(c) == -1
            assert says in capfd.readouterr().err
    wide = pages(n_kv=512, hs=16, id=512 * 1024, head=1024, s_id=512, s_head=1)
    for kw, says in ((dict(seqs=65536), "sequences of 512 kv heads"), (dict(seqs=32769), "sequences of 512 kv heads"),
                     (dict(seqs=32767), "not device memory")):
        assert attend(wide, heads=512, **kw) == -1
        assert says in capfd.readouterr().err
