"""What the operators on device memory refuse (no GPU: nothing here reaches one)."""
import ctypes as C

import pytest

from helpers import pkg

F32, BF16, I8, E4M3 = range(4)


def cache(type=I8, n_seq=1, n_kv=2, hs=64, ctx=32, **kw):
    P = pkg()
    mem = 0x10000
    d = dict(k=mem, v=mem, k_scale=mem, v_scale=mem, type=type, n_seq=n_seq, n_kv=n_kv, hs=hs, ctx=ctx,
             seq=n_kv * ctx * hs, head=ctx * hs, pos=hs, s_seq=n_kv * ctx, s_head=ctx, s_pos=1)
    d.update(kw)
    return P.LlmKv(**d)


def rows(type=F32, **kw):
    d = dict(p=0x10000, type=type, seq=128, tok=128, head=64)
    d.update(kw)
    return pkg().LlmRows(**d)


def write(c, r=None, v=None, n=1):
    r = r or rows()
    return pkg().lib().llm_kv_write(C.byref(c), C.byref(r), C.byref(v or r), 0x10000, None, n, None)


def attend(c, q=None, out=None, heads=4, n=1, work=0):
    q = q or rows()
    return pkg().lib().llm_tree_attention(C.byref(c), C.byref(q), C.byref(out or q), heads, 0x10000, None, None, n, 10, 0.1,
                                          0, None, work, None)


def logp(type=F32, rows=1, vocab=100, stride=100, t=1.0, n=0, top=0, p=0x10000):
    return pkg().lib().llm_logprobs(p, type, rows, vocab, stride, t, None, n, None, None, None, top, None, None, None, 0,
                                    None)


@pytest.mark.parametrize("kw,says", [
    (dict(type=4), "type 4"), (dict(hs=8), "8 values"), (dict(hs=72), "72 values"), (dict(hs=272), "272 values"),
    (dict(n_kv=0), "0 heads"), (dict(ctx=0), "0 positions"), (dict(n_seq=-1), "-1 sequences"),
    (dict(pos=63), "multiples of 4"), (dict(pos=62), "multiples of 4"), (dict(pos=48), "at least a row"),
    (dict(pos=(16 << 20) + 4), "16 MiB"), (dict(k=0x10001), "multiples of 4"), (dict(head=-64), "multiples of 4"),
    (dict(), "not device memory"), (dict(k=0, v=0), "not device memory")])
def test_caches_refused(kw, says, capfd):
    for f in (write, attend):
        assert f(cache(**kw)) == -1
        assert says in capfd.readouterr().err


def test_arguments_refused(capfd):
    assert write(cache(), n=-1) == -1
    assert attend(cache(), heads=3) == -1
    assert attend(cache(), heads=0) == -1
    assert attend(cache(), heads=2 * 65) == -1
    assert attend(cache(), n=65) == -1
    assert attend(cache(), n=-1) == -1
    for kw in (dict(type=I8), dict(rows=-1), dict(vocab=0), dict(rows=2, stride=99), dict(t=0.0), dict(t=-1.0),
               dict(t=float("nan")), dict(t=float("inf")), dict(n=-1), dict(top=33), dict(vocab=4, top=5), dict(top=-1),
               dict(p=0x10002), dict(vocab=(1 << 28) + 1, stride=1 << 29)):
        assert logp(**kw) == -1
    err = capfd.readouterr().err
    assert err.count("bad arguments") == 20
    assert logp() == -1
    assert "logits is not device memory" in capfd.readouterr().err


def test_nothing_to_do():
    assert write(cache(n_seq=0)) == 0
    assert attend(cache(n_seq=0)) == 0
    assert logp(rows=0) == 0


def test_work_sizes():
    L = pkg().lib()
    c = cache(ctx=32768)
    assert L.llm_tree_attention_work(C.byref(c), 3, 1, 100) == 0
    assert L.llm_tree_attention_work(C.byref(c), 4, 1, 100) == 0  # one slice
    b = L.llm_tree_attention_work(C.byref(c), 4, 1, 32767)
    assert b >= 2 * 2 * (64 + 2) * 4 and b % 8 == 0  # at least a slice for each kv head
    assert L.llm_logprobs_work(1000, 151936, 20) == 0
    assert L.llm_logprobs_work(1, 65536, 20) > 0


def test_tensors_refused():
    torch = pytest.importorskip("torch")
    P = pkg()
    k = torch.zeros(1, 2, 8, 64)
    r = torch.zeros(1, 1, 2, 64)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        P.kv_write(r, r, k, k, i)
    with pytest.raises(ValueError):
        P.kv_read(k, k, i, 1)
    with pytest.raises(ValueError):
        P.tree_attention(torch.zeros(1, 1, 4, 64), k, k, i)
    with pytest.raises(ValueError):
        P.logprobs(torch.zeros(2, 10))


def test_models_refused():
    """a NULL model and bad arguments, before any device is touched"""
    L = pkg().lib()
    ids = (C.c_int * 2)(1, 2)
    assert L.llm_set_kv(None, 0) == -1 and L.llm_get_kv(None) == -1
    assert L.llm_verify(None, 0, ids, None, 2, None, None, None) == -1
    assert L.llm_keep(None, 0, ids, 2) == -1
    assert L.llm_score(None, ids, 2, 1.0, None, None, 0, None, None) == -1
