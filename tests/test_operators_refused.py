"""Further calls that the operators on device memory refuse (no GPU: nothing here reaches one)."""
import ctypes as C

import pytest

from helpers import pkg
from test_operators import F32, cache, rows


def test_tensors_that_require_a_gradient_are_refused():
    """where gradients are on; without them the next refusal is that of host tensors"""
    torch = pytest.importorskip("torch")
    P = pkg()
    names = ("k_rows", "v_rows", "k", "v", "k_scale", "v_scale", "q", "out", "logits")
    for which in names:
        k = [torch.zeros(1, 2, 8, 64) for _ in range(2)]
        r = [torch.zeros(1, 1, 2, 64) for _ in range(2)]
        s = [torch.zeros(1, 2, 8) for _ in range(2)]
        q, out, logits, i = torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4, 64), torch.zeros(2, 10), torch.zeros(1, dtype=torch.int32)
        dict(zip(names, (*r, *k, *s, q, out, logits)))[which].requires_grad_(True)
        c = [torch.zeros(1, 2, 8, 64, dtype=torch.int8) for _ in range(2)] if "scale" in which else k
        kw = dict(k_scale=s[0], v_scale=s[1]) if "scale" in which else {}
        calls = {"kv_write": lambda: P.kv_write(*r, *c, i, **kw), "kv_read": lambda: P.kv_read(*c, i, 1, out=r, **kw),
                 "tree": lambda: P.tree_attention(q, *c, i, out=out, **kw), "logprobs": lambda: P.logprobs(logits)}
        for name, call in calls.items():
            if which in {"kv_write": names[:6], "kv_read": names[:6], "tree": names[2:8], "logprobs": names[8:]}[name]:
                with pytest.raises(ValueError, match="no gradient"):
                    call()
                with torch.no_grad(), pytest.raises(ValueError, match="device tensors"):
                    call()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38])
def test_softmax_scales_refused(scale, capfd):
    c, q = cache(), rows()
    assert pkg().lib().llm_tree_attention(C.byref(c), C.byref(q), C.byref(q), 4, 0x10000, None, None, 1, 10, scale, 0, None, 0,
                                          None) == -1
    assert "llm_tree_attention: scale" in capfd.readouterr().err


def test_memory_that_lies_on_itself_is_not_written(capfd):
    """strides of zero where there is more than one, in what a call writes"""
    L = pkg().lib()
    at = 0x10000

    def write(**kw):
        c, r = cache(**kw), rows()
        return L.llm_kv_write(C.byref(c), C.byref(r), C.byref(r), at, None, 2, None)

    def read(n=2, **kw):
        c, r, o = cache(n_seq=2), rows(), rows(**kw)
        return L.llm_kv_read(C.byref(c), C.byref(r), C.byref(o), at, None, n, 0, None)

    def attend(n=2, **kw):
        c, q, o = cache(n_seq=2), rows(), rows(**kw)
        return L.llm_tree_attention(C.byref(c), C.byref(q), C.byref(o), 4, at, None, None, n, 10, 0.1, 0, None, 0, None)

    for call in (lambda: write(n_seq=2, seq=0), lambda: write(head=0), lambda: write(n_seq=2, s_seq=0), lambda: write(s_head=0),
                 lambda: read(seq=0), lambda: read(tok=0), lambda: read(head=0), lambda: attend(seq=0), lambda: attend(tok=0),
                 lambda: attend(head=0)):
        assert call() == -1
        assert "a stride of zero" in capfd.readouterr().err
    # of one there is nothing to lie on: these are refused for their addresses
    for call in (lambda: write(seq=0, s_seq=0), lambda: write(type=F32, s_head=0), lambda: read(n=1, tok=0),
                 lambda: attend(n=1, tok=0)):
        assert call() == -1
        assert "not device memory" in capfd.readouterr().err


def test_masks_of_another_shape_are_refused():
    torch = pytest.importorskip("torch")
    k, q = torch.zeros(2, 2, 8, 64), torch.zeros(2, 3, 4, 64)
    lens = torch.zeros(2, dtype=torch.int32)
    for shape in ((3, 2), (1, 6), (2, 3, 1)):
        with pytest.raises(ValueError, match="mask"):
            pkg().tree_attention(q, k, k, lens, mask=torch.zeros(shape, dtype=torch.int64))
    for shape in ((2, 3), (6,)):
        with pytest.raises(ValueError, match="device tensors"):
            pkg().tree_attention(q, k, k, lens, mask=torch.zeros(shape, dtype=torch.int64))
