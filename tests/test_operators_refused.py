"""Further calls that the operators on device memory refuse (no GPU: nothing here reaches one)."""
import ctypes as C

import pytest

from helpers import pkg
from test_operators import cache, rows


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
