"""Tensors that the operators change in place, as torch's autograd sees them."""
import pytest

from helpers import pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_changes_in_place_are_counted():
    """a graph that saved a cache, or an output, refuses its backward pass after the operators have written it"""
    P = pkg()
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    rows = torch.randn(1, 3, 2, 64, device=DEV)

    def new():
        return (torch.randn(1, 2, 8, 64, device=DEV), torch.randn(1, 2, 8, 64, device=DEV))

    def write(k, v, r, o):
        P.kv_write(rows, rows, k, v, pos)

    def read(k, v, r, o):
        P.kv_read(k, v, pos, 3, out=(r, r.clone()))

    def attend(k, v, r, o):
        P.tree_attention(torch.ones_like(o), k, v, pos, out=o)

    for call, changed in ((write, {0, 1}), (read, {2}), (attend, {3})):
        k, v = new()
        r, o = torch.zeros(1, 3, 2, 64, device=DEV), torch.zeros(1, 3, 4, 64, device=DEV)
        for i, t in enumerate((k, v, r, o)):
            w = torch.ones_like(t, requires_grad=True)
            y = (w * t).sum()
            call(k, v, r, o)
            if i in changed:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.backward()
            else:
                y.backward()
    # scales too, and in inference mode nothing is counted or refused
    k, v = (x.to(torch.int8) for x in new())
    s = [torch.ones(1, 2, 8, device=DEV) for _ in range(2)]
    before = [t._version for t in (k, v, *s)]
    P.kv_write(rows, rows, k, v, pos, k_scale=s[0], v_scale=s[1])
    assert all(t._version > n for t, n in zip((k, v, *s), before))
    with torch.inference_mode():
        k, v = new()
        P.kv_write(rows, rows, k, v, pos)
        P.kv_read(k, v, pos, 3, out=(torch.zeros_like(rows), torch.zeros_like(rows)))
