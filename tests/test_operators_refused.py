"""Further calls that the operators on device memory refuse (no GPU: nothing here reaches one)."""
import ctypes as C

import pytest

from helpers import pkg
from test_operators import cache, rows


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38])
def test_softmax_scales_refused(scale, capfd):
    c, q = cache(), rows()
    assert pkg().lib().llm_tree_attention(C.byref(c), C.byref(q), C.byref(q), 4, 0x10000, None, None, 1, 10, scale, 0, None, 0,
                                          None) == -1
    assert "llm_tree_attention: scale" in capfd.readouterr().err
