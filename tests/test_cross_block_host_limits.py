"""The cross-attention block's C-ABI on shapes that its calls refuse (nothing is launched)."""
import ctypes

import pytest

from tests.test_cross_block_host import _args


@pytest.mark.parametrize("over", [dict(H=1, Hkv=2), dict(H=3, Hkv=2), dict(hd=136), dict(Lk=(1 << 31) - 1), dict(Lq=1 << 30), dict(B=1 << 30, H=4)])
@pytest.mark.parametrize("backward", [0, 1])
def test_workspace_of_a_refused_shape_is_none(pkg, over, backward):
    """fewer query heads than key heads left no row block, and the query divided by it"""
    lib = pkg.hip.lib()
    a = _args(pkg, **over)
    assert lib.marship_cross_attn_ws(ctypes.byref(a), backward) == 0
    assert lib.marship_cross_attn(ctypes.byref(a), None) == -1
