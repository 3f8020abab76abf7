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


def _bwd_args(pkg, **over):
    a = _args(pkg)
    a.stat = a.dout = a.dq = a.dk = a.dv = a.ws = 4096
    a.ws_bytes = 1 << 60
    for n in ("dout_s", "dq_s", "dk_s", "dv_s"):
        setattr(a, n, (ctypes.c_int64 * 3)(1024, 128, 64))
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over", [dict(Lq=65535 * 128 + 1, bias=4096, dbias=4096), dict(H=65536, Hkv=65536, bias=4096, dbias=4096), dict(B=1 << 23), dict(B=1 << 22, mask=4096)])
def test_launch_limits_come_before_any_launch(pkg, over):
    """a call that some launch of it would refuse is refused as a whole (where there is no GPU, a launch would fail with another error)"""
    lib = pkg.hip.lib()
    a = _bwd_args(pkg, **over)
    assert lib.marship_cross_attn_bwd(ctypes.byref(a), None) == -1
    assert "than a launch takes" in lib.marship_last_error().decode()


@pytest.mark.parametrize("over", [dict(B=1 << 23), dict(B=1 << 22, mask=4096)])
def test_forward_launch_limits(pkg, over):
    lib = pkg.hip.lib()
    a = _bwd_args(pkg, **over)
    assert lib.marship_cross_attn(ctypes.byref(a), None) == -1
    assert "than a launch takes" in lib.marship_last_error().decode()


@pytest.mark.parametrize("shape", [(1 << 30, 1 << 30, 1, 1 << 29, 1, 8, 8), (1, 1 << 15, 1 << 14, 8, 8, 8, 8), (70000, 1, 8, 8, 8, 8, 8), (1, 1, 8, 1 << 29, 1, 8, 8), (0, 1, 8, 1, 8, 1, 8)])
def test_bias_workspace_of_a_refused_shape_is_none(pkg, shape):
    """the count of workgroups left 64 bits, came out as zero and was divided by"""
    lib = pkg.hip.lib()
    P = ctypes.c_void_p(4096)
    assert lib.marship_bucket_bias_bwd_ws(*shape) == 0
    assert lib.marship_bucket_bias_bwd(P, 1 << 62, 1 << 40, P, P, P, *shape, P, 1 << 60, None) == -1


def test_bias_workspace_is_counted_in_64_bits(pkg):
    """2^31 workgroups: the largest grids the call takes, in more than 32 bits (and more than a launch takes)"""
    lib = pkg.hip.lib()
    P = ctypes.c_void_p(4096)
    shape = (1, 1 << 20, 1, 1 << 17, 1, 8, 8)
    assert lib.marship_bucket_bias_bwd_ws(*shape) == (1 << 31) * 64 * 4
    assert lib.marship_bucket_bias_bwd(P, 1 << 62, 1 << 17, P, P, P, *shape, P, 1 << 60, None) == -1
    assert "more workgroups" in lib.marship_last_error().decode()
