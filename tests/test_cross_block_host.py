"""The cross-attention block's host side: bucket maps, workspace sizes, and the C-ABI's own refusals (nothing is launched)."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ops


def _bucket(d, buckets, reach):
    """the rule by its words, borders by exact comparison"""
    side = buckets // 2
    near = side // 2
    n = abs(d)
    if n < near:
        b = n
    else:
        steps = side - near
        b = near + max(t for t in range(steps) if n ** steps * near ** t >= reach ** t * near ** steps)
    return b + (side if d > 0 else 0)


@pytest.mark.parametrize("nq,nk,buckets,reach", [(1, 1, 8, 16), (5, 9, 8, 16), (40, 40, 32, 128), (1, 300, 32, 128), (200, 3, 16, 20), (64, 64, 32, 64), (3, 3, 4, 2)])
def test_bucket_map(ops, nq, nk, buckets, reach):
    m = ops.bucket_map(nq, nk, buckets, reach)
    assert m.dtype == torch.int32 and m.tolist() == [_bucket(d, buckets, reach) for d in range(-(nq - 1), nk)]
    assert 0 <= int(m.min()) and int(m.max()) < buckets


def test_bucket_map_borders_and_sides(ops):
    # 8 buckets a side, 4 of them shared up to 64: borders 4, 8, 16, 32 exactly
    m = ops.bucket_map(101, 101, 16, 64)
    side = {d: int(m[100 + d]) for d in range(-100, 101)}
    assert [side[-d] for d in (0, 1, 2, 3, 4, 7, 8, 15, 16, 31, 32, 63, 64, 100)] == [0, 1, 2, 3, 4, 4, 5, 5, 6, 6, 7, 7, 7, 7]
    assert all(side[d] == side[-d] + 8 for d in range(1, 101))
    one = ops.bucket_map(101, 101, 8, 64, bidirectional=False)
    assert all(int(one[100 + d]) == 0 for d in range(1, 101)) and [int(one[100 - d]) for d in (0, 3, 4, 8, 64)] == [0, 3, 4, 5, 7]
    # a single query at position 40 sees row 40 of the whole map
    assert torch.equal(ops.bucket_map(1, 101, 16, 64, offset=40), m[60:161])


def test_bucket_map_refusals(ops):
    for a, kw in (((0, 4, 8, 16), {}), ((4, 4, 7, 16), {}), ((4, 4, 2, 16), {}), ((4, 4, 8, 2), {}), ((4, 4, 1, 16), dict(bidirectional=False))):
        with pytest.raises(ValueError, match="bucket_map"):
            ops.bucket_map(*a, **kw)


def _args(pkg, **over):
    a = pkg.hip.MarsCrossAttn()
    a.q = a.k = a.v = a.out = 4096
    for n in ("q_s", "k_s", "v_s", "out_s"):
        setattr(a, n, (ctypes.c_int64 * 3)(1024, 128, 64))
    a.B, a.Lq, a.Lk, a.H, a.Hkv, a.hd, a.scale, a.dtype = 1, 8, 8, 2, 2, 64, 0.125, 1
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(q=None), "null"), (dict(dtype=2), "dtype"), (dict(B=0), "bad shape"), (dict(Lk=-1), "bad shape"), (dict(Hkv=3), "multiple"), (dict(hd=136), "head dim"),
    (dict(hd=12), "head dim"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(k=4100), "aligned"), (dict(v_s=(ctypes.c_int64 * 3)(1024, 4, 64)), "aligned"),
    (dict(mask=4096), "workspace")])
def test_cross_attn_c_refusals(pkg, over, text):
    lib = pkg.hip.lib()
    a = _args(pkg, **over)
    assert lib.marship_cross_attn(ctypes.byref(a), None) == -1
    assert text in lib.marship_last_error().decode()


@pytest.mark.parametrize("over,text", [(dict(), "null"), (dict(dbias=4096), "bias that is not there"), (dict(dq_s=(ctypes.c_int64 * 3)(1, 128, 64)), "aligned"), (dict(ws=None), "workspace")])
def test_cross_attn_bwd_c_refusals(pkg, over, text):
    lib = pkg.hip.lib()
    a = _args(pkg)
    if over:
        a.stat = a.dout = a.dq = a.dk = a.dv = 4096
        for n in ("dout_s", "dq_s", "dk_s", "dv_s"):
            setattr(a, n, (ctypes.c_int64 * 3)(1024, 128, 64))
        for n, v in over.items():
            setattr(a, n, v)
    assert lib.marship_cross_attn_bwd(ctypes.byref(a), None) == -1
    assert text in lib.marship_last_error().decode()


def test_other_c_refusals(pkg):
    lib = pkg.hip.lib()
    P = ctypes.c_void_p(4096)
    err = lambda: lib.marship_last_error().decode()
    assert lib.marship_bucket_bias(None, P, P, P, 64, 8, 1, 1, 8, 1, 8, 1, 8, None) == -1 and "null" in err()
    assert lib.marship_bucket_bias(P, P, P, P, 64, 7, 1, 1, 8, 1, 8, 1, 8, None) == -1 and "overlap" in err()
    assert lib.marship_bucket_bias(P, P, P, P, 64, 8, 1, 0, 8, 1, 8, 1, 8, None) == -1 and "empty" in err()
    assert lib.marship_bucket_bias_bwd(P, 64, 8, P, P, P, 1, 1, 8, 1, 8, 1, 8, None, 0, None) == -1 and "workspace" in err()
    gn = lambda N=1, PP=4, C=8, G=2, act=0, ws=P, nws=1 << 20, xd=0: lib.marship_group_norm_act(P, 32, 8, P, P, P, 32, 8, N, PP, C, G, 1e-5, act, xd, 0, None, ws, nws, None)
    assert gn(N=0) == -1 and "bad shape" in err()
    assert gn(G=3) == -1 and "divide" in err()
    assert gn(act=5) == -1 and "activation" in err()
    assert gn(xd=3) == -1 and "dtype" in err()
    assert gn(nws=8) == -1 and "workspace" in err()
    assert lib.marship_group_norm_act_bwd(P, 32, 8, P, P, None, P, 32, 8, P, 32, 8, P, P, 1, 4, 8, 2, 0, 0, 0, P, 1 << 20, None) == -1 and "null" in err()


def test_workspace_sizes(pkg):
    lib = pkg.hip.lib()
    a = _args(pkg)
    assert lib.marship_cross_attn_ws(ctypes.byref(a), 0) == 0                                # eight rows, eight keys: one launch
    a.Lk = 100000
    assert lib.marship_cross_attn_ws(ctypes.byref(a), 0) > 0                                 # a long axis is cut
    assert lib.marship_cross_attn_ws(None, 0) == 0
    assert lib.marship_group_norm_act_ws(2, 100, 64, 3, 0) == 0                              # (refused by the call itself)
