"""Attention between two token sets where it once went wrong, or could: very large scores with a bias, a few attended keys of a long axis."""
import ctypes
import math

import pytest
import torch

from tests.test_gpu_cross_attn import DT, U32, check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bias", [None, "rand", "inf", "low"])
@pytest.mark.parametrize("Lq,keys", [(128, "all"), (33, "all"), (70, "mask"), (96, "len"), (97, "all")])
def test_gradients_of_large_scores(pkg, cuda, dtype, bias, Lq, keys):
    """Raw scores far above 88.7, where exp leaves f32: in rows that are the last of a tile, and in the last row of all, which a tile that ends behind it
    holds again.  Query rows in whole tiles (128) and not (of 32 rows: 33, 70, 97; of 64: 96 too)."""
    c = make(cuda, dtype, 2, Lq, 130, 4, 2, 64, seed=Lq, keys=keys, bias=bias)
    c["q"] = c["q"] * 40
    on = c["att"][0].to(cuda)
    last = c["q"][0, -1, 1].float() @ c["k"][0, on, 0].float().t() * c["scale"]        # (rows of heads 0 and 1 are one list: the last is head 1's)
    assert float(last.max()) > 100
    check(pkg, c)


@pytest.mark.parametrize("how", ["mask", "len"])
@pytest.mark.parametrize("bias", [None, "rand"])
@pytest.mark.parametrize("hd", [16, 64, 80, 128])
def test_masked_keys_and_absent_keys_give_the_same_gradient(pkg, cuda, how, bias, hd):
    """dQ over the attended keys of a long axis against dQ over those keys alone, bf16: the same precision however the keys are left out.

    Both calls multiply the same numbers and differ in the order of f32 sums over n keys: by at most c U32 M for a sum of magnitudes M, with c = n + 8 for each of
    them, on a value x before its rounding to bf16.  A rounding turns that into a whole step (at most 2^-7 |x|) with probability c U32 M / step and into
    nothing otherwise, so the squares of the differences add up to about sum c U32 M 2^-7 |x|; four times that for the spread of a count of flips."""
    counts = [70, 256, 257, 300]
    c = make(cuda, torch.bfloat16, 4, 150, 1369, 2, 2, hd, seed=hd, bias=bias)
    g = torch.Generator().manual_seed(hd)
    att = torch.zeros(4, 1369, dtype=torch.bool)
    for b, n in enumerate(counts):
        att[b, torch.randperm(1369, generator=g)[:n] if how == "mask" else torch.arange(n)] = True
    c["att"] = att
    if how == "mask":
        c["mask"] = att.to(cuda)
    else:
        c["kv_len"] = torch.tensor(counts, dtype=torch.int32, device=cuda)
    got = run(pkg, c)["dq"]
    for b, n in enumerate(counts):
        keys = torch.nonzero(att[b]).flatten().to(cuda)
        one = dict(c, B=1, Lk=n, att=torch.ones(1, n, dtype=torch.bool), mask=None, kv_len=None, k=c["k"][b:b + 1, keys].contiguous(), v=c["v"][b:b + 1, keys].contiguous(),
                   bias=None if bias is None else c["bias"][:, :, keys].contiguous())
        for x in ("q", "dout"):
            one[x] = c[x][b:b + 1].contiguous()
        want = run(pkg, one)["dq"][0].double()
        bound = 0.0
        for h in range(2):
            Q, K, V, dO = (one[x][0, :, h].double() for x in ("q", "k", "v", "dout"))
            S = Q @ K.t() * c["scale"] + (0.0 if bias is None else one["bias"][h].double())
            P = torch.softmax(S, 1)
            D = (dO * (P @ V)).sum(1, keepdim=True)
            dS = (P * (dO @ V.t() - D)).abs() + P * 2.0 ** -8 * (dO.abs() * (P @ V).abs()).sum(1, keepdim=True)      # (dS' with D from a rounded O)
            M = c["scale"] * (dS @ K.abs() + dS.sum(1, keepdim=True) * (P @ K.abs()))
            bound += float((2 * (n + 8) * U32 * M * 2.0 ** -7 * want[:, h].abs()).sum())
        diff = float((got[b].double() - want).square().sum())
        assert diff <= 4 * bound, f"{n} keys: {(diff / float(want.square().sum())) ** 0.5:.2e} of the norm, bound {(4 * bound / float(want.square().sum())) ** 0.5:.2e}"


def test_scale_is_taken_by_value(pkg, cuda):
    """a scale that comes as a zero-dimensional tensor or a numpy number counts by its value at the call, also the second time"""
    c = make(cuda, torch.float32, 1, 9, 30, 2, 2, 16, seed=3)
    stat, res = torch.empty(1, 2, 9, 2, device=cuda), {}
    outs = lambda: [torch.empty_like(c[n]) for n in ("q", "q", "k", "v")]
    held = torch.tensor(0.25)
    for value in (0.25, 0.75):
        held.fill_(value)
        for name, scale in (("float", value), ("tensor", held), ("numpy", held.numpy()[()])):
            out, dq, dk, dv = res[name] = outs()
            pkg.ops.cross_attn(c["q"], c["k"], c["v"], out, stat=stat, scale=scale)
            pkg.ops.cross_attn_bwd(c["q"], c["k"], c["v"], out, stat, c["dout"], dq, dk, dv, scale=scale)
        for name in ("tensor", "numpy"):
            assert all(torch.equal(a, b) for a, b in zip(res[name], res["float"])), name


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq", [5, 150])
@pytest.mark.parametrize("Lk,keys", [(64, "all"), (65, "all"), (33, "all"), (100, "mask"), (100, "len"), (3000, "mask"), (3001, "all")])
def test_infinite_value_of_the_last_key(pkg, cuda, dtype, Lq, Lk, keys):
    """an overflowed value of the last attended key is an infinity in its own column of the result and nothing anywhere else, whether a tile of keys ends
    with that key or not (what a tile holds behind it is that key again)"""
    c = make(cuda, dtype, 2, Lq, Lk, 4, 2, 64, seed=Lk, keys=keys)
    last = int(torch.nonzero(c["att"][0]).max())
    c["v"][0, last, 1, 7] = 0.0
    want = run(pkg, c, backward=False)["out"].clone()
    c["v"][0, last, 1, 7] = math.inf
    got = run(pkg, c, backward=False)["out"]
    assert bool((got[0, :, 2:, 7] == math.inf).all())
    got[0, :, 2:, 7] = want[0, :, 2:, 7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,Lq,Lk", [(torch.float32, 300, 1100), (torch.bfloat16, 300, 5000)])
@pytest.mark.parametrize("keys,bias", [("all", None), ("mask", "rand")])
def test_keys_cut_where_a_round_of_workgroups_is_left_over(pkg, cuda, dtype, Lq, Lk, keys, bias):
    """384 blocks of query rows on 256 CUs: the keys are cut in two or more and joined"""
    c = make(cuda, dtype, 2, Lq, Lk, 64, 64, 64, seed=7, keys=keys, bias=bias)
    a = pkg.ops._cross_block("test", c["q"], c["k"], c["v"], torch.empty_like(c["q"]), None, c["scale"], c["kv_len"], None, c["bias"])
    assert pkg.hip.lib().marship_cross_attn_ws(ctypes.byref(a), 0) > 0
    check(pkg, c, backward=False)
