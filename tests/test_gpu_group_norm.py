"""Group norm with an activation on channels-last maps, forward and backward, against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = 2.0 ** -24


def _act(z, act):
    """value and slope"""
    if act == 1:
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act in (2, 4):
        a = 1.702 if act == 2 else 1.0
        s = torch.sigmoid(a * z)
        return z * s, s + a * z * s * (1 - s)
    if act == 3:
        return z.clamp_min(0), (z > 0).double()
    return z, torch.ones_like(z)


def reference(x, w, b, dy, G, act, out_dtype):
    """results in 64 bits and how far f32 statistics, f32 elementwise arithmetic and one final rounding may be off.

    mean and rstd: sums of n values joined in pieces of a few thousand at most; with X the largest magnitude of the group, the mean is off by at most
    c U X and (x - mean) by (c + 2) U X; rstd by c U of itself and by the share of the mean's error in the deviations."""
    N, P, C = x.shape
    x, dy, w, b = x.double(), dy.double(), w.double(), b.double()
    g = x.reshape(N, P, G, C // G)
    n = P * (C // G)
    mean = g.mean((1, 3), keepdim=True)
    var = ((g - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + EPS)
    X = g.abs().amax((1, 3), keepdim=True)
    c = 64 + min(n, 4096) / 8                                       # longest chain of additions a value passes through, with room
    xh = (g - mean) * rstd
    e_xh = c * U * (X * rstd + xh.abs() * (2 + X * rstd * X * rstd * U * c))
    w4, b4 = w.view(G, C // G), b.view(G, C // G)
    z = xh * w4 + b4
    e_z = e_xh * w4.abs() + 2 * U * (xh * w4).abs() + U * z.abs()
    y, slope = _act(z, act)
    e_y = 1.2 * e_z + 16 * U * (y.abs() + z.abs())                  # (slopes are below 1.13; exponential, division and erf: a few U each)
    half = torch.finfo(out_dtype).eps / 2
    res = dict(out=y, mean=mean, rstd=rstd)
    tol = dict(out=e_y + half * (y.abs() + e_y) + 1e-30)
    dz = dy.reshape(N, P, G, C // G) * slope
    curve = {0: 0.0, 1: 0.8, 2: 0.9, 3: 0.0, 4: 0.5}[act]           # bounds of the second derivative
    e_dz = dy.reshape(N, P, G, C // G).abs() * (curve * e_z + 16 * U * (slope.abs() + z.abs()))
    res["db"], res["dw"] = dz.sum((0, 1)).view(C), (dz * xh).sum((0, 1)).view(C)
    k = 64 + P / 8 + N
    tol["db"] = (e_dz + k * U * dz.abs()).sum((0, 1)).view(C) + 1e-30
    tol["dw"] = (e_dz * xh.abs() + dz.abs() * e_xh + k * U * (dz * xh).abs()).sum((0, 1)).view(C) + 1e-30
    dh = dz * w4
    m1, m2 = dh.mean((1, 3), keepdim=True), (dh * xh).mean((1, 3), keepdim=True)
    e_dh = e_dz * w4.abs() + U * dh.abs()
    e_m1 = e_dh.mean((1, 3), keepdim=True) + (k + c) * U * dh.abs().mean((1, 3), keepdim=True)
    e_m2 = (e_dh * xh.abs() + dh.abs() * e_xh).mean((1, 3), keepdim=True) + (k + c) * U * (dh * xh).abs().mean((1, 3), keepdim=True)
    res["dx"] = rstd * (dh - m1 - xh * m2)
    mag = dh.abs() + m1.abs() + (xh * m2).abs()
    e = rstd * (e_dh + e_m1 + e_xh * m2.abs() + xh.abs() * e_m2 + 2 * c * U * mag)
    for n_ in ("out", "dx"):
        res[n_] = res[n_].reshape(N, P, C)
    tol["out"] = tol["out"].reshape(N, P, C)
    tol["dx"] = e.reshape(N, P, C)
    return res, tol


def check(pkg, cuda, N, P, C, G, act, dx_t=torch.float32, dy_t=torch.float32, pad=0, off=0, shift=0.0, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rows(t, dtype):
        buf = torch.full((N, P + 1, C + pad + off), 7.0, dtype=dtype, device=cuda)
        view = buf[:, :P, off:off + C]
        if t is not None:
            view.copy_(t)
        return buf, view

    x0 = torch.randn(N, P, C, generator=g) * (0.3 + torch.rand(C, generator=g)) + shift + torch.randn(C, generator=g) * 0.5
    _, x = rows(x0, dx_t)
    _, dy = rows(torch.randn(N, P, C, generator=g), dy_t)
    w, b = (1 + 0.3 * torch.randn(C, generator=g)).to(cuda), (0.3 * torch.randn(C, generator=g)).to(cuda)
    if act == 3:                                                    # the slope of ReLU jumps at 0: arguments that stay off it
        w, b = w * 0.1, torch.where(b > 0, torch.ones_like(b), -torch.ones_like(b))
    obuf, out = rows(None, dy_t)
    dbuf, dx = rows(None, dx_t)
    stat = torch.full((N, G, 2), math.nan, device=cuda)
    dw, db = torch.full((C,), math.nan, device=cuda), torch.full((C,), math.nan, device=cuda)
    pkg.ops.group_norm_act(x, w, b, out, G, EPS, act, stat=stat)
    pkg.ops.group_norm_act_bwd(x, w, b, stat, dy, dx, dw, db, G, act)
    res, tol = reference(x, w, b, dy, G, act, dy_t)
    tol["dx"] = tol["dx"] + torch.finfo(dx_t).eps / 2 * (res["dx"].abs() + tol["dx"]) + 1e-30
    for n in ("out", "dx", "dw", "db"):
        t = dict(out=out, dx=dx, dw=dw, db=db)[n]
        err = (t.double() - res[n]).abs()
        worst = float((err / tol[n]).max())
        assert worst <= 1.0, f"{n}: {worst:.2f} of the bound, error {float(err.max()):.3e}"
    for buf in (obuf, dbuf):
        assert bool((buf[:, P:] == 7).all()) and bool((buf[..., :off] == 7).all()) and bool((buf[..., off + C:] == 7).all())
    # without statistics to keep the same result, and in place (rows laid out alike: the alignment chooses the order of the sums)
    _, again = rows(None, dy_t)
    pkg.ops.group_norm_act(x, w, b, again, G, EPS, act)
    assert torch.equal(again, out)
    if dx_t == dy_t:
        _, y = rows(x, dx_t)
        pkg.ops.group_norm_act(y, w, b, y, G, EPS, act)
        assert torch.equal(y, out)
        _, d = rows(dy, dy_t)
        pkg.ops.group_norm_act_bwd(x, w, b, stat, d, d, dw, db, G, act)
        assert torch.equal(d, dx)


T = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("dtype", T)
def test_activations(pkg, cuda, act, dtype):
    check(pkg, cuda, 2, 150, 64, 8, act, dtype, dtype, seed=act)


@pytest.mark.parametrize("dx_t,dy_t", [(a, b) for a in T for b in T])
def test_types(pkg, cuda, dx_t, dy_t):
    check(pkg, cuda, 3, 77, 96, 4, 4, dx_t, dy_t, seed=1)


@pytest.mark.parametrize("N,P,C,G", [(1, 1, 8, 1), (1, 1, 16, 2), (2, 1369, 64, 32), (1, 5, 2048, 1), (1, 300, 4104, 3), (1, 9, 4096, 64), (5, 33, 24, 8), (2, 50, 30, 3),
                                     (3, 40, 7, 7), (2, 17, 10, 1), (1, 4096, 32, 4), (40, 3, 40, 5), (1, 20000, 8, 1), (2, 70, 1000, 125)])
@pytest.mark.parametrize("dtype", T)
def test_shapes(pkg, cuda, N, P, C, G, dtype):
    check(pkg, cuda, N, P, C, G, 4, dtype, dtype, seed=P + C)


@pytest.mark.parametrize("pad,off", [(8, 8), (3, 0), (0, 1), (2, 2), (4, 4)])
@pytest.mark.parametrize("dtype", T)
def test_rows_and_alignment(pkg, cuda, pad, off, dtype):
    check(pkg, cuda, 2, 61, 48, 6, 1, dtype, dtype, pad=pad, off=off, seed=pad)


def test_means_far_from_zero(pkg, cuda):
    """a mean a thousand times the spread: the variance is not taken from a difference of large sums"""
    check(pkg, cuda, 2, 500, 64, 8, 0, shift=1000.0, seed=3)


def test_constant_group_and_nan(pkg, cuda):
    x = torch.full((2, 30, 16), 3.0, device=cuda)
    w, b, out = torch.ones(16, device=cuda), torch.full((16,), 0.25, device=cuda), torch.empty(2, 30, 16, device=cuda)
    pkg.ops.group_norm_act(x, w, b, out, 2, EPS)
    assert bool((out == 0.25).all())
    x[0, 3, 2] = math.nan
    pkg.ops.group_norm_act(x, w, b, out, 2, EPS)
    assert bool(torch.isnan(out[0, :, :8]).all()) and bool((out[0, :, 8:] == 0.25).all()) and bool((out[1] == 0.25).all())


def test_groups_of_one_value_have_no_gradient(pkg, cuda):
    x, dy, w, b = (torch.randn(*s, device=cuda) for s in ((3, 1, 24), (3, 1, 24), (24,), (24,)))
    stat, out, dx, dw, db = (torch.empty(*s, device=cuda) for s in ((3, 24, 2), (3, 1, 24), (3, 1, 24), (24,), (24,)))
    pkg.ops.group_norm_act(x, w, b, out, 24, EPS, 4, stat=stat)
    assert torch.equal(stat[..., 0], x[:, 0])
    pkg.ops.group_norm_act_bwd(x, w, b, stat, dy, dx, dw, db, 24, 4)
    assert bool((dx == 0).all()) and bool((dw == 0).all())


@pytest.mark.parametrize("act", [0, 1, 2, 4])
def test_gradients_against_differences(pkg, cuda, act):
    """<gradient, direction> against central differences of the definition in 64 bits (step 1e-4: off by about 1e-8 of the magnitudes)"""
    N, P, C, G = 2, 23, 24, 3
    g = torch.Generator().manual_seed(act)
    x, dy, w, b = (torch.randn(*s, generator=g) for s in ((N, P, C), (N, P, C), (C,), (C,)))
    dev = [t.to(cuda) for t in (x, w, b)]
    stat, out, dx, dw, db = (torch.empty(*s, device=cuda) for s in ((N, G, 2), (N, P, C), (N, P, C), (C,), (C,)))
    pkg.ops.group_norm_act(*dev, out, G, EPS, act, stat=stat)
    pkg.ops.group_norm_act_bwd(*dev, stat, dy.to(cuda), dx, dw, db, G, act)

    def loss(x, w, b):
        v = x.view(N, P, G, C // G)
        m = v.mean((1, 3), keepdim=True)
        xh = ((v - m) / torch.sqrt(((v - m) ** 2).mean((1, 3), keepdim=True) + EPS)).reshape(N, P, C)
        return (_act(xh * w + b, act)[0] * dy.double()).sum()

    _, tol = reference(x, w, b, dy, G, act, torch.float32)
    at = dict(x=x.double(), w=w.double(), b=b.double())
    for n, grad in (("x", dx), ("w", dw), ("b", db)):
        d = torch.randn(at[n].shape, generator=g, dtype=torch.float64)
        hi, lo = (loss(**{m: at[m] + (s * 1e-4 * d if m == n else 0.0) for m in at}) for s in (1.0, -1.0))
        prod = grad.cpu().double() * d
        bound = float((tol["d" + n] * d.abs()).sum()) + 1e-6 * float(prod.abs().sum())
        assert abs(float(prod.sum()) - float(hi - lo) / 2e-4) <= bound, n


def test_captured_and_replayed(pkg, cuda):
    x, dy = torch.randn(2, 3000, 64, device=cuda).bfloat16(), torch.randn(2, 3000, 64, device=cuda).bfloat16()
    w, b = torch.randn(64, device=cuda), torch.randn(64, device=cuda)
    res = [torch.empty_like(x), torch.empty_like(x), torch.empty(64, device=cuda), torch.empty(64, device=cuda), torch.empty(2, 4, 2, device=cuda)]

    def both():
        pkg.ops.group_norm_act(x, w, b, res[0], 4, EPS, 4, stat=res[4])
        pkg.ops.group_norm_act_bwd(x, w, b, res[4], dy, *res[1:4], 4, 4)

    both()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        both()
    for _ in range(3):
        x.normal_()
        both()
        want = [t.clone() for t in res]
        for t in res:
            t.fill_(math.nan)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(res, want))


def test_refusals(pkg, cuda):
    o = pkg.ops
    x, w = torch.zeros(2, 4, 12, device=cuda), torch.ones(12, device=cuda)
    out, stat = torch.empty_like(x), torch.empty(2, 3, 2, device=cuda)
    for match, call in [
        ("groups", lambda: o.group_norm_act(x, w, w, out, 5, EPS)),
        ("activation", lambda: o.group_norm_act(x, w, w, out, 3, EPS, 9)),
        ("w must", lambda: o.group_norm_act(x, w[:6], w, out, 3, EPS)),
        ("b must", lambda: o.group_norm_act(x, w, w.bfloat16(), out, 3, EPS)),
        ("out must", lambda: o.group_norm_act(x, w, w, out[:, :2], 3, EPS)),
        ("x must", lambda: o.group_norm_act(x.half(), w, w, out, 3, EPS)),
        ("x must", lambda: o.group_norm_act(x[:, :0], w, w, out[:, :0], 3, EPS)),
        ("contiguous channels", lambda: o.group_norm_act(x.transpose(1, 2), w[:4], w[:4], out.transpose(1, 2), 2, EPS)),
        ("stat", lambda: o.group_norm_act(x, w, w, out, 3, EPS, stat=stat[:1])),
        ("share memory", lambda: o.group_norm_act(x, w, w, torch.empty(1, 4, 12, device=cuda).expand(2, 4, 12), 3, EPS)),
        ("GPU", lambda: o.group_norm_act(x.cpu(), w, w, out, 3, EPS)),
        ("x's dtype", lambda: o.group_norm_act_bwd(x, w, w, stat, x, out.bfloat16(), w.clone(), w.clone(), 3)),
        ("another operand", lambda: o.group_norm_act_bwd(x, w, w, stat, x, out, w, w.clone(), 3)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
