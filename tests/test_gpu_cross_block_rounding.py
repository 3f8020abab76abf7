"""The bf16 cross-attention block against the definition with exactly the roundings to bf16 that the chain makes, and no others."""
import pytest
import torch

from tests.test_gpu_cross_block import EPS, Head

OUTPUTS = ("out", "dk", "dv", "dtable", "dx", "dw", "db")


def rounded(h, round_to=torch.bfloat16, arith=torch.float64, without=()):
    """the chain of ``Head.run``, rounded where the kernels round: every stored map, the exponentials and dS in front of a matrix instruction (dS of dQ goes there in two
    terms, up to 256 attended keys: not rounded), and nothing else; D of a rounded O is mended by the row sum of dS'.  ``without``: mistakes to plant"""
    f = lambda x: x.detach().cpu().to(arith)
    r = lambda x: x.to(round_to).to(arith)
    N, P, C, H, hd, G, groups = h.N, h.P, h.C, h.H, h.hd, h.G, h.groups
    w, b = f(h.w), f(h.b)

    def normed(x):
        v = f(x).view(N, P, groups, C // groups)
        m = v.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt(((v - m) ** 2).mean((1, 3), keepdim=True) + EPS)
        xh = ((v - m) * rstd).reshape(N, P, C)
        z = xh * w + b
        return r(z * torch.sigmoid(z)), xh, z, rstd

    heads = lambda x: x.view(N, P, H, hd).transpose(1, 2)
    back = lambda x: x.transpose(1, 2)
    (nq, xh, z, rstd), (ns, _, _, _) = normed(h.xq), normed(h.xs)
    q, k, v = (heads(r(n @ f(m).t())) for n, m in ((nq, h.wq), (ns, h.wk), (ns, h.wv)))
    i = torch.arange(P)
    dy, dx = (i // G)[None] - (i // G)[:, None] + G - 1, (i % G)[None] - (i % G)[:, None] + G - 1
    iy, ix = h.by.cpu().long()[dy], h.bx.cpu().long()[dx]
    scale = hd ** -0.5
    on = h.mask.cpu()[:, None, None]
    S = (q @ k.transpose(2, 3) * scale + f(h.table)[iy, ix].permute(2, 0, 1)).masked_fill(~on, -1e30)
    E = torch.exp(S - S.amax(-1, keepdim=True)) * on
    l = E.sum(-1, keepdim=True).clamp_min(1e-30)
    pr = E / l
    out = r(r(E) @ v / l)
    dO = heads(f(h.dout))
    dP, D = dO @ v.transpose(2, 3), (dO * out).sum(-1, keepdim=True)
    dS1 = pr * (dP - D)
    e = dS1.sum(-1, keepdim=True)
    dq = r((dS1 @ k - (0 if "dq mending" in without else e) * (r(pr) @ k)) * scale)
    dS = dS1 if "D mending" in without else pr * (dP - D - e)
    dk, dv = r(r(dS).transpose(2, 3) @ q * scale), r(r(pr).transpose(2, 3) @ dO)
    if "a key" in without:
        dk[1, :, 3] = 0
    dbias = dS.sum(0)
    dtable = torch.zeros(64, H, dtype=arith).index_add_(0, (iy * 8 + ix).reshape(-1), dbias.reshape(H, -1).t().contiguous()).view(8, 8, H)
    dn = r(back(dq).reshape(N, P, H * hd) @ f(h.wq_t).t())
    s = torch.sigmoid(z)
    dz = dn * s * (1 + z * (1 - s))
    gh, xg = (dz * w).view(N, P, groups, -1), xh.view(N, P, groups, -1)
    m1, m2 = gh.mean((1, 3), keepdim=True), (gh * xg).mean((1, 3), keepdim=True)
    dxq = r((rstd * (gh - (0 if "norm mean" in without else m1) - xg * m2)).reshape(N, P, C))
    return dict(out=back(out), dk=back(dk), dv=back(dv), dtable=dtable, dx=dxq, dw=(dz * xh).sum((0, 1)), db=dz.sum((0, 1)))


def shares(h, got):
    """for every output, how far it is from the rounded chain, as a share of what the roundings themselves make"""
    want, exact = rounded(h), rounded(h, round_to=torch.float64)
    return {n: float((got[n].cpu().double() - want[n]).norm() / (want[n] - exact[n]).norm()) for n in OUTPUTS}


# A value whose f32 sum of n terms is off by up to n 2^-24 of its magnitudes M falls on the other side of a rounding border with a probability of at most 2 n 2^-24 M / (2^-8 |x|), about
# n 2^-15 M / |x|: with the 64 to 200 terms of a stage and M up to eight times |x| that is under 5 %, and errors of that share of the values make up sqrt(0.05) = 0.22 of the norm of all.
# The stages behind hand both on alike.  Half as much again leaves room for the spread of counts.
SHARE = 0.35


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 5])
@pytest.mark.parametrize("shape", [dict(), dict(N=4, G=9, C=128, H=4, hd=32, groups=4)])
def test_bf16_chain_makes_no_roundings_but_its_own(pkg, cuda, seed, shape):
    h = Head(pkg, cuda, torch.bfloat16, seed=seed, **shape)
    got = h.run()
    for n, share in shares(h, got).items():
        assert share <= SHARE, f"{n}: {share:.2f} of the roundings"


@pytest.mark.parametrize("seed", [0, 5])
@pytest.mark.parametrize("shape", [dict(), dict(N=4, G=9, C=128, H=4, hd=32, groups=4)])
def test_the_bound_tells_a_lost_term(pkg, seed, shape):
    """on the CPU: the same chain in f32 is inside the bound, one that lacks a term of the size of the roundings is not"""
    h = Head(pkg, "cpu", torch.bfloat16, seed=seed, **shape)
    assert max(shares(h, rounded(h, arith=torch.float32)).values()) <= SHARE
    for mistake, output in (("dq mending", "dx"), ("D mending", "dtable"), ("a key", "dk"), ("norm mean", "dx")):
        assert shares(h, rounded(h, without=(mistake,)))[output] > SHARE, mistake
