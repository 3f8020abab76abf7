"""The operators of a trained cross-attention block run together, as a head on patch features uses them: norm of the query and support maps, projections, position
bias, attention over the support's foreground, and the whole way back to the maps, the projections' outputs and the bias table."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-5


class Head:
    """N query maps on a G x G grid over supports on the same grid, H heads of hd"""

    def __init__(self, pkg, dev, dtype, seed=0, N=3, G=7, C=64, H=4, hd=16, groups=8):
        self.pkg, self.N, self.G, self.P, self.C, self.H, self.hd, self.groups, self.dtype = pkg, N, G, G * G, C, H, hd, groups, dtype
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).to(dev)
        self.xq, self.xs = rnd(N, self.P, C).to(dtype), rnd(N, self.P, C).to(dtype)
        self.w, self.b = 1 + rnd(C, k=0.2), rnd(C, k=0.2)
        self.wq, self.wk, self.wv = (rnd(H * hd, C, k=C ** -0.5).to(dtype) for _ in range(3))
        self.table = rnd(8, 8, H, k=0.5)
        self.by = pkg.ops.bucket_map(G, G, 8, 6).to(dev)
        self.bx = self.by.clone()
        self.mask = (torch.rand(N, self.P, generator=g) < 0.4).to(dev)
        self.mask[0] = False                                        # a support without foreground
        self.mask[1, 3] = True
        self.dout = rnd(N, self.P, H, hd).to(dtype)
        e = lambda *s, d=dtype: torch.empty(*s, device=dev, dtype=d)
        self.buf = dict(nq=e(N, self.P, C), ns=e(N, self.P, C), sq=e(N, groups, 2, d=torch.float32), q=e(N * self.P, H * hd), k=e(N * self.P, H * hd),
                        v=e(N * self.P, H * hd), bias=e(H, self.P, self.P, d=torch.float32), out=e(N, self.P, H, hd), stat=e(N, H, self.P, 2, d=torch.float32),
                        dq=e(N, self.P, H, hd), dk=e(N, self.P, H, hd), dv=e(N, self.P, H, hd), dbias=e(H, self.P, self.P, d=torch.float32),
                        dtable=e(8, 8, H, d=torch.float32), dn=e(N * self.P, C), dx=e(N, self.P, C), dw=e(C, d=torch.float32), db=e(C, d=torch.float32))
        self.wq_t = self.wq.t().contiguous()

    def run(self):
        o, act, t = self.pkg.ops, self.pkg.hip.ACT_SILU, self.buf
        N, P, C, H, hd = self.N, self.P, self.C, self.H, self.hd
        grids = dict(q_grid=(self.G, self.G), k_grid=(self.G, self.G))
        o.group_norm_act(self.xq, self.w, self.b, t["nq"], self.groups, EPS, act, stat=t["sq"])
        o.group_norm_act(self.xs, self.w, self.b, t["ns"], self.groups, EPS, act)
        o.linear(t["nq"].view(N * P, C), self.wq, t["q"])
        o.linear(t["ns"].view(N * P, C), self.wk, t["k"])
        o.linear(t["ns"].view(N * P, C), self.wv, t["v"])
        q, k, v = (t[n].view(N, P, H, hd) for n in "qkv")
        o.bucket_bias(self.table, self.by, self.bx, t["bias"], **grids)
        o.cross_attn(q, k, v, t["out"], stat=t["stat"], mask=self.mask, bias=t["bias"])
        o.cross_attn_bwd(q, k, v, t["out"], t["stat"], self.dout, t["dq"], t["dk"], t["dv"], dbias=t["dbias"], mask=self.mask, bias=t["bias"])
        o.bucket_bias_bwd(t["dbias"], self.by, self.bx, t["dtable"], **grids)
        o.linear(t["dq"].view(N * P, H * hd), self.wq_t, t["dn"])
        o.group_norm_act_bwd(self.xq, self.w, self.b, t["sq"], t["dn"].view(N, P, C), t["dx"], t["dw"], t["db"], self.groups, act)
        return {n: t[n] for n in ("out", "dk", "dv", "dtable", "dx", "dw", "db")}

    def reference(self):
        """the same in 64 bits with torch's own differentiation"""
        f = lambda x: x.detach().cpu().double()
        N, P, C, H, hd, G = self.N, self.P, self.C, self.H, self.hd, self.G
        xq, w, b, table = (f(x).requires_grad_() for x in (self.xq, self.w, self.b, self.table))

        def norm(x, w, b):
            v = x.view(N, P, self.groups, C // self.groups)
            m = v.mean((1, 3), keepdim=True)
            z = ((v - m) / torch.sqrt(((v - m) ** 2).mean((1, 3), keepdim=True) + EPS)).reshape(N, P, C) * w + b
            return z * torch.sigmoid(z)

        q = norm(xq, w, b) @ f(self.wq).t()
        ns = norm(f(self.xs), w.detach(), b.detach())
        k, v = ((ns @ f(m).t()).requires_grad_() for m in (self.wk, self.wv))
        i = torch.arange(P)
        dy, dx = (i // G)[None] - (i // G)[:, None] + G - 1, (i % G)[None] - (i % G)[:, None] + G - 1
        bias = table[self.by.cpu().long()[dy], self.bx.cpu().long()[dx]].permute(2, 0, 1)
        heads = lambda x: x.view(N, P, H, hd).transpose(1, 2)
        S = heads(q) @ heads(k).transpose(2, 3) * hd ** -0.5 + bias
        on = self.mask.cpu()[:, None, None]
        Pr = torch.softmax(S.masked_fill(~on, -1e300), -1) * on.any(-1, keepdim=True)
        out = (Pr @ heads(v)).transpose(1, 2)
        (out * f(self.dout)).sum().backward()
        # cross_attn is given its gradient of q alone (the key and value projections end the chain): dx through the queries
        return dict(out=out.detach(), dk=k.grad.view(N, P, H, hd), dv=v.grad.view(N, P, H, hd), dtable=table.grad, dx=xq.grad, dw=w.grad, db=b.grad), float(S.detach().abs().max())


def test_forward_and_gradients(pkg, cuda):
    """f32 throughout: every result within the roundings of the chain, norm against norm.  A stage that contracts n terms adds at most n 2^-24 of its
    magnitudes: the group norms 8 P, the projections C and H hd, the attention's products hd and P each way; an error of a score moves its probability
    by as much, which the largest score bounds as a factor; two for each of the stages being passed forward and back."""
    h = Head(pkg, cuda, torch.float32)
    got = h.run()
    want, smax = h.reference()
    terms = 8 * h.P + 2 * h.C + 2 * h.H * h.hd + 4 * (h.hd + h.P)
    bound = 2 * terms * (1 + smax) * 2.0 ** -24
    for n, t in got.items():
        err = float((t.cpu().double() - want[n]).norm() / want[n].norm())
        assert err <= bound, f"{n}: {err:.2e} of {bound:.2e}"
    assert bool((got["out"][0] == 0).all()) and bool((got["dk"][0] == 0).all()) and bool((got["dv"][0] == 0).all()) and bool((got["dx"][0] == 0).all())


def test_bf16_follows_f32(pkg, cuda):
    """the same head in bf16 against the f32 one on the same (bf16) values: seven roundings to bf16 lie between an input and the last gradient
    (norm, projection, P, out, dS, dq, dn), each half a step of 2^-8, passed on through the largest score as above"""
    h = Head(pkg, cuda, torch.bfloat16)
    f = Head(pkg, cuda, torch.float32)
    for n in ("xq", "xs", "wq", "wk", "wv", "wq_t", "dout"):
        setattr(f, n, getattr(h, n).float())
    want, smax = f.reference()
    for n, t in h.run().items():
        err = float((t.cpu().double() - want[n]).norm() / want[n].norm())
        assert err <= 7 * 2.0 ** -8 * (1 + smax), f"{n}: {err:.2e}"


def test_captured_and_replayed(pkg, cuda):
    h = Head(pkg, cuda, torch.bfloat16, seed=1)
    h.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = h.run()
    for i in range(3):
        h.xq.normal_()
        want = {n: t.clone() for n, t in h.run().items()}
        for t in res.values():
            t.fill_(math.nan)
        g.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(res[n], want[n]), n


@pytest.mark.parametrize("hd,bias", [(64, False), (64, True), (80, False)])
def test_same_bits_with_the_chip_full(pkg, cuda, hd, bias):
    """every CU busy, tiles handed over as fast as they come: the same bits every time (a tile that is read before all of its fills have landed shows here)"""
    B, L, H = 2, 1500, 8
    q, k, v, d = (torch.randn(B, L, H, hd, device=cuda).bfloat16() for _ in range(4))
    bi = torch.randn(H, L, L, device=cuda) if bias else None
    first = None
    for _ in range(4):
        out, stat = torch.empty_like(q), torch.empty(B, H, L, 2, device=cuda)
        res = [torch.empty_like(q) for _ in range(3)] + ([torch.empty_like(bi)] if bias else [])
        pkg.ops.cross_attn(q, k, v, out, stat=stat, bias=bi)
        pkg.ops.cross_attn_bwd(q, k, v, out, stat, d, *res[:3], bias=bi, dbias=res[3] if bias else None)
        res += [out, stat]
        if first is None:
            first = res
        assert all(torch.equal(a, b) for a, b in zip(first, res))


def test_known_layouts_with_other_addresses(pkg, cuda):
    """calls of one layout share what was checked before: other tensors, other results; a bad address is still refused"""
    q, k = torch.randn(1, 5, 2, 64, device=cuda), torch.randn(1, 33, 2, 64, device=cuda)
    o1, o2 = torch.empty_like(q), torch.empty_like(q)
    pkg.ops.cross_attn(q, k, k, o1)
    pkg.ops.cross_attn(q * 2, k, k + 1, o2)
    S = torch.einsum("blhd,bmhd->bhlm", q.double() * 2, k.double()) / 8
    want = torch.einsum("bhlm,bmhd->blhd", S.softmax(-1), k.double() + 1)
    bound = 2 * (64 + 33 + 16) * 2.0 ** -24 * (1 + S.abs().max()) * (k.abs().max() + 1)           # contractions of hd and Lk terms, errors of the scores
    assert float((o2.double() - want).abs().max()) <= float(bound) and not torch.equal(o1, o2)
    buf = torch.zeros(5 * 2 * 64 + 1, device=cuda)
    with pytest.raises(ValueError, match="aligned"):
        pkg.ops.cross_attn(buf[1:].view(1, 5, 2, 64), k, k, o1)
    with pytest.raises(ValueError, match="another operand"):
        pkg.ops.cross_attn(q, k, k, q)
    with pytest.raises(ValueError, match="GPU"):
        pkg.ops.cross_attn(q.cpu(), k, k, o1)
