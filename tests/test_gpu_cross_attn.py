"""Attention between two token sets, forward and backward, against the definition in 64 bits with bounds derived from the
roundings that the kernels make."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24                       # half a step of f32


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _randn(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, dtype=torch.float32) * scale


def make(cuda, dtype, B, Lq, Lk, H, Hkv, hd, *, seed=0, keys="all", bias=None, layout="plain"):
    """Operands of one case.  keys: all, len, mask, both; bias: None, "rand", "inf", "low"."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = _randn(g, B, Lq, H, hd, scale=1.3), _randn(g, B, Lk, Hkv, hd, scale=1.3), _randn(g, B, Lk, Hkv, hd)
    dout = _randn(g, B, Lq, H, hd)
    c = dict(B=B, Lq=Lq, Lk=Lk, H=H, Hkv=Hkv, hd=hd, dtype=dtype, scale=hd ** -0.5)
    att = torch.ones(B, Lk, dtype=torch.bool)
    c["kv_len"] = c["mask"] = None
    if keys in ("len", "both"):
        n = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32)
        n[0] = Lk
        if B > 1:
            n[-1] = 0
        att &= torch.arange(Lk)[None] < n[:, None]
        c["kv_len"] = n.to(cuda)
    if keys in ("mask", "both"):
        m = torch.rand(B, Lk, generator=g) < 0.4
        m[0, Lk // 2] = True
        if B > 2:
            m[1] = False
        att &= m
        c["mask"] = m.to(cuda)
    c["att"] = att
    b = None
    if bias is not None:
        b = _randn(g, H, Lq, Lk)
        if bias == "inf":
            b[torch.rand(H, Lq, Lk, generator=g) < 0.3] = -math.inf
            b[0, Lq // 2] = -math.inf                                       # a row that nothing is left of
        if bias == "low":
            b[torch.rand(H, Lq, Lk, generator=g) < 0.3] = torch.finfo(torch.float32).min
            b[H - 1, Lq // 2] = torch.finfo(torch.float32).min              # a row of nothing but the lowest value: even weights
    c["bias"] = None if b is None else b.to(cuda)
    # what stands in a key that is not attended must not matter
    k[~att] = math.nan
    v[~att] = math.inf
    c["q"], c["k"], c["v"], c["dout"] = (_lay(t.to(cuda).to(dtype), layout, i) for i, t in enumerate((q, k, v, dout)))
    return c


def _lay(t, layout, i):
    if layout == "plain":
        return t.contiguous()
    if layout == "heads_first":                                             # [B, H, L, hd] in memory
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "wide":                                                    # rows and heads inside a wider buffer, at an offset
        B, L, H, hd = t.shape
        buf = torch.full((B + 1, L + 3, 2 * H * hd + 32), math.nan, dtype=t.dtype, device=t.device)
        view = buf[1:, 2:-1, 16:16 + 2 * H * hd].view(B, L, H, 2 * hd)[..., hd:] if hd % 8 == 0 else None
        assert view is not None
        view.copy_(t)
        return view
    raise AssertionError(layout)


def empty_like(t, layout):
    x = _lay(torch.zeros_like(t, memory_format=torch.contiguous_format), layout, 0)
    x.fill_(math.nan)
    return x


def reference(c):
    """out, stat, gradients and, beside each, how far the kernels may be off.

    A relative error r of a probability comes from its exponent (f32 products over hd elements, the scale, the bias, the subtraction of the
    maximum) and from the exponential and the reciprocal; u is the rounding of P and dS in front of the matrix instruction (0 for f32, which it
    takes as they are); sums of n terms in f32 add at most n U32 of the sum of the magnitudes."""
    B, Lq, Lk, H, Hkv, hd, dtype = (c[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "hd", "dtype"))
    u, ro = (_half(dtype), _half(dtype)) if dtype == torch.bfloat16 else (0.0, U32)
    dev = c["q"].device
    f = dict(dtype=torch.float64, device=dev)
    res = {n: torch.zeros(s, **f) for n, s in (("out", (B, Lq, H, hd)), ("dq", (B, Lq, H, hd)), ("dk", (B, Lk, Hkv, hd)), ("dv", (B, Lk, Hkv, hd)),
                                               ("dbias", (H, Lq, Lk)))}
    tol = {n: torch.zeros_like(t) for n, t in res.items()}
    res["sum"] = torch.zeros(B, H, Lq, **f)
    res["max"] = torch.full((B, H, Lq), -math.inf, **f)
    for b in range(B):
        keys = torch.nonzero(c["att"][b]).flatten().to(dev)
        n = keys.numel()
        if n == 0:
            continue
        for h in range(H):
            j = h // (H // Hkv)
            Q, K, V, dO = (x.double() for x in (c["q"][b, :, h], c["k"][b, keys, j], c["v"][b, keys, j], c["dout"][b, :, h]))
            S = Q @ K.t() * c["scale"]
            mag = Q.abs() @ K.abs().t() * c["scale"]
            if c["bias"] is not None:
                bb = c["bias"][h][:, keys].double()
                S = S + bb
                S = torch.where(bb <= torch.finfo(torch.float32).min, bb, S)        # (the lowest float swallows the product in f32)
                mag = mag + torch.where(torch.isfinite(bb) & (bb > -1e30), bb.abs(), torch.zeros_like(bb))
            m = S.amax(1, keepdim=True)
            ok = m > -math.inf
            E = torch.where(ok, torch.exp(S - torch.where(ok, m, torch.zeros_like(m))), torch.zeros_like(S))
            l = E.sum(1, keepdim=True)
            P = torch.where(ok, E / l.clamp_min(1e-300), torch.zeros_like(S))
            res["sum"][b, h], res["max"][b, h] = l[:, 0], m[:, 0]
            O = P @ V
            res["out"][b, :, h] = O
            # exponent: hd products and sums, then scale, bias, subtraction and log2(e): each at most U32 of what it works on
            r = (hd + 8) * U32 * 2 * mag.amax(1, keepdim=True) + 16 * U32
            r = 2 * r + (n + 8) * U32
            A = P @ V.abs()
            tO = A * (u + r + (n + 8) * U32) + ro * O.abs() + 1e-30
            tol["out"][b, :, h] = tO
            dP = dO @ V.t()
            D = (dO * O).sum(1, keepdim=True)
            dS = P * (dP - D)
            mdP = dO.abs() @ V.abs().t()
            e0 = (dO.abs() * tO).sum(1, keepdim=True)                               # D' = dO . (rounded O) against D
            t1 = P * (dP - D).abs() * (r + 4 * U32) + P * mdP * (hd + 2) * U32      # of dS, but for D
            tE = (t1 + P * ((dP - D).abs() + e0) * (r + n * U32)).sum(1, keepdim=True)
            # bf16: D = D' + sum dS' (the probabilities add up to 1 within r); f32: D = D'
            tD = tE + (D.abs() + e0) * (r + 2 * U32) if u else e0 + hd * U32 * (dO * O).abs().sum(1, keepdim=True)
            tS = t1 + P * tD
            tSr = tS + u * dS.abs() * 1.01                                          # rounded for the matrix instruction
            PK = P @ K.abs()
            res["dq"][b, :, h] = dS @ K * c["scale"]
            if u:       # sum dS' K - e sum P K: dS' and P rounded, e = D' - D of the size e0
                tq = (t1 + u * (dS.abs() + P * e0) * 1.01 + n * U32 * (dS.abs() + P * e0)) @ K.abs() + (e0 * (u + r + n * U32) + tD) * PK
            else:
                tq = (tS + n * U32 * dS.abs()) @ K.abs()
            tol["dq"][b, :, h] = c["scale"] * tq + ro * res["dq"][b, :, h].abs() + 1e-30
            res["dk"][b, keys, j] += dS.t() @ Q * c["scale"]
            tol["dk"][b, keys, j] += c["scale"] * ((tSr + H * Lq * U32 * dS.abs()).t() @ Q.abs())
            res["dv"][b, keys, j] += P.t() @ dO
            tol["dv"][b, keys, j] += (P * (u + r + H * Lq * U32)).t() @ dO.abs()
            res["dbias"][h, :, keys] += dS
            tol["dbias"][h, :, keys] += tS + B * U32 * dS.abs() + 1e-30
    tol["dk"] += ro * res["dk"].abs() + 1e-30
    tol["dv"] += ro * res["dv"].abs() + 1e-30
    return res, tol


def run(pkg, c, layout="plain", backward=True):
    o = pkg.ops
    out = empty_like(c["q"], layout)
    stat = torch.full((c["B"], c["H"], c["Lq"], 2), math.nan, device=c["q"].device)
    kw = dict(scale=c["scale"], kv_len=c["kv_len"], mask=c["mask"], bias=c["bias"])
    o.cross_attn(c["q"], c["k"], c["v"], out, stat=stat, **kw)
    got = dict(out=out, stat=stat)
    if backward:
        for n, s in (("dq", "q"), ("dk", "k"), ("dv", "v")):
            got[n] = empty_like(c[s], layout)
        got["dbias"] = None if c["bias"] is None else torch.full_like(c["bias"], math.nan)
        o.cross_attn_bwd(c["q"], c["k"], c["v"], out, stat, c["dout"], got["dq"], got["dk"], got["dv"], dbias=got["dbias"], **kw)
    return got


def check(pkg, c, layout="plain", backward=True):
    got = run(pkg, c, layout, backward)
    res, tol = reference(c)
    for n in ("out", "dq", "dk", "dv", "dbias"):
        if got.get(n) is None:
            continue
        err = (got[n].double() - res[n]).abs()
        assert bool(torch.isfinite(got[n]).all()), f"{n}: not finite"
        worst = float((err / tol[n].clamp_min(1e-300)).max())
        assert worst <= 1.0, f"{n}: {worst:.2f} of the bound, error {float(err.max()):.3e}"
    empty = res["sum"] == 0
    assert torch.equal(got["stat"][..., 1] == 0, empty)
    assert bool((got["stat"][..., 0][empty] == -math.inf).all())
    assert bool((got["out"].transpose(1, 2)[empty] == 0).all())
    return got


DT = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 65), (7, 200), (31, 64), (33, 1), (128, 63), (129, 129), (300, 257)])
def test_lengths(pkg, cuda, dtype, Lq, Lk):
    check(pkg, make(cuda, dtype, 2, Lq, Lk, 3, 3, 64, seed=Lq * 1000 + Lk))


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, h) for h in (8, 16, 24, 32, 40, 72, 80, 96, 104, 128)] + [(torch.float32, h) for h in (4, 12, 32, 68, 80, 128)])
def test_head_dims(pkg, cuda, dtype, hd):
    check(pkg, make(cuda, dtype, 2, 70, 133, 2, 2, hd, seed=hd))
    check(pkg, make(cuda, dtype, 2, 5, 133, 2, 2, hd, seed=hd + 1, keys="mask", bias="rand"))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,Hkv,Lq", [(8, 2, 1), (6, 1, 3), (8, 4, 50), (16, 1, 20)])
def test_shared_key_heads(pkg, cuda, dtype, H, Hkv, Lq):
    check(pkg, make(cuda, dtype, 2, Lq, 150, H, Hkv, 64, seed=H + Lq))
    check(pkg, make(cuda, dtype, 3, Lq, 150, H, Hkv, 48, seed=H + Lq + 1, keys="both", bias="inf"))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("keys", ["len", "mask", "both"])
@pytest.mark.parametrize("Lq", [4, 140])
def test_masks(pkg, cuda, dtype, keys, Lq):
    """NaN and infinities at keys that are not attended, entries without any key, ragged lists."""
    check(pkg, make(cuda, dtype, 4, Lq, 300, 2, 2, 64, seed=5, keys=keys))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq,Lk,how,bias", [(9, 1, "all", "rand"), (200, 1, "all", None), (40, 70, "len", "rand"), (150, 300, "mask", None), (3, 3000, "mask", "rand")])
def test_one_attended_key_has_no_gradient_of_scores(pkg, cuda, dtype, Lq, Lk, how, bias):
    """the softmax over one key is 1: q, k and the bias have a gradient of exactly zero"""
    c = make(cuda, dtype, 2, Lq, Lk, 4, 2, 64, seed=13, bias=bias)
    att = torch.zeros(2, Lk, dtype=torch.bool)
    att[:, 0 if how == "len" else Lk // 2] = True
    c["att"] = att
    if how == "len":
        c["kv_len"] = torch.ones(2, dtype=torch.int32, device=cuda)
    if how == "mask":
        c["mask"] = att.to(cuda)
    got = run(pkg, c)
    for n in ("dq", "dk", "dbias"):
        assert got[n] is None or bool((got[n] == 0).all()), n
    res, tol = reference(c)
    assert bool(((got["dv"].double() - res["dv"]).abs() <= tol["dv"]).all()) and bool(((got["out"].double() - res["out"]).abs() <= tol["out"]).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bias", ["rand", "inf", "low"])
@pytest.mark.parametrize("Lq,Lk,keys", [(6, 90, "all"), (150, 131, "mask"), (40, 700, "len")])
def test_bias(pkg, cuda, dtype, bias, Lq, Lk, keys):
    check(pkg, make(cuda, dtype, 3, Lq, Lk, 2, 2, 64, seed=11, keys=keys, bias=bias))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("layout", ["heads_first", "wide"])
@pytest.mark.parametrize("Lq", [3, 130])
def test_layouts(pkg, cuda, dtype, layout, Lq):
    check(pkg, make(cuda, dtype, 2, Lq, 190, 4, 2, 40, seed=21, layout=layout, keys="mask"), layout)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq,Lk,H,Hkv,keys,bias", [(1, 5000, 4, 1, "len", None), (20, 4097, 2, 2, "mask", None), (60, 3000, 2, 2, "all", "rand"), (2500, 40, 1, 1, "mask", None),
                                                   (900, 77, 4, 2, "all", "inf")])
def test_long_axes_are_split(pkg, cuda, dtype, Lq, Lk, H, Hkv, keys, bias):
    """few rows against a long other axis: the work is cut along it and joined"""
    check(pkg, make(cuda, dtype, 2, Lq, Lk, H, Hkv, 64, seed=31, keys=keys, bias=bias))


def test_packed_projections(pkg, cuda):
    """q, k, v as views of one buffer, gradients into views of another"""
    B, L, H, hd = 2, 150, 4, 64
    c = make(cuda, torch.bfloat16, B, L, L, H, H, hd, seed=41)
    buf = torch.stack([c["q"], c["k"], c["v"]], 2).reshape(B, L, 3 * H * hd)
    grad = torch.full_like(buf, math.nan)
    q, k, v = buf.view(B, L, 3, H, hd).unbind(2)
    dq, dk, dv = grad.view(B, L, 3, H, hd).unbind(2)
    plain = run(pkg, c)
    out, stat = torch.empty_like(c["q"]), torch.empty(B, H, L, 2, device=cuda)
    pkg.ops.cross_attn(q, k, v, out, stat=stat, scale=c["scale"])
    pkg.ops.cross_attn_bwd(q, k, v, out, stat, c["dout"], dq, dk, dv, scale=c["scale"])
    for got, n in ((out, "out"), (dq, "dq"), (dk, "dk"), (dv, "dv")):
        assert torch.equal(got, plain[n])


def test_broadcast_keys(pkg, cuda):
    """one support set for a whole batch: expanded operands are read, their gradients come for each entry"""
    c = make(cuda, torch.bfloat16, 1, 40, 100, 2, 2, 64, seed=42)
    B = 3
    q = torch.cat([c["q"] * s for s in (1.0, 0.5, -1.0)])
    big = dict(c, B=B, q=q, k=c["k"].expand(B, -1, -1, -1), v=c["v"].expand(B, -1, -1, -1), dout=c["dout"].expand(B, -1, -1, -1).contiguous(),
               att=c["att"].expand(B, -1))
    check(pkg, big)
    with pytest.raises(ValueError, match="share memory"):
        pkg.ops.cross_attn(q, big["k"], big["v"], torch.empty_like(c["q"]).expand(B, -1, -1, -1))


@pytest.mark.parametrize("dtype", DT)
def test_gradients_against_differences(pkg, cuda, dtype):
    """<gradient, direction> against central differences of the definition in 64 bits: step 1e-4 of smooth functions of order one, so the differences are
    off by about 1e-8 of the magnitudes; the rest is the kernels' own bound"""
    c = make(cuda, dtype, 2, 17, 45, 4, 2, 32, seed=51, keys="len", bias="rand")
    got = run(pkg, c)
    _, tol = reference(c)
    g = torch.Generator().manual_seed(52)
    att = c["att"].to(cuda)

    def loss(q, k, v, bias):
        k, v = (x.repeat_interleave(c["H"] // c["Hkv"], 2) for x in (k, v))
        S = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1).contiguous()) * c["scale"] + bias
        S = S.masked_fill(~att[:, None, None], -1e300)
        P = torch.softmax(S, -1) * att[:, None, None].any(-1, keepdim=True)
        return (torch.matmul(P, v.transpose(1, 2).contiguous()).transpose(1, 2) * c["dout"].double()).sum()

    at = {n: torch.nan_to_num(c[n].double(), 0.0, 0.0, 0.0) for n in ("q", "k", "v")}
    at["v"][~att], at["k"][~att] = 0.0, 0.0
    at["bias"] = c["bias"].double()
    for n in at:
        d = torch.randn(at[n].shape, generator=g, dtype=torch.float64).to(cuda)
        h = 1e-4
        hi, lo = (loss(**{m: at[m] + (s * h * d if m == n else 0.0) for m in at}) for s in (1.0, -1.0))
        diff = float((hi - lo) / (2 * h))
        grad = got["d" + n].double()
        bound = float((tol["d" + n] * d.abs()).sum()) + 1e-6 * float((grad * d).abs().sum())
        assert abs(float((grad * d).sum()) - diff) <= bound, n


@pytest.mark.parametrize("dtype", DT)
def test_same_bits_every_call(pkg, cuda, dtype):
    c = make(cuda, dtype, 3, 200, 400, 4, 2, 64, seed=61, keys="both", bias="rand")
    a, b = run(pkg, c), run(pkg, c)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_large_scores_do_not_overflow(pkg, cuda):
    for dtype in DT:
        c = make(cuda, dtype, 1, 33, 130, 2, 2, 64, seed=62)
        c["q"] = c["q"] * 40
        got = run(pkg, c)
        assert all(bool(torch.isfinite(t).all()) for t in got.values() if t is not None)
        check(pkg, c, backward=False)


def test_nan_query_row_stays_alone(pkg, cuda):
    c = make(cuda, torch.bfloat16, 1, 100, 90, 2, 2, 64, seed=63)
    want = run(pkg, c, backward=False)["out"].clone()
    c["q"][0, 37, 1] = math.nan
    got = run(pkg, c, backward=False)["out"]
    assert bool(torch.isnan(got[0, 37, 1]).all())
    got[0, 37, 1] = want[0, 37, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("Lq", [1, 130])
def test_offsets_beyond_32_bits(pkg, cuda, Lq):
    """keys of a long cache: the second entry, and the last tokens, lie more than 2^32 bytes behind the first"""
    B, Lk, H, hd = 2, 90, 2, 64
    c = make(cuda, torch.bfloat16, B, Lq, Lk, H, H, hd, seed=71)
    tok = 1 << 25                                                           # elements from token to token: 90 of them are 6 GB
    buf = torch.empty((Lk - 1) * tok + 4 * H * hd, dtype=torch.bfloat16, device=cuda)
    k = buf.as_strided((B, Lk, H, hd), (2 * H * hd, tok, hd, 1))
    k.copy_(c["k"])
    want = run(pkg, c)
    c["k"] = k
    got = run(pkg, c)
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(got[n], want[n]), n


def test_rows_around_the_outputs_stay(pkg, cuda):
    B, Lq, Lk, H, hd = 2, 45, 77, 2, 64
    c = make(cuda, torch.bfloat16, B, Lq, Lk, H, H, hd, seed=81, keys="mask")
    bufs = {n: torch.full((B, L + 9, H, hd + 8), 7.0, dtype=torch.bfloat16, device=cuda) for n, L in (("out", Lq), ("dq", Lq), ("dk", Lk), ("dv", Lk))}
    view = {n: t[:, 4:-5, :, :hd] for n, t in bufs.items()}
    stat = torch.empty(B, H, Lq, 2, device=cuda)
    pkg.ops.cross_attn(c["q"], c["k"], c["v"], view["out"], stat=stat, mask=c["mask"])
    pkg.ops.cross_attn_bwd(c["q"], c["k"], c["v"], view["out"], stat, c["dout"], view["dq"], view["dk"], view["dv"], mask=c["mask"])
    for n, t in bufs.items():
        assert bool((t[:, :4] == 7).all()) and bool((t[:, -5:] == 7).all()) and bool((t[..., hd:] == 7).all()), n
        assert bool(torch.isfinite(view[n]).all())


def test_captured_and_replayed(pkg, cuda):
    """two graphs of the same shapes, replayed in turn with the program's own eager calls between; every replay against the eager result"""
    cases = [make(cuda, torch.bfloat16, 2, 5, 900, 4, 2, 64, seed=s, keys="both", bias="rand") for s in (91, 92)]
    want = [{n: t.clone() for n, t in run(pkg, c).items()} for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = run(pkg, c)
        graphs.append((gr, got))
    for _ in range(3):
        for (gr, got), w in zip(graphs, want):
            for t in got.values():
                t.fill_(math.nan)
            gr.replay()
            run(pkg, cases[0])
            torch.cuda.synchronize()
            for n in w:
                assert torch.equal(got[n], w[n]), n
    c, (gr, got) = cases[0], graphs[0]
    c["q"].copy_(cases[1]["q"])                                            # new values in the captured operands
    c["kv_len"].copy_(cases[1]["kv_len"])
    c["att"] = (torch.arange(c["Lk"])[None] < c["kv_len"].cpu()[:, None]) & c["mask"].cpu()
    c["k"].copy_(torch.where(c["att"][..., None, None].to(cuda), torch.nan_to_num(c["k"], 0.5), c["k"]))
    c["v"].copy_(torch.where(c["att"][..., None, None].to(cuda), torch.nan_to_num(c["v"], 0.5, 0.5), c["v"]))
    gr.replay()
    torch.cuda.synchronize()
    now = {n: t.clone() for n, t in got.items()}
    for n, t in run(pkg, c).items():
        assert torch.equal(now[n], t), n


def test_two_streams_at_once(pkg, cuda):
    cases = [make(cuda, torch.bfloat16, 2, 3, 3500, 4, 4, 64, seed=s, keys="mask") for s in (95, 96)]
    want = [run(pkg, c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i] = run(pkg, c)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for n in w:
            assert w[n] is None or torch.equal(g[n], w[n]), n


def test_agrees_with_the_decoder_attention(pkg, cuda):
    """the mask decoder's tokens -> image attention (8 heads of 16), f32, through both entry points: both within f32 roundings of the definition"""
    B, Lq, Lk, H, hd = 2, 7, 600, 8, 16
    c = make(cuda, torch.float32, B, Lq, Lk, H, H, hd, seed=97)
    got = check(pkg, c, backward=False)["out"]
    small = torch.empty(B * Lq, H * hd, device=cuda)
    pkg.ops.attn_small(c["q"].reshape(B * Lq, -1), c["k"].reshape(B * Lk, -1), c["v"].reshape(B * Lk, -1), small, B, H, hd, Lq, Lk, c["scale"])
    _, tol = reference(c)
    assert bool(((got.reshape(B * Lq, -1) - small).abs().double() <= 2 * tol["out"].reshape(B * Lq, -1)).all())


def test_refusals(pkg, cuda):
    o = pkg.ops
    c = make(cuda, torch.bfloat16, 2, 8, 16, 4, 2, 64, seed=99)
    q, k, v, out = c["q"], c["k"], c["v"], torch.empty_like(c["q"])
    stat = torch.empty(2, 4, 8, 2, device=cuda)
    bad = [
        ("GPU", lambda: o.cross_attn(q.cpu(), k, v, out)),
        ("one dtype", lambda: o.cross_attn(q, k.float(), v, out)),
        ("one dtype", lambda: o.cross_attn(q.half(), k.half(), v.half(), out.half())),
        ("shape mismatch", lambda: o.cross_attn(q, k, v[:, :8], out)),
        ("shape mismatch", lambda: o.cross_attn(q, k, v, out[:, :4])),
        ("no multiple", lambda: o.cross_attn(q[:, :, :3], k, v, out[:, :, :3])),
        ("head dim", lambda: o.cross_attn(q[..., :60], k[..., :60], v[..., :60], out[..., :60])),
        ("aligned", lambda: o.cross_attn(q[..., 4:12], k[..., :8], v[..., :8], out[..., :8])),
        ("contiguous", lambda: o.cross_attn(q.transpose(2, 3), k.transpose(2, 3), v.transpose(2, 3), out.transpose(2, 3))),
        ("empty", lambda: o.cross_attn(q[:, :0], k, v, out[:, :0])),
        ("empty", lambda: o.cross_attn(q, k[:, :0], v[:, :0], out)),
        ("kv_len", lambda: o.cross_attn(q, k, v, out, kv_len=torch.ones(2, dtype=torch.int64, device=cuda))),
        ("mask", lambda: o.cross_attn(q, k, v, out, mask=torch.ones(2, 8, dtype=torch.uint8, device=cuda))),
        ("bias", lambda: o.cross_attn(q, k, v, out, bias=torch.zeros(4, 8, 16, dtype=torch.bfloat16, device=cuda))),
        ("scale", lambda: o.cross_attn(q, k, v, out, scale=0.0)),
        ("stat", lambda: o.cross_attn(q, k, v, out, stat=stat[:1])),
        ("another operand", lambda: o.cross_attn(q, k, v, q)),
        ("not there", lambda: o.cross_attn_bwd(q, k, v, out, stat, out.clone(), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v),
                                               dbias=torch.empty(4, 8, 16, device=cuda))),
        ("another operand", lambda: o.cross_attn_bwd(q, k, v, out, stat, out.clone(), q, torch.empty_like(k), torch.empty_like(v))),
    ]
    for match, call in bad:
        with pytest.raises(ValueError, match=match):
            call()
