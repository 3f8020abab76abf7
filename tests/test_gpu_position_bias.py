"""Learned position bias by buckets: values to the bit, gradient within the rounding of its sums, and both together with the attention."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def index(q_grid, k_grid, by, bx):
    """(row, column) of the table for every pair, by the definition, on the CPU"""
    (qh, qw), (kh, kw) = q_grid, k_grid
    i, j = torch.arange(qh * qw), torch.arange(kh * kw)
    iy = (j // kw)[None] - (i // qw)[:, None] + qh - 1
    ix = (j % kw)[None] - (i % qw)[:, None] + qw - 1
    return by.long()[iy], bx.long()[ix]


def maps(pkg, q_grid, k_grid, ny, nx, reach=32, offset=0):
    by = pkg.ops.bucket_map(q_grid[0], k_grid[0], ny, reach) if ny > 1 else torch.zeros(q_grid[0] + k_grid[0] - 1, dtype=torch.int32)
    return by, pkg.ops.bucket_map(q_grid[1], k_grid[1], nx, reach, offset=offset)


GRIDS = [((1, 1), (1, 1), 1, 8), ((1, 1), (5, 7), 4, 8), ((9, 5), (3, 11), 8, 12), ((37, 37), (37, 37), 16, 16), ((1, 40), (1, 300), 1, 32), ((1, 1030), (1, 5), 1, 32),
         ((1, 3), (1, 9000), 1, 64), ((70, 2), (2, 70), 16, 128), ((2, 600), (3, 90), 4, 130)]


@pytest.mark.parametrize("q_grid,k_grid,ny,nx", GRIDS)
@pytest.mark.parametrize("H,pad", [(1, 0), (5, 13)])
def test_values_and_gradient(pkg, cuda, q_grid, k_grid, ny, nx, H, pad):
    g = torch.Generator().manual_seed(nx + H)
    by, bx = maps(pkg, q_grid, k_grid, ny, nx, 2048 if k_grid[1] > 1000 else 200)
    Lq, Lk = q_grid[0] * q_grid[1], k_grid[0] * k_grid[1]
    table = torch.randn(ny, nx, H, generator=g)
    iy, ix = index(q_grid, k_grid, by, bx)
    want = table[iy, ix].permute(2, 0, 1)
    buf = torch.full((H, Lq + 1, Lk + pad), 7.0, device=cuda)
    out = buf[:, :Lq, :Lk]
    dev = [t.to(cuda) for t in (by, bx)]
    pkg.ops.bucket_bias(table.to(cuda), *dev, out, q_grid=q_grid, k_grid=k_grid)
    assert torch.equal(out.cpu(), want)
    assert bool((buf[:, Lq:] == 7).all()) and bool((buf[..., Lk:] == 7).all())

    buf.normal_()
    d = out.cpu().double()
    grad, mag = torch.zeros(ny * nx, H, dtype=torch.float64), torch.zeros(ny * nx, H, dtype=torch.float64)
    rows = (iy * nx + ix).reshape(-1)
    grad.index_add_(0, rows, d.reshape(H, -1).t().contiguous())
    mag.index_add_(0, rows, d.abs().reshape(H, -1).t().contiguous())
    got = torch.full((ny, nx, H), math.nan, device=cuda)
    pkg.ops.bucket_bias_bwd(out, *dev, got, q_grid=q_grid, k_grid=k_grid)
    # no value passes through more additions than: the rows a thread adds (1024 at most), the row subsets and offsets of a workgroup (8 + 64 + 8), the
    # pieces of a bucket
    parts = (Lq // 1024 + 1) * ((q_grid[1] + k_grid[1]) // 512 + 1) * (q_grid[0] + k_grid[0])
    bound = (1104 + parts) * 2.0 ** -24 * mag + 1e-30
    assert bool(((got.cpu().double().view(-1, H) - grad).abs() <= bound).all())
    again = torch.empty_like(got)
    pkg.ops.bucket_bias_bwd(out, *dev, again, q_grid=q_grid, k_grid=k_grid)
    assert torch.equal(got, again)


def test_offsets_outside_the_table(pkg, cuda):
    """entries of the maps outside the table: no bias, and what the gradient holds there (NaN) reaches nothing"""
    q_grid, k_grid, ny, nx, H = (4, 6), (5, 3), 3, 4, 2
    by = torch.tensor([-1, 0, 1, 2, 1, 3, 0, 2], dtype=torch.int32)
    bx = torch.tensor([0, 1, 2, 3, 4, -7, 1, 0], dtype=torch.int32)
    iy, ix = index(q_grid, k_grid, by, bx)
    ok = (iy >= 0) & (iy < ny) & (ix >= 0) & (ix < nx)
    table = torch.arange(1.0, ny * nx * H + 1).view(ny, nx, H)
    want = torch.where(ok[..., None], table[iy.clamp(0, ny - 1), ix.clamp(0, nx - 1)], torch.zeros(())).permute(2, 0, 1)
    out = torch.full((H, 24, 15), math.nan, device=cuda)
    pkg.ops.bucket_bias(table.to(cuda), by.to(cuda), bx.to(cuda), out, q_grid=q_grid, k_grid=k_grid)
    assert torch.equal(out.cpu(), want)
    d = torch.where(ok, torch.ones(()), torch.full((), math.nan)).expand(H, -1, -1).contiguous().to(cuda)
    got = torch.empty(ny, nx, H, device=cuda)
    pkg.ops.bucket_bias_bwd(d, by.to(cuda), bx.to(cuda), got, q_grid=q_grid, k_grid=k_grid)
    count = torch.zeros(ny * nx).index_add_(0, (iy * nx + ix)[ok], torch.ones(int(ok.sum())))
    assert torch.equal(got.cpu(), count.view(ny, nx, 1).expand(-1, -1, H))


def test_one_token_of_a_sequence(pkg, cuda):
    """the bias row of the token at position t, made alone, is row t of the whole bias"""
    L, H, nx = 50, 3, 16
    table = torch.randn(1, nx, H, device=cuda)
    zero = torch.zeros(2 * L - 1, dtype=torch.int32, device=cuda)[:1]
    whole, row = torch.empty(H, L, L, device=cuda), torch.empty(H, 1, L, device=cuda)
    pkg.ops.bucket_bias(table, zero, pkg.ops.bucket_map(L, L, nx, 30).to(cuda), whole, q_grid=(1, L), k_grid=(1, L))
    for t in (0, 17, L - 1):
        pkg.ops.bucket_bias(table, zero, pkg.ops.bucket_map(1, L, nx, 30, offset=t).to(cuda), row, q_grid=(1, 1), k_grid=(1, L))
        assert torch.equal(row[:, 0], whole[:, t])


def test_captured_and_replayed(pkg, cuda):
    q_grid = k_grid = (12, 12)
    by, bx = (t.to(cuda) for t in maps(pkg, q_grid, k_grid, 8, 8))
    table, out = torch.randn(8, 8, 4, device=cuda), torch.empty(4, 144, 144, device=cuda)
    got = torch.empty_like(table)

    def both():
        pkg.ops.bucket_bias(table, by, bx, out, q_grid=q_grid, k_grid=k_grid)
        pkg.ops.bucket_bias_bwd(out, by, bx, got, q_grid=q_grid, k_grid=k_grid)

    both()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        both()
    for i in range(3):
        table.normal_()
        both()
        want = (out.clone(), got.clone())
        out.fill_(math.nan), got.fill_(math.nan)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(got, want[1])


def test_refusals(pkg, cuda):
    o = pkg.ops
    table, out = torch.zeros(4, 4, 2, device=cuda), torch.empty(2, 6, 6, device=cuda)
    by, bx = torch.zeros(3, dtype=torch.int32, device=cuda), torch.zeros(5, dtype=torch.int32, device=cuda)
    kw = dict(q_grid=(2, 3), k_grid=(2, 3))
    o.bucket_bias(table, by, bx, out, **kw)
    for match, call in [
        ("by must", lambda: o.bucket_bias(table, by[:2], bx, out, **kw)),
        ("bx must", lambda: o.bucket_bias(table, by, bx.long(), out, **kw)),
        ("table", lambda: o.bucket_bias(table.bfloat16(), by, bx, out, **kw)),
        ("bias must", lambda: o.bucket_bias(table, by, bx, out[:1], **kw)),
        ("bias must", lambda: o.bucket_bias(table, by, bx, out.bfloat16(), **kw)),
        ("overlap", lambda: o.bucket_bias(table, by, bx, torch.empty(2, 1, 6, device=cuda).expand(2, 6, 6), **kw)),
        ("share memory", lambda: o.bucket_bias(table, by, bx, torch.empty(1, 6, 6, device=cuda).expand(2, 6, 6), **kw)),
        ("empty grid", lambda: o.bucket_bias(table, by, bx, out, q_grid=(0, 3), k_grid=(2, 3))),
        ("table", lambda: o.bucket_bias_bwd(out, by, bx, table.double(), **kw)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
