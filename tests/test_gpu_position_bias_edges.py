"""The gradient of the position bias reads the pairs of its grids and nothing around them."""
import math

import pytest
import torch

from tests.test_gpu_position_bias import index, maps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_grid", [(3, n) for n in (1, 2, 3, 5, 9, 17, 33)] + [(1, 7)])
@pytest.mark.parametrize("k_grid", [(8, 1), (8, 6), (9, 40), (64, 5), (70, 3)])
def test_nothing_around_the_rows_is_read(pkg, cuda, q_grid, k_grid):
    """rows of whole numbers inside a buffer of NaN, query columns in ragged groups: exact sums (every partial sum is below 2^24)"""
    g = torch.Generator().manual_seed(q_grid[1])
    H, ny, nx = 2, 8, 8
    by, bx = maps(pkg, q_grid, k_grid, ny, nx, 100)
    Lq, Lk = q_grid[0] * q_grid[1], k_grid[0] * k_grid[1]
    d = torch.randint(-8, 9, (H, Lq, Lk), generator=g).float()
    buf = torch.full((H, Lq + 2, Lk + 2 * q_grid[1] + 6), math.nan, device=cuda)
    view = buf[:, 1:-1, q_grid[1] + 3:q_grid[1] + 3 + Lk]
    view.copy_(d)
    iy, ix = index(q_grid, k_grid, by, bx)
    want = torch.zeros(ny * nx, H).index_add_(0, (iy * nx + ix).reshape(-1), d.reshape(H, -1).t().contiguous())
    got = torch.full((ny, nx, H), math.nan, device=cuda)
    pkg.ops.bucket_bias_bwd(view, by.to(cuda), bx.to(cuda), got, q_grid=q_grid, k_grid=k_grid)
    assert torch.equal(got.cpu().view(-1, H), want)
