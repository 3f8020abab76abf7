"""Attention between two token sets where it once went wrong, or could: very large scores with a bias."""
import pytest
import torch

from tests.test_gpu_cross_attn import DT, check, make

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
