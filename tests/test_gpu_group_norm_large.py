"""Group norm on maps whose results are stored past the caches."""
import pytest
import torch

from tests.test_gpu_group_norm import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,N", [(torch.bfloat16, 4), (torch.float32, 12)])
def test_results_past_the_caches(pkg, cuda, dtype, N):
    """2^24 values in bf16, 3 * 2^24 in f32, and one map less than that"""
    check(pkg, cuda, N, 16384, 256, 32, 4, dtype, dtype, seed=N)
    check(pkg, cuda, N - 1, 16384, 256, 32, 1, dtype, dtype, seed=N)
