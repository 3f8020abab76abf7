"""The activations of group norm far from zero, where a value is small beside its argument."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("C,G", [(4096, 1), (4096, 512)])           # one workgroup a group, and pieces of 32 bytes: three launches
def test_gelu_keeps_its_digits_in_the_tail(pkg, cuda, C, G):
    """Arguments from -12 to 12 exactly (w = 0, so z = b), f32.  Relative to z Phi(z) the value may be off by the roundings of the exponential's argument z^2 / 2 (the square,
    the factor, its constant: 3 U of it, in the exponent) and by a few U each of the exponential, the reciprocal, eight multiply-adds and three products: 40 U.
    The slope is Phi + z phi: the same, of the sum of their magnitudes."""
    g = torch.Generator().manual_seed(C + G)
    x, dy = torch.randn(1, 3, C, generator=g).to(cuda), torch.ones(1, 3, C, device=cuda)
    b = torch.linspace(-12.0, 12.0, C).to(cuda)
    w = torch.zeros(C, device=cuda)
    out, dx, stat = torch.empty_like(x), torch.empty_like(x), torch.empty(1, G, 2, device=cuda)
    dw, db = torch.empty(C, device=cuda), torch.empty(C, device=cuda)
    pkg.ops.group_norm_act(x, w, b, out, G, 1e-5, pkg.hip.ACT_GELU, stat=stat)
    pkg.ops.group_norm_act_bwd(x, w, b, stat, dy, dx, dw, db, G, pkg.hip.ACT_GELU)
    z = b.double()
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    rel = (1.5 * z * z + 40) * U
    worst = float(((out.double() - z * cdf).abs() / (rel * (z * cdf).abs())).max())
    assert worst <= 1.0, f"value: {worst:.1f} of the bound"
    worst = float(((db.double() - 3 * (cdf + z * pdf)).abs() / (3 * (rel + 2 * U) * (cdf + (z * pdf).abs()))).max())
    assert worst <= 1.0, f"slope: {worst:.1f} of the bound"
