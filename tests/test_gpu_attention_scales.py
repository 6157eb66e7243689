"""Scales that fp32 cannot hold, or whose product with log2 e it cannot hold: PyTorch's operators take them, as they do on the CPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


@pytest.mark.parametrize("scale", [1e-46, 1e-39, 2.0 ** -126, 2.0 ** 126, 3e38])
@pytest.mark.parametrize("joint", [False, True])
def test_extreme_scales(scale, joint):
    """Queries of zero: every score is zero whatever the scale, and a row is the mean of the values up to it."""
    from bluefog_b200.ops import fused_attention as fa
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(140, 2, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.zeros_like(k)
    if joint:
        out = fa.causal_self_attention(torch.cat([t.flatten(1) for t in (q, k, v)], 1), 2, scale=scale)
    else:
        out = fa.causal_attention(q, k, v, scale=scale)
    fa.check_sequences()
    count = torch.arange(1, 141, device="cuda", dtype=torch.float64)[:, None, None]
    want = v.double().cumsum(0) / count
    # weights and result are rounded once each
    bound = 1.1 * U * (want.abs() + v.double().abs().cumsum(0) / count) + 1e-5
    assert ((out.double() - want).abs() <= bound).all()
