"""Gradients of the gated block over the range of bf16.  Multiplying the incoming gradient by a power of two multiplies every number
of the backward pass by it, and no rounding changes, as long as none of them leaves the range of its type: so the gradients have
to be the same bits but for the exponent."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,f,n", [(8, 64, 136, 72), (100, 72, 64, 64), (300, 264, 200, 136), (600, 512, 1376, 512)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_scale_with_the_incoming_one(m, k, f, n, act):
    from bluefog_b200.ops import gemm
    g = torch.Generator(device="cuda").manual_seed(m)
    x, wgu, wd, dy = ((torch.randn(*s, generator=g, device="cuda") * std).to(torch.bfloat16).requires_grad_(True)
                      for s, std in (((m, k), 1.0), ((2 * f, k), k ** -0.5), ((n, f), f ** -0.5), ((m, n), 1.0)))
    leaves = [x, wgu, wd]
    want = torch.autograd.grad(gemm.gated_mlp(*leaves, act=act), leaves, dy.detach())
    for exponent in (-40, 20, 37, 40, 64, 100):
        got = torch.autograd.grad(gemm.gated_mlp(*leaves, act=act), leaves, dy.detach() * 2.0 ** exponent)
        for name, a, b in zip(("da", "dw_gate_up", "dw_down"), got, want):
            assert torch.equal(a, b * 2.0 ** exponent), (name, exponent, a.isinf().sum().item(), a.isnan().sum().item())
