"""Results of the gated block and of dropout changed in place, as a residual stream that is added to does."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _bf16(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("lead", [(8,), (200,), (2, 100), (1, 1, 70), ()])
@pytest.mark.parametrize("residual", [False, True])
def test_gated_block(lead, residual):
    from bluefog_b200.ops import gemm
    leaves = [t.requires_grad_(True) for t in (_bf16(*lead, 64), _bf16(272, 64, seed=1), _bf16(72, 136, seed=2))]
    x, dy = _bf16(*lead, 72, seed=3).requires_grad_(True), _bf16(*lead, 72, seed=4)

    def run(in_place):
        y = gemm.gated_mlp(*leaves, residual=x if residual else None)
        if in_place:
            y += x
            y.mul_(0.5)
        else:
            y = (y + x) * 0.5
        return [y.detach(), *torch.autograd.grad(y, leaves + [x], dy)]

    assert run(False)[0].shape == dy.shape
    assert all(torch.equal(a, b) for a, b in zip(run(True), run(False)))
    with torch.no_grad():
        y = gemm.gated_mlp(*leaves)
        assert y.shape == dy.shape and y._base is None
        y += x


def test_dropout():
    from bluefog_b200.ops import fused_dropout
    x, r, dy = (_bf16(9, 16, seed=i) for i in range(3))
    key = fused_dropout.new_key(5, "cuda")

    def run(in_place):
        leaves = [t.clone().requires_grad_(True) for t in (x, r)]
        y = fused_dropout.dropout_add(*leaves, 0.3, key)
        if in_place:
            y += leaves[1]
        else:
            y = y + leaves[1]
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    assert all(torch.equal(a, b) for a, b in zip(run(True), run(False)))
