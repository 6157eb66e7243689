"""Forward-mode differentiation of the transformer-block operators: the kernels have no such rule, and a tangent that reaches them is
an error instead of a result without one."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _bf16(*shape):
    return torch.randn(*shape, device="cuda").to(torch.bfloat16)


def _operators():
    from bluefog_b200.ops import fused_attention as fa, fused_dropout as fd, gemm
    key = fd.new_key(3, "cuda")
    return {
        "attention": (fa.causal_attention, [_bf16(20, 2, 64), _bf16(20, 1, 64), _bf16(20, 1, 64)]),
        "joint": (lambda qkv: fa.causal_self_attention(qkv, 2, 1), [_bf16(20, 256)]),
        "dropout": (lambda x, r: fd.dropout_add(x, r, 0.1, key), [_bf16(9, 16), _bf16(9, 16)]),
        "gated": (lambda a, u, d, r: gemm.gated_mlp(a, u, d, residual=r), [_bf16(9, 64), _bf16(32, 64), _bf16(24, 16), _bf16(9, 24)]),
    }


@pytest.mark.parametrize("name,count", [("attention", 3), ("joint", 1), ("dropout", 2), ("gated", 4)])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, count, grad):
    op, args = _operators()[name]
    assert len(args) == count
    args = [a.requires_grad_(grad) for a in args]
    want = op(*args)
    for i in range(count):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward"):
                op(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                op(*dual)
            assert torch.equal(op(*args), want)                       # without a tangent, inside the same level


@pytest.mark.parametrize("name", ["attention", "joint", "dropout", "gated"])
def test_tangents_of_incoming_gradients_are_refused(name):
    op, args = _operators()[name]
    args = [a.requires_grad_(True) for a in args]
    out = op(*args)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(out, args[:1], dy)


def test_a_level_that_is_switched_off_does_not_count():
    op, args = _operators()["joint"]
    want = op(*args)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with forward_ad._set_fwd_grad_enabled(False):
            out = op(dual)
        assert torch.equal(out, want)
