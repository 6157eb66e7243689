"""Attention on gradients and inputs that are broadcast along the tokens, the sequences or the heads: the same numbers as on dense
copies of them, bit for bit, since the kernels then run on such a copy."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _bf16(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _grads(lead, h, hkv, d, reduce, cu, dense):
    from bluefog_b200.ops import fused_attention as fa
    leaves = [_bf16(*lead, n, d, seed=n + i).requires_grad_(True) for i, n in enumerate((h, hkv, hkv))]
    out = fa.causal_attention(*leaves, cu_seqlens=cu)
    seen = []
    out.register_hook(lambda g: seen.append(g.stride()) or (g.clone(memory_format=torch.contiguous_format) if dense else None))
    z = reduce(out)
    grads = torch.autograd.grad(z, leaves, _bf16(*z.shape, seed=9))
    return seen[0], grads


@pytest.mark.parametrize("lead,h,hkv,d,dims,packed", [
    ((150,), 4, 4, 64, 0, False), ((150,), 4, 2, 64, 0, True), ((1, 150), 4, 1, 128, 1, False), ((3, 70), 2, 2, 64, 1, False),
    ((2, 129), 4, 2, 80, 1, False), ((3, 70), 2, 2, 64, 0, False), ((3, 70), 4, 2, 64, (0, 1), False), ((3, 70), 4, 2, 64, 2, False),
    ((70, 1), 2, 1, 64, 0, False)])
def test_gradients_of_sums(lead, h, hkv, d, dims, packed):
    cu = torch.tensor([0, 31, 31, 140], dtype=torch.int32, device="cuda") if packed else None
    strides, got = _grads(lead, h, hkv, d, lambda y: y.sum(dims), cu, False)
    assert 0 in strides
    _, want = _grads(lead, h, hkv, d, lambda y: y.sum(dims), cu, True)
    for name, a, b in zip("qkv", got, want):
        assert torch.equal(a, b), name


def test_gradient_of_a_sum_behind_flattened_heads():
    strides, got = _grads((2, 130), 4, 2, 64, lambda y: y.flatten(-2).sum(1), None, False)
    assert 0 in strides
    _, want = _grads((2, 130), 4, 2, 64, lambda y: y.flatten(-2).sum(1), None, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("shape,full", [((1, 2, 64), (150, 2, 64)), ((2, 1, 2, 64), (2, 130, 2, 64)), ((1, 130, 2, 64), (3, 130, 2, 64))])
def test_broadcast_inputs(shape, full):
    from bluefog_b200.ops import fused_attention as fa

    def run(dense):
        leaves = [_bf16(*shape, seed=i).requires_grad_(True) for i in range(3)]
        views = [t.expand(full) for t in leaves]
        out = fa.causal_attention(*[v.contiguous() if dense else v for v in views])
        return [out.detach(), *torch.autograd.grad(out, leaves, _bf16(*full, seed=5))]

    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))


@pytest.mark.parametrize("shape,full", [((1, 256), (150, 256)), ((2, 1, 256), (2, 130, 256)), ((1, 130, 256), (3, 130, 256)), ((1, 1, 256), (2, 70, 256))])
def test_broadcast_joint_projection(shape, full):
    from bluefog_b200.ops import fused_attention as fa

    def run(dense):
        leaf = _bf16(*shape).requires_grad_(True)
        qkv = leaf.expand(full)
        out = fa.causal_self_attention(qkv.contiguous() if dense else qkv, 2, 1)
        return [out.detach(), *torch.autograd.grad(out, leaf, _bf16(*out.shape, seed=5))]

    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))
