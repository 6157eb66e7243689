"""Transformer-block operators on the CPU: PyTorch's operators take their place, and wrong arguments are refused."""
import math

import pytest
import torch


def _attention(q, k, v, lengths):
    """The definition, row by row."""
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    start = 0
    for n in lengths:
        for h in range(q.shape[1]):
            for i in range(start, start + n):
                w = torch.softmax(k[start:i + 1, h // group] @ q[i, h] / math.sqrt(q.shape[2]), 0)
                out[i, h] = w @ v[start:i + 1, h // group]
        start += n
    return out


def test_attention_on_the_cpu_is_the_definition():
    from bluefog_b200.ops import fused_attention as fa
    torch.manual_seed(0)
    q, k, v = (torch.randn(17, n, 6, dtype=torch.float64) for n in (4, 2, 2))
    cu = torch.tensor([0, 5, 5, 6, 14], dtype=torch.int32)
    torch.testing.assert_close(fa.causal_attention(q, k, v, cu_seqlens=cu), _attention(q, k, v, [5, 0, 1, 8]))
    torch.testing.assert_close(fa.causal_attention(q, k, v), _attention(q, k, v, [17]))
    batch = fa.causal_attention(*(t[:16].view(2, 8, *t.shape[1:]) for t in (q, k, v)))
    torch.testing.assert_close(batch.flatten(0, 1), _attention(q[:16], k[:16], v[:16], [8, 8]))
    qkv = torch.cat([t.flatten(1) for t in (q, k, v)], 1)
    torch.testing.assert_close(fa.causal_self_attention(qkv, 4, 2, cu_seqlens=cu), _attention(q, k, v, [5, 0, 1, 8]))


def test_attention_gradients_on_the_cpu():
    from bluefog_b200.ops import fused_attention as fa
    torch.manual_seed(1)
    qkv = torch.randn(7, 4 * 4, dtype=torch.float64, requires_grad=True)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32)
    assert torch.autograd.gradcheck(lambda x: fa.causal_self_attention(x, 2, 1, cu_seqlens=cu), (qkv,))


def test_attention_of_no_tokens():
    from bluefog_b200.ops import fused_attention as fa
    q, k = torch.randn(0, 2, 8, requires_grad=True), torch.randn(0, 1, 8, requires_grad=True)
    out = fa.causal_attention(q, k, k, cu_seqlens=torch.zeros(3, dtype=torch.int32))
    assert out.shape == (0, 2, 8)
    out.sum().backward()
    assert q.grad.shape == q.shape and k.grad.shape == k.shape


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(4, 3, 8)), dict(k=torch.zeros(5, 2, 8), v=torch.zeros(5, 2, 8)), dict(v=torch.zeros(4, 2, 6)),
    dict(q=torch.zeros(4, 3, 8)), dict(q=torch.zeros(4, 4)), dict(q=torch.zeros(4, 4, 8, dtype=torch.float64)),
    dict(cu_seqlens=torch.tensor([0, 4])), dict(cu_seqlens=torch.tensor([0], dtype=torch.int32)),
    dict(cu_seqlens=torch.tensor([[0, 4]], dtype=torch.int32)), dict(cu_seqlens=torch.tensor([0, 3, 2], dtype=torch.int32)),
    dict(cu_seqlens=torch.tensor([1, 4], dtype=torch.int32)), dict(cu_seqlens=torch.tensor([0, 5], dtype=torch.int32)),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)])
def test_attention_refuses(change):
    from bluefog_b200.ops import fused_attention as fa
    args = dict(q=torch.zeros(4, 4, 8), k=torch.zeros(4, 2, 8), v=torch.zeros(4, 2, 8))
    args.update(change)
    with pytest.raises(ValueError):
        fa.causal_attention(**args)


@pytest.mark.parametrize("shape,h,hkv", [((4, 30), 2, 1), ((4, 32), 0, 1), ((4, 32), 2, 0), ((32,), 2, 1), ((2, 2, 2, 32), 2, 1), ((4, 35), 3, 2)])
def test_side_by_side_projection_refuses(shape, h, hkv):
    from bluefog_b200.ops import fused_attention as fa
    with pytest.raises(ValueError):
        fa.causal_self_attention(torch.zeros(shape), h, hkv)
