"""Attention calls queued one behind the other without a pause.  The launches of a backward pass overlap, and the allocator gives every
call the workspace of the one before: a launch that read its row sums before they were there would find those of another call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(tokens, h, hkv, d, count):
    g = torch.Generator(device="cuda").manual_seed(tokens + h + d)
    mk = lambda n, scale: (torch.randn(tokens, n, d, generator=g, device="cuda") * scale).to(torch.bfloat16)
    # gradients of very different size: a row sum of another call shows in every digit
    return [([mk(n, 1.0).requires_grad_(True) for n in (h, hkv, hkv)], mk(h, 4.0 ** i)) for i in range(count)]


def _step(leaves, dout, cu):
    from bluefog_b200.ops import fused_attention as fa
    return torch.autograd.grad(fa.causal_attention(*leaves, cu_seqlens=cu), leaves, dout)


# key tiles shared by clusters of 2, 4 and 8 (query tiles are a launch of their own) or by none
SHAPES = [(700, 4, 2, 64), (700, 8, 1, 64), (2100, 16, 4, 64), (900, 16, 2, 128), (1500, 8, 8, 64), (1100, 2, 2, 128), (64, 4, 1, 64)]


@pytest.mark.parametrize("tokens,h,hkv,d", SHAPES)
@pytest.mark.parametrize("packed", [False, True])
def test_queued_calls_equal_separate_ones(tokens, h, hkv, d, packed):
    cu = torch.tensor([0, 1, tokens // 3, tokens // 3, tokens - 5], dtype=torch.int32, device="cuda") if packed else None
    calls = _inputs(tokens, h, hkv, d, 6)
    alone = []
    for leaves, dout in calls:
        torch.cuda.synchronize()
        alone.append([g.clone() for g in _step(leaves, dout, cu)])
    torch.cuda.synchronize()
    for _ in range(5):
        queued = [_step(leaves, dout, cu) for leaves, dout in calls]
        for got, want in zip(queued, alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tokens,h,hkv,d", SHAPES[1:4])
def test_replayed_calls_equal_separate_ones(tokens, h, hkv, d):
    calls = _inputs(tokens, h, hkv, d, 3)
    alone = [[g.clone() for g in _step(leaves, dout, None)] for leaves, dout in calls]
    fresh = [([t.detach().clone().requires_grad_(True) for t in leaves], dout) for leaves, dout in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [_step(leaves, dout, None) for leaves, dout in fresh]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, alone):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
