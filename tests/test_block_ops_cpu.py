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


def test_philox_reference_vectors():
    """The generator against the three test vectors published with it."""
    from test_gpu_dropout import philox
    ones = 0xFFFFFFFF
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("count,p,seed,step,site", [(1, 0.5, 0, 0, 0), (41, 0.1, -5, 2 ** 33 + 1, 7), (64, 1.0, 1, 1, 1), (64, 0.0, 1, 1, 1)])
def test_dropout_on_the_cpu(count, p, seed, step, site):
    from bluefog_b200.ops import fused_dropout
    from test_gpu_dropout import kept
    x = torch.randn(count, dtype=torch.float64, requires_grad=True)
    r = torch.randn(count, dtype=torch.float64)
    keep = kept(count, p, seed, step, site)
    y = fused_dropout.dropout_add(x, r, p, torch.tensor([seed, step]), site)
    q = round(65536 * p) / 65536
    factor = keep.double() / (1 - q) if q < 1 else torch.zeros(count, dtype=torch.float64)
    torch.testing.assert_close(y, r + x * factor)
    (g,) = torch.autograd.grad(y.sum(), x)
    torch.testing.assert_close(g, factor)


@pytest.mark.parametrize("change", [
    dict(p=-0.1), dict(p=1.1), dict(p=math.nan), dict(x=torch.zeros(4, 4, dtype=torch.int64)), dict(residual=torch.zeros(4)),
    dict(residual=torch.zeros(4, 4, dtype=torch.float64)), dict(key=torch.zeros(2)), dict(key=torch.zeros(3, dtype=torch.int64)),
    dict(site=-1), dict(site=65536)])
def test_dropout_refuses(change):
    from bluefog_b200.ops import fused_dropout
    args = dict(x=torch.zeros(4, 4), residual=None, p=0.1, key=fused_dropout.new_key(0))
    args.update(change)
    with pytest.raises(ValueError):
        fused_dropout.dropout_add(**args)


def test_gated_mlp_on_the_cpu():
    import torch.nn.functional as F
    from bluefog_b200.ops import gemm
    torch.manual_seed(0)
    a, wgu, wd, r = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((3, 5, 6), (14, 6), (4, 7), (3, 5, 4)))
    g, u = F.linear(a, wgu[:7]), F.linear(a, wgu[7:])
    torch.testing.assert_close(gemm.gated_mlp(a, wgu, wd, residual=r), F.linear(F.silu(g) * u, wd) + r)
    torch.testing.assert_close(gemm.gated_mlp(a, wgu, wd, act="gelu"), F.linear(F.gelu(g, approximate="tanh") * u, wd))
    assert torch.autograd.gradcheck(lambda *t: gemm.gated_mlp(*t), (a, wgu, wd))


@pytest.mark.parametrize("change", [
    dict(act="relu"), dict(a=torch.zeros(3, 5)), dict(w_gate_up=torch.zeros(13, 6)), dict(w_down=torch.zeros(4, 6)),
    dict(w_down=torch.zeros(7)), dict(residual=torch.zeros(4)), dict(residual=torch.zeros(3, 6)),
    dict(residual=torch.zeros(3, 4, dtype=torch.float64)), dict(a=torch.zeros(3, 6, dtype=torch.float64))])
def test_gated_mlp_refuses(change):
    from bluefog_b200.ops import gemm
    args = dict(a=torch.zeros(3, 6), w_gate_up=torch.zeros(14, 6), w_down=torch.zeros(4, 7))
    args.update(change)
    with pytest.raises(ValueError):
        gemm.gated_mlp(**args)


def _gpt2(**kw):
    from bluefog_b200.models import gpt2
    torch.manual_seed(0)
    return gpt2.GPT2(vocab_size=101, n_positions=16, d_model=32, n_layer=2, n_head=4, **kw)


def test_gpt2_keeps_its_parameters_and_results_without_the_options():
    a = _gpt2()
    assert a.h[0].attn.c_attn.weight.shape == (96, 32) and a.h[0].mlp.c_fc.weight.shape == (128, 32)
    assert not any("dropout" in n for n in a.state_dict())
    idx = torch.randint(0, 101, (2, 16))
    torch.testing.assert_close(_gpt2(use_b200_attention=True)(idx), a(idx))


def test_gpt2_documents_do_not_see_each_other():
    m = _gpt2(n_kv_head=2, mlp="swiglu")
    assert m.h[0].attn.c_attn.weight.shape == (64, 32) and m.h[0].mlp.c_fc.weight.shape == (2 * 128, 32)
    idx = torch.randint(0, 101, (1, 16))
    cu = torch.tensor([0, 5, 16], dtype=torch.int32)
    want = m(idx, cu_seqlens=cu)
    other = idx.clone()
    other[:, :5] = (other[:, :5] + 1) % 101
    got = m(other, cu_seqlens=cu)
    assert torch.equal(got[:, 5:], want[:, 5:]) and not torch.equal(got[:, :5], want[:, :5])
    assert not torch.equal(m(other)[:, 5:], m(idx)[:, 5:])


def test_gpt2_dropout_draws_a_mask_per_step_and_none_in_evaluation():
    m = _gpt2(dropout=0.3, mlp="geglu")
    assert m.dropout_key.tolist()[1] == 0 and "dropout_key" in m.state_dict()
    idx = torch.randint(0, 101, (2, 16))
    a, b = m(idx), m(idx)
    assert not torch.equal(a, b) and m.dropout_key.tolist()[1] == 2
    m.dropout_key[1] = 0
    assert torch.equal(m(idx), a)
    m.eval()
    assert torch.equal(m(idx), m(idx)) and m.dropout_key.tolist()[1] == 1
    m.train()
    m(idx, torch.randint(0, 101, (2, 16))).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


@pytest.mark.parametrize("kw", [dict(n_kv_head=3), dict(n_kv_head=0), dict(mlp="relu"), dict(dropout=1.0), dict(dropout=-0.1)])
def test_gpt2_refuses(kw):
    with pytest.raises(ValueError):
        _gpt2(**kw)
