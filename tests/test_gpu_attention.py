"""Causal attention kernels against the definition in fp64: results and gradients at the sizes, head layouts, strides and
sequence boundaries where they can go wrong.

Tolerances count roundings.  With u = 2^-8 (half a step of bf16 relative to the value) P, dS and the results are rounded
once each, so elementwise  |out|: u |out| + u P|v|;  delta = rowsum(dout * out) inherits |dout| times that;
dS: u |dS| + P * delta's error;  and each gradient adds u of itself to what its operands' errors make of it.  fp32
arithmetic inside (exponentials to 2^-21, sums of up to some thousand terms) is covered by one tenth on top and 1e-5 of
the largest value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def _oracle(q, k, v, dout, lengths, scale):
    """out, dq, dk, dv in fp64 and how far each may be off; all [tokens, heads, D]."""
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    h, hkv = q.shape[1], k.shape[1]
    res = [torch.zeros_like(t) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in (q, q, k, v)]
    start = 0
    for n in lengths:
        s = slice(start, start + n)
        start += n
        for i in range(h if n else 0):
            j = i * hkv // h
            a, b, c, d = q[s, i], k[s, j], v[s, j], dout[s, i]
            mask = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
            p = torch.softmax((scale * a @ b.t()).masked_fill(~mask, -math.inf), -1)
            out = p @ c
            t_out = U * out.abs() + U * (p @ c.abs())
            dp = d @ c.t()
            ds = p * (dp - (d * out).sum(1, keepdim=True))
            t_ds = U * ds.abs() + p * (d.abs() * t_out).sum(1, keepdim=True)
            res[0][s, i], tol[0][s, i] = out, t_out
            res[1][s, i], tol[1][s, i] = scale * ds @ b, scale * t_ds @ b.abs()
            res[2][s, j] += scale * ds.t() @ a
            tol[2][s, j] += scale * t_ds.t() @ a.abs()
            res[3][s, j] += p.t() @ d
            tol[3][s, j] += U * p.t() @ d.abs()
    for r, t in zip(res[1:], tol[1:]):
        t += U * r.abs()
    return res, [1.1 * t + 1e-5 * max(1.0, r.abs().max().item()) for r, t in zip(res, tol)]


def _compare(got, lengths, q, k, v, dout, scale=None):
    flat = [t.detach().reshape(-1, *t.shape[-2:]) for t in (q, k, v, dout)]
    res, tol = _oracle(*flat, lengths, 1 / math.sqrt(q.shape[-1]) if scale is None else scale)
    for name, g, r, t in zip(("out", "dq", "dk", "dv"), got, res, tol):
        g = g.detach().reshape(r.shape).double()
        assert torch.isfinite(g).all(), name
        worst = ((g - r).abs() / t).max().item()
        assert worst <= 1.0, (name, worst)


def _inputs(tokens, h, hkv, d, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + tokens + 7 * h + d)
    return [torch.randn(*tokens, n, d, generator=g, device="cuda").to(torch.bfloat16)
            for tokens, n in ((t, n) for t, n in (((tokens,), h), ((tokens,), hkv), ((tokens,), hkv), ((tokens,), h)))]


def _run(q, k, v, dout, **kw):
    from bluefog_b200.ops import fused_attention as fa
    assert fa._eligible(q, q.shape[-1])
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = fa.causal_attention(*leaves, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _cu(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


DENSE = [(1, 1, 1, 1, 64), (2, 37, 3, 3, 64), (1, 128, 2, 1, 64), (1, 129, 2, 2, 128), (3, 200, 4, 2, 32), (1, 300, 6, 2, 80),
         (2, 513, 2, 1, 128), (1, 1100, 1, 1, 8), (2, 1024, 4, 4, 64), (1, 700, 8, 1, 64), (5, 2, 2, 2, 128), (1, 2050, 2, 1, 128)]


@pytest.mark.parametrize("b,t,h,hkv,d", DENSE)
def test_sequences_of_one_length(b, t, h, hkv, d):
    q, k, v, dout = (z.view(b, t, *z.shape[1:]) for z in _inputs(b * t, h, hkv, d))
    _compare(_run(q, k, v, dout), [t] * b, q, k, v, dout)


PACKED = [([5, 1, 0, 130, 128, 3], 0, 2, 2, 64), ([256, 257, 255], 31, 4, 2, 128), ([1], 0, 1, 1, 64), ([0, 0, 9], 400, 2, 1, 64),
          ([1] * 150, 5, 2, 2, 32), ([700, 64, 1, 1, 500], 1, 3, 1, 64), ([0, 127], 129, 2, 2, 128), ([1, 1000, 40], 0, 4, 1, 96),
          ([3] * 1100, 0, 1, 1, 64)]


@pytest.mark.parametrize("lengths,padding,h,hkv,d", PACKED)
def test_packed_sequences(lengths, padding, h, hkv, d):
    n = sum(lengths)
    q, k, v, dout = _inputs(n + padding, h, hkv, d)
    got = _run(q, k, v, dout, cu_seqlens=_cu(lengths))
    _compare([g[:n] for g in got], lengths, q[:n], k[:n], v[:n], dout[:n])
    assert all((g[n:] == 0).all() for g in got)                       # tokens behind the last sequence
    from bluefog_b200.ops import fused_attention
    fused_attention.check_sequences()


@pytest.mark.parametrize("d", [64, 128])
def test_nothing_leaks_out_of_another_sequence_or_the_padding(d):
    lengths, padding = [100, 200, 30, 129], 77
    n = sum(lengths)
    q, k, v, dout = _inputs(n + padding, 4, 2, d)
    clean = _run(q, k, v, dout, cu_seqlens=_cu(lengths))
    bad = [t.clone() for t in (q, k, v, dout)]
    for i, t in enumerate(bad):
        t[100:300] = math.nan if i % 2 else math.inf
        t[n:] = math.inf if i % 2 else math.nan
    got = _run(*bad, cu_seqlens=_cu(lengths))
    for a, b in zip(clean, got):
        assert torch.equal(a[:100], b[:100]) and torch.equal(a[300:], b[300:])
        assert b[100:300].isnan().any()


@pytest.mark.parametrize("d", [64, 128])
def test_rising_scores_rescale_the_output(d):
    """Keys grow towards the end and, separately, towards the start: the maximum of a row moves from tile to tile by far
    more than the kernel's threshold."""
    t = 700
    for flip in (False, True):
        q, k, v, dout = _inputs(t, 2, 1, d)
        ramp = torch.linspace(0.05, 6, t, device="cuda")
        k = (k.float() * (ramp.flip(0) if flip else ramp)[:, None, None]).to(torch.bfloat16)
        _compare(_run(q, k, v, dout), [t], q, k, v, dout)


def test_scale_and_equal_scores():
    q, k, v, dout = _inputs(260, 2, 2, 64)
    _compare(_run(q, k, v, dout, scale=0.7), [260], q, k, v, dout, scale=0.7)
    zero = torch.zeros_like(q)
    _compare(_run(zero, k, v, dout), [260], zero, k, v, dout)


def test_strided_and_unaligned_inputs():
    from bluefog_b200.ops import fused_attention as fa
    b, t, h, hkv, d = 2, 150, 4, 2, 64
    q, k, v, dout = (z.view(b, t, *z.shape[1:]) for z in _inputs(b * t, h, hkv, d))
    want = _run(q, k, v, dout)

    def gap(z):                                                       # rows apart, heads together
        return torch.empty(*z.shape[:2], z.shape[2] + 3, z.shape[3], dtype=z.dtype, device="cuda")[:, :, 1:1 + z.shape[2]].copy_(z)

    def heads_first(z):                                               # memory [b, h, t, d]
        return z.transpose(1, 2).contiguous().transpose(1, 2)

    def off(z):                                                       # base not 16-byte aligned
        return torch.empty(z.numel() + 1, dtype=z.dtype, device="cuda")[1:].view(z.shape).copy_(z)

    def columns(z):                                                   # last dimension not contiguous
        return z.transpose(-1, -2).contiguous().transpose(-1, -2)

    for change in (gap, heads_first, off, columns):
        for a, w in zip(_run(*(change(z) for z in (q, k, v, dout))), want):
            assert torch.equal(a, w), change.__name__
    # a gradient without strides of its own
    leaves = [z.clone().requires_grad_(True) for z in (q, k, v)]
    fa.causal_attention(*leaves).sum().backward()
    for a, w in zip([z.grad for z in leaves], _run(q, k, v, torch.ones_like(dout))[1:]):
        assert torch.equal(a, w)


@pytest.mark.parametrize("lead,h,hkv,d", [((2, 150), 4, 4, 64), ((2, 150), 4, 1, 128), ((333,), 6, 2, 32)])
def test_side_by_side_projection(lead, h, hkv, d):
    from bluefog_b200.ops import fused_attention as fa
    torch.manual_seed(3)
    qkv = torch.randn(*lead, (h + 2 * hkv) * d, device="cuda").to(torch.bfloat16).requires_grad_(True)
    out = fa.causal_self_attention(qkv, h, hkv)
    dout = torch.randn(out.shape, device="cuda").to(torch.bfloat16)
    (grad,) = torch.autograd.grad(out, qkv, dout)
    q, k, v = (z.detach() for z in fa._split(qkv, h, hkv))
    want = _run(q, k, v, dout)
    assert torch.equal(out, want[0])
    for g, w in zip(fa._split(grad, h, hkv), want[1:]):
        assert torch.equal(g, w)
    with torch.no_grad():
        assert torch.equal(fa.causal_self_attention(qkv, h, hkv), out)


def test_same_bits_in_every_run_on_any_stream_and_in_a_graph():
    from bluefog_b200.ops import fused_attention as fa
    q, k, v, dout = _inputs(900, 4, 2, 64)
    cu = _cu([300, 1, 599])
    want = _run(q, k, v, dout, cu_seqlens=cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, w in zip(_run(q, k, v, dout, cu_seqlens=cu), want):
            assert torch.equal(a, w)
    torch.cuda.current_stream().wait_stream(side)
    leaves = [z.clone().requires_grad_(True) for z in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.causal_attention(*leaves, cu_seqlens=cu)
        grads = torch.autograd.grad(out, leaves, dout)
    for new in (2, 1):
        with torch.no_grad():
            for z, src in zip(leaves, (q, k, v)):
                z.copy_(src / new)
        graph.replay()
    for a, w in zip([out, *grads], want):
        assert torch.equal(a, w)
    # other boundaries of the same count through the captured launches
    cu.copy_(_cu([10, 500, 200]))
    graph.replay()
    for a, w in zip([out, *grads], _run(q, k, v, dout, cu_seqlens=cu)):
        assert torch.equal(a, w)
    fa.check_sequences()


def test_boundaries_that_fall_are_reported_and_stay_in_bounds():
    from bluefog_b200.ops import fused_attention as fa
    q, k, v, dout = _inputs(300, 2, 2, 64)
    for bad in ([0, 200, 100, 300], [0, 100, 400], [0, -5, 300], [0, 2 ** 31 - 1, 7]):
        fa.check_sequences()
        _run(q, k, v, dout, cu_seqlens=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(IndexError):
            fa.check_sequences()


def test_gradient_against_differences():
    """The directional derivative of the fp64 forward pass by central differences against the kernels' gradients."""
    from bluefog_b200.ops import fused_attention as fa
    lengths = [140, 33]
    q, k, v, dout = _inputs(173, 2, 1, 64)
    grads = _run(q, k, v, dout, cu_seqlens=_cu(lengths))[1:]
    torch.manual_seed(9)
    steps = [torch.randn(z.shape, device="cuda", dtype=torch.float64) for z in (q, k, v)]
    h = 1e-5

    def loss(sign):
        a, b, c = (z.double() + sign * h * s for z, s in zip((q, k, v), steps))
        return (fa._plain(a, b, c, _cu(lengths), 1 / 8.0) * dout.double()).sum().item()

    want = (loss(1) - loss(-1)) / (2 * h)
    got = sum((g.double() * s).sum().item() for g, s in zip(grads, steps))
    _, tol = _oracle(q, k, v, dout, lengths, 1 / 8.0)
    bound = math.sqrt(sum((t * s).square().sum().item() for t, s in zip(tol[1:], steps)))   # independent roundings
    assert abs(got - want) <= 4 * bound + 1e-6 * abs(want), (got, want, bound)


def test_offsets_past_32_bits():
    """Key and value rows that start more than 2^31 elements into their tensors."""
    from bluefog_b200.ops import fused_attention as fa
    t, h, d = 34 * 1000, 1, 64
    stride = 65536                                                    # elements from token to token
    big = torch.empty(t * stride, dtype=torch.bfloat16, device="cuda").view(t, stride)
    lengths = [t - 150, 150]
    small = torch.randn(t, 3 * d, device="cuda").to(torch.bfloat16)
    big[:, :3 * d] = small
    with torch.no_grad():
        out = fa.causal_attention(*(big[:, i * d:(i + 1) * d].unsqueeze(1) for i in range(3)), cu_seqlens=_cu(lengths))
        want = fa.causal_attention(*(small[:, i * d:(i + 1) * d].unsqueeze(1) for i in range(3)), cu_seqlens=_cu(lengths))
    assert torch.equal(out, want)


def test_gradients_of_gradients_are_refused():
    from bluefog_b200.ops import fused_attention as fa
    q, k, v, dout = _inputs(60, 2, 2, 64)
    q.requires_grad_(True)
    qkv = torch.randn(60, 3 * 128, device="cuda").to(torch.bfloat16).requires_grad_(True)
    for leaf, out in ((q, fa.causal_attention(q, k, v)), (qkv, fa.causal_self_attention(qkv, 2))):
        (g,) = torch.autograd.grad(out, leaf, dout.view(out.shape), create_graph=True)
        with pytest.raises(RuntimeError, match="only once"):
            g.float().sum().backward()


def test_gradients_where_few_keys_share_the_weight():
    """In sequences of eight tokens delta is as large as the dP that it is subtracted from, so a delta from the rounded result
    would show.  A rounding to bf16 is off by 2^-8 sqrt((1 - 1/4) / (2 ln 2) / 3) = 0.00166 of the value in the quadratic mean over
    mantissas; dq and dk may have three of them (dS, P through delta, their own).  A delta from the rounded result adds two."""
    q, k, v, dout = _inputs(8 * 64, 8, 8, 64, seed=3)
    cu = _cu([8] * 64)
    got = _run(q, k, v, dout, cu_seqlens=cu)
    want, _ = _oracle(q, k, v, dout, [8] * 64, 1 / 8.0)
    for name, a, b in zip(("dq", "dk"), got[1:3], want[1:3]):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= math.sqrt(3) * 0.00166, (name, off)


def test_calls_one_right_behind_the_other():
    """The backward launches start beside the ones in front of them: calls in a row, whose memory is used again at once."""
    cases = [(_inputs(900, 8, 2, 64), _cu([500, 1, 300])), (_inputs(300, 4, 4, 64), None), (_inputs(513, 8, 1, 128), _cu([13, 500])),
             (_inputs(130, 2, 1, 32), _cu([0, 130]))]
    want = []
    for x, cu in cases:
        want.append(_run(*x, cu_seqlens=cu))
        torch.cuda.synchronize()
    got = [_run(*cases[i][0], cu_seqlens=cases[i][1]) for _ in range(10) for i in range(4)]
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 4])), i
    for _ in range(5):                                                # results dropped at once
        for x, cu in cases:
            _run(*x, cu_seqlens=cu)
    for i, (x, cu) in enumerate(cases):
        assert all(torch.equal(a, b) for a, b in zip(_run(*x, cu_seqlens=cu), want[i]))
