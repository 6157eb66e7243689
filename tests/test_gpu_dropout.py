"""The dropout kernel against the generator and the formula in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def philox(counter, key):
    """Philox4x32-10 of one counter in Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ c[3] ^ k[1], a % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def kept(count, p, seed, step, site):
    out = np.empty(((count + 7) // 8, 8), dtype=bool)
    for g in range(out.shape[0]):
        words = philox((g % 2 ** 32, (g >> 32) | site << 16, step % 2 ** 32, (step >> 32) % 2 ** 32), (seed % 2 ** 32, (seed >> 32) % 2 ** 32))
        for i in range(8):
            out[g, i] = (words[i // 2] >> 16 * (i % 2)) % 65536 >= round(65536 * p)
    return torch.from_numpy(out.reshape(-1)[:count])


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("shape,p,seed,step,site,residual", [
    ((1,), 0.5, 0, 0, 0, True), ((7,), 0.1, 1, 2, 3, False), ((8,), 0.9, -1, -1, 65535, True), ((3, 5, 11), 0.3, 2 ** 63 - 1, 2 ** 40 + 3, 1, True),
    ((37, 771), 0.1, 123456789012, 7, 0, True), ((64, 264), 0.0, 5, 5, 5, False), ((300,), 1.0, 9, 9, 9, True)])
def test_mask_values_and_gradients(dtype, shape, p, seed, step, site, residual):
    from bluefog_b200.ops import fused_dropout
    torch.manual_seed(1)
    x, r, dy = (torch.randn(shape, device="cuda").to(dtype) for _ in range(3))
    x.requires_grad_(True)
    r = r.requires_grad_(True) if residual else None
    key = torch.tensor([seed, step], device="cuda")
    assert fused_dropout._eligible(x)
    y = fused_dropout.dropout_add(x, r, p, key, site)
    y.backward(dy)
    keep = kept(x.numel(), p, seed, step, site).view(shape).cuda()
    q = round(65536 * p) / 65536
    factor = keep.double() / (1 - q) if q < 1 else torch.zeros(shape, device="cuda", dtype=torch.float64)
    u = HALF_STEP[dtype]
    # x * factor and the sum are rounded in fp32 (the factor itself too), the result once to the type
    fine = 3 * 2.0 ** -24
    scaled = factor * x.detach().double()
    want = scaled + (r.detach().double() if residual else 0)
    tol = u * want.abs() * (1 + fine) + fine * (scaled.abs() + want.abs()) + 2.0 ** -24 * (dtype == torch.float16)
    assert ((y.double() - want).abs() <= tol).all()
    want = factor * dy.double()
    assert ((x.grad.double() - want).abs() <= u * want.abs() + fine * want.abs() + 2.0 ** -24 * (dtype == torch.float16)).all()
    assert ((x.grad == 0) | keep).all()
    if residual:
        assert torch.equal(r.grad, dy)
    # the same mask on the CPU
    cpu = fused_dropout.dropout_add(torch.ones(shape), None, p, key.cpu(), site)
    assert torch.equal(cpu != 0, keep.cpu())


def test_what_is_dropped_is_zero_whatever_it_holds():
    from bluefog_b200.ops import fused_dropout
    x = torch.full((1000,), math.nan, device="cuda")
    y = fused_dropout.dropout_add(x, torch.ones_like(x), 0.5, fused_dropout.new_key(4, "cuda"))
    keep = kept(1000, 0.5, 4, 0, 0).cuda()
    assert y[keep].isnan().all() and (y[~keep] == 1).all()


def test_strides_and_alignment():
    from bluefog_b200.ops import fused_dropout
    key = fused_dropout.new_key(11, "cuda")
    x, r = (torch.randn(60, 50, device="cuda").to(torch.bfloat16) for _ in range(2))
    want = fused_dropout.dropout_add(x, r, 0.2, key)
    off = torch.empty(3001, dtype=x.dtype, device="cuda")[1:].view(60, 50).copy_(x)
    for a, b in ((x.t().contiguous().t(), r), (off, r), (x, r.t().contiguous().t())):
        assert torch.equal(fused_dropout.dropout_add(a, b, 0.2, key), want)


def test_captured_graph_draws_new_masks_when_its_key_advances():
    from bluefog_b200.ops import fused_dropout
    key = fused_dropout.new_key(21, "cuda")
    x = torch.ones(5000, device="cuda", requires_grad=True)
    fused_dropout.dropout_add(x, None, 0.5, key).sum().backward()      # warm-up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        now = key.clone()
        y = fused_dropout.dropout_add(x, None, 0.5, now, site=3)
        (dx,) = torch.autograd.grad(y.sum(), x)
        key[1] += 1
    for step in range(3):
        graph.replay()
        keep = kept(5000, 0.5, 21, step, 3).cuda()
        assert torch.equal(y != 0, keep) and torch.equal(dx != 0, keep)


def test_key_that_changed_before_the_backward_pass_is_reported():
    from bluefog_b200.ops import fused_dropout
    key = fused_dropout.new_key(1, "cuda")
    x = torch.ones(64, device="cuda", requires_grad=True)
    y = fused_dropout.dropout_add(x, None, 0.5, key)
    key[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_share_of_dropped_elements():
    from bluefog_b200.ops import fused_dropout
    n = 1 << 22
    y = fused_dropout.dropout_add(torch.ones(n, device="cuda"), None, 0.1, fused_dropout.new_key(77, "cuda"))
    share = (y == 0).float().mean().item()
    q = round(6553.6) / 65536
    assert abs(share - q) <= 5 * math.sqrt(q * (1 - q) / n)            # five standard deviations of a binomial share
