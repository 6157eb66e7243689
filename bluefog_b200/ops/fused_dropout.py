"""Dropout from a counter-based generator, joined with the residual stream (``csrc/cuda/dropout_kernels.cu``).

``dropout_add(x, residual, p, key)`` is ``residual + keep * x / (1 - p)``.  Which elements are kept is a function of the
key (int64 ``[seed, step]`` on the device of x), the ``site`` (a number below 65536 that tells the layers of one step
apart) and the element's place in x, so no mask is stored: the backward pass computes it again, and the same call gives
the same mask on every device, in every type.  The key is read on the device: a captured graph whose key is advanced
between (or inside) replays draws new masks.  The key must not change between a forward pass and its backward pass
(autograd reports it); keep one and hand out copies, as ``models/gpt2.py`` does.  Ranks that start from one another's state
(``broadcast_parameters(model.state_dict())``) hold the same key: ``rank_key`` gives each of them a copy of its own.

Element i takes the 16-bit word i % 8 of block i // 8 of Philox4x32-10 (Salmon et al., SC 2011) and is dropped if that is
below ``round(65536 p)``; p is thereby rounded to a multiple of 2^-16 and the factor uses the rounded value.  Dropped
elements are zero whatever x holds.  CUDA tensors in fp32, fp16 or bf16 take the kernel, the arithmetic is fp32; the rest
takes the same generator in PyTorch's operators.  Forward-mode differentiation of the kernel is an error.  The reference has
no dropout of its own.
"""
import torch

from bluefog_b200.common.basics import get_basics

_b = get_basics()


def new_key(seed, device=None):
    """A key for ``dropout_add``: ``[seed, 0]``; add to its second element from step to step."""
    return torch.tensor([seed, 0], dtype=torch.int64, device=device)


def rank_key(key):
    """A copy of ``key`` for this rank's masks: the seed plus a multiple of the rank, so rank 0 (and a process that has not called
    ``init``) draws those of the key itself.  The multiple is 2^64 over the golden ratio: no two ranks with small seeds of their
    own can meet."""
    rank = _b.rank() if _b.is_initialized() else 0
    own = key.clone()
    if rank != 0:
        own[0] += (rank * 0x9E3779B97F4A7C15 + 2 ** 63) % 2 ** 64 - 2 ** 63      # wraps, as the addition does
    return own


def _eligible(x):
    return x.is_cuda and x.dtype in (torch.float32, torch.float16, torch.bfloat16) and x.numel() < 2 ** 51


def _keep(count, threshold, key, site):
    """The mask in PyTorch's integer operators (64-bit products wrap, which leaves both their words right)."""
    low = 0xFFFFFFFF
    index = torch.arange((count + 7) // 8, dtype=torch.int64, device=key.device)
    seed, step = key[0], key[1]
    c = [index & low, (index >> 32) | (site << 16), (step & low).expand_as(index), ((step >> 32) & low).expand_as(index)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack(c, 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:count] >= threshold


def dropout_add(x, residual, p, key, site=0):
    """``residual + dropout(x, p)`` (``residual`` may be None); ``key``: int64 ``[seed, step]``, see the module's notes."""
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout_add: p has to lie between 0 and 1, got %r" % (p,))
    if not x.is_floating_point():
        raise ValueError("dropout_add: x has to be a floating-point tensor")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("dropout_add: residual has to match x in shape, type and device")
    if key.dtype != torch.int64 or key.shape != (2,) or key.device != x.device:
        raise ValueError("dropout_add: key has to be int64 [seed, step] on the device of x")
    if not 0 <= site < 65536:
        raise ValueError("dropout_add: site has to lie in [0, 65536)")
    threshold = round(p * 65536)
    factor = 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0
    if x.numel() > 0 and _eligible(x):
        return _b.native.dropout_add(x, residual, threshold, factor, key, site)
    keep = _keep(x.numel(), threshold, key, site).view(x.shape)
    y = torch.where(keep, x * factor, torch.zeros((), dtype=x.dtype, device=x.device))
    return y if residual is None else y + residual
