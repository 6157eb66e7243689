"""Causal attention with grouped heads over packed sequences on the tcgen05 kernels of ``csrc/cuda/attn_tcgen05.cu``.

``causal_attention(q, k, v)`` takes q ``[..., T, H, D]`` and k, v ``[..., T, Hkv, D]`` (H a multiple of Hkv: query head h
reads key head ``h * Hkv // H``); ``causal_self_attention(qkv, n_head, n_kv_head)`` takes the three side by side in one
matrix ``[..., T, (H + 2 Hkv) D]``, as a fused projection leaves them, and hands its backward pass one gradient of that
shape.  Both return ``[..., T, H, D]``: position i attends to the positions up to i of its own sequence.

Without ``cu_seqlens`` every row of T tokens is one sequence.  With it (int32 ``[B + 1]`` on the inputs' device, starting
at 0 and never falling) all tokens together, in order, hold sequences of different lengths: sequence b is
``[cu_seqlens[b], cu_seqlens[b + 1])`` and may be empty; tokens behind the last one belong to none, and their results and
gradients are zero whatever they hold.  The lengths stay on the device.  The kernels take the first boundary as 0, clip
boundaries that fall or reach past the last token, and ``check_sequences`` reports them.

bf16 CUDA tensors with D a multiple of 8 up to 128 take the kernels, forward and backward, with any row spacing that is
a multiple of 16 bytes; everything else (CPU, fp32, fp16, other widths, scales that fp32 cannot hold, 2^30 tiles of 128
rows and a head) takes PyTorch's operators, sequence by sequence.  Results and gradients are the same in every run.  As in
a softmax written out, a weight of zero does not hide an infinite or NaN value of a later position of the same sequence:
earlier positions may become NaN.  Before a forward and backward pass is captured into a graph, drop eager results of the
same leaves: autograd would join their stream with the captured one, which PyTorch answers with an error or worse.
Gradients of gradients and forward-mode differentiation of the kernels are errors.  The reference has no attention code;
``models/gpt2.py`` calls this.
"""
import math

import torch
import torch.nn.functional as F

from bluefog_b200.common.basics import get_basics

_b = get_basics()


def _eligible(t, d):
    """Whether the kernels take ``t`` (q, or q, k and v side by side) with heads of width ``d``."""
    return (t.is_cuda and t.dtype == torch.bfloat16 and d % 8 == 0 and 8 <= d <= 128 and t.numel() // d < 2 ** 31 - 256
            and _b.native.gemm_supported())


def _fits(lead, heads, batch):
    """Whether tokens [*lead] with this many query heads, in ``batch`` packed sequences or one per row (None), stay within the
    31 bits that the kernels' grids and row coordinates have: 128-row tiles times heads, twice in the backward pass."""
    tokens = math.prod(lead)
    tiles = tokens // lead[-1] * ((lead[-1] + 127) // 128) if batch is None else tokens // 128 + batch + 1
    return tokens < 2 ** 31 - 256 and tiles * heads < 2 ** 30


def _takes(t, d, inner, heads, cu, scale):
    """Whether the kernels take the call, ``inner`` trailing dimensions of t being a row; scales are fp32 numbers there, and so is
    their product with log2 e."""
    if not (2.0 ** -126 <= scale <= 2.0 ** 126 and _eligible(t, d)):
        return False
    if t.numel() < 2 ** 30 and (cu is None or cu.numel() * heads < 2 ** 28):
        return True                                                   # at most a tile per token and boundary, which takes less time to see
    return _fits(t.shape[:-inner], heads, None if cu is None else cu.numel() - 1)


def _split(qkv, h, hkv):
    d = qkv.shape[-1] // (h + 2 * hkv)
    lead = qkv.shape[:-1]
    return (qkv[..., :h * d].view(*lead, h, d), qkv[..., h * d:(h + hkv) * d].view(*lead, hkv, d),
            qkv[..., (h + hkv) * d:].view(*lead, hkv, d))


def _plain(q, k, v, cu, scale):
    """The same with PyTorch's operators; q [.., T, H, D]."""
    group = q.shape[-2] // k.shape[-2]

    def one(a, b, c):
        a, b, c = (z.transpose(-3, -2) for z in (a, b.repeat_interleave(group, -2), c.repeat_interleave(group, -2)))
        return F.scaled_dot_product_attention(a, b, c, is_causal=True, scale=scale).transpose(-3, -2)

    if cu is None:
        return one(q, k, v).contiguous()
    shape = q.shape
    q, k, v = (z.reshape(-1, *z.shape[-2:]) for z in (q, k, v))
    ends = cu.tolist()
    if ends[0] != 0 or any(a > b for a, b in zip(ends, ends[1:])) or ends[-1] > q.shape[0]:
        raise ValueError("cu_seqlens has to start at 0, never fall and stay within the %d tokens" % q.shape[0])
    parts = [one(q[a:b], k[a:b], v[a:b]) for a, b in zip(ends, ends[1:]) if b > a]
    parts.append(torch.zeros_like(q[ends[-1]:]))
    return torch.cat(parts).reshape(shape)


def _check(h, hkv, d, device, cu, scale):
    if h < 1 or hkv < 1 or h % hkv != 0:
        raise ValueError("attention: the number of query heads (%d) has to be a multiple of the key heads' (%d)" % (h, hkv))
    if d < 1:
        raise ValueError("attention: heads without columns")
    if cu is not None and (cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 2 or cu.device != device):
        raise ValueError("cu_seqlens has to be an int32 vector of at least two boundaries on the device of the inputs")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (0.0 < scale < math.inf):
        raise ValueError("attention: scale has to be positive and finite")
    return scale


def causal_attention(q, k, v, cu_seqlens=None, scale=None):
    """``softmax(scale * q @ k.T, causal) @ v`` per head and sequence; scale defaults to ``1 / sqrt(D)``."""
    if not (q.dim() == k.dim() == v.dim() and q.dim() in (3, 4) and k.shape == v.shape and q.shape[:-2] == k.shape[:-2]
            and q.shape[-1] == k.shape[-1]):
        raise ValueError("causal_attention: q [.., T, H, D], k and v [.., T, Hkv, D] with one or two leading dimensions; got %s, %s, %s"
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not (q.device == k.device == v.device and q.dtype == k.dtype == v.dtype):
        raise ValueError("causal_attention: q, k and v have to share a device and a type")
    scale = _check(q.shape[-2], k.shape[-2], q.shape[-1], q.device, cu_seqlens, scale)
    if q.numel() == 0:
        return q + (k.sum() + v.sum()) * 0
    if not _takes(q, q.shape[-1], 2, q.shape[-2], cu_seqlens, scale):
        return _plain(q, k, v, cu_seqlens, scale)
    return _b.native.causal_attention(q, k, v, None if cu_seqlens is None else cu_seqlens.contiguous(), scale)


def causal_self_attention(qkv, n_head, n_kv_head=None, cu_seqlens=None, scale=None):
    """``causal_attention`` of the columns [q | k | v] of ``qkv`` [.., T, (n_head + 2 n_kv_head) D]."""
    hkv = n_head if n_kv_head is None else n_kv_head
    if qkv.dim() not in (2, 3) or n_head < 1 or hkv < 1 or qkv.shape[-1] % (n_head + 2 * hkv) != 0:
        raise ValueError("causal_self_attention: %d columns are not (%d + 2 * %d) heads of equal width in a [.., T, columns] tensor"
                         % (qkv.shape[-1], n_head, hkv))
    scale = _check(n_head, hkv, qkv.shape[-1] // (n_head + 2 * hkv), qkv.device, cu_seqlens, scale)
    d = qkv.shape[-1] // (n_head + 2 * hkv)
    if qkv.numel() == 0 or not _takes(qkv, d, 1, n_head, cu_seqlens, scale):
        return causal_attention(*_split(qkv, n_head, hkv), cu_seqlens, scale)
    return _b.native.causal_self_attention(qkv, n_head, hkv, None if cu_seqlens is None else cu_seqlens.contiguous(), scale)


def check_sequences(device=None):
    """Raises IndexError if a kernel on ``device`` (default: the current one) since the last check was given ``cu_seqlens``
    that do not start at 0, fall or reach past the last token, and RuntimeError if a kernel gave up waiting.  Waits for the device, all streams."""
    index = torch.device(device).index if device is not None else None
    status = _b.native.attn_status(torch.cuda.current_device() if index is None else index)
    if status & 1:
        raise RuntimeError("an attention kernel ran into its time limit")
    if status & 2:
        raise IndexError("cu_seqlens do not start at 0, fall or reach past the last token")
