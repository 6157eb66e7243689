"""GPT-2 (decoder-only transformer) with Hugging Face parameter names.

Used by the GPT-2-medium data-parallel workload (24 layers, d_model 1024, 16 heads, vocab
50257, sequence 1024).  The reference has no transformer code; the library only needs a
single-GPU model whose parameters the distributed optimizers average.  Linear layers run on
the hand-written tcgen05 GEMM when the activations are bf16 (``use_b200_gemm``), LayerNorm on the
row-in-registers kernels of ``bluefog_b200.ops.fused_ln``; attention uses PyTorch's fused
scaled-dot-product attention, or with ``use_b200_attention`` the kernels of ``bluefog_b200.ops.fused_attention``.

Beyond the original model, all off by default: ``n_kv_head`` (grouped heads), ``mlp="swiglu"`` / ``"geglu"`` (a gated
feed-forward block without biases, ``gemm.gated_mlp``), ``dropout`` (of the embedding and of both sub-layers' outputs,
``fused_dropout.dropout_add``) and ``forward(..., cu_seqlens=)`` (documents packed one after the other: attention stays
inside a document, positions count along the row).
"""
import math

import os

import torch
import torch.nn as nn
import torch.nn.functional as F

from bluefog_b200.ops import fused_attention, fused_dropout, fused_embedding, gemm as _gemm
from bluefog_b200.ops.fused_ln import LayerNorm


class B200Linear(nn.Linear):
    """nn.Linear ([out, in] weight) that routes bf16 CUDA inputs to the tcgen05 GEMM."""

    def __init__(self, in_features, out_features, bias=True, use_b200_gemm=True, act=None):
        super().__init__(in_features, out_features, bias=bias)
        self.use_b200_gemm = use_b200_gemm

    def forward(self, x, residual=None):
        """``residual`` (same shape as the output) is added to the result; on the kernel path inside the GEMM epilogue."""
        if self.use_b200_gemm and x.is_cuda and x.dtype == torch.bfloat16 and self.weight.dtype == torch.bfloat16:
            from bluefog_b200.ops import gemm
            if gemm.available() and self.in_features % 8 == 0:
                res2d = None if residual is None else residual.reshape(-1, self.out_features)
                y = gemm.linear(x.reshape(-1, self.in_features), self.weight, self.bias, res2d)
                return y.view(*x.shape[:-1], self.out_features)
        y = F.linear(x, self.weight, self.bias)
        return y if residual is None else y + residual


class Attention(nn.Module):
    def __init__(self, d_model, n_head, use_b200_gemm, n_kv_head=None, use_b200_attention=False):
        super().__init__()
        self.n_head = n_head
        self.n_kv_head = n_head if n_kv_head is None else n_kv_head
        if self.n_kv_head < 1 or d_model % n_head != 0 or n_head % self.n_kv_head != 0:
            raise ValueError("d_model %d, n_head %d and n_kv_head %d do not divide" % (d_model, n_head, self.n_kv_head))
        self.use_b200_attention = use_b200_attention
        self.c_attn = B200Linear(d_model, (n_head + 2 * self.n_kv_head) * (d_model // n_head), use_b200_gemm=use_b200_gemm)
        self.c_proj = B200Linear(d_model, d_model, use_b200_gemm=use_b200_gemm)

    def forward(self, x, residual=None, cu_seqlens=None):
        b, t, c = x.shape
        if self.use_b200_attention or self.n_kv_head != self.n_head or cu_seqlens is not None:
            y = fused_attention.causal_self_attention(self.c_attn(x), self.n_head, self.n_kv_head, cu_seqlens=cu_seqlens)
            return self.c_proj(y.reshape(b, t, c), residual)
        q, k, v = self.c_attn(x).split(c, dim=2)
        shape = (b, t, self.n_head, c // self.n_head)
        q, k, v = (z.view(shape).transpose(1, 2) for z in (q, k, v))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.c_proj(y.transpose(1, 2).reshape(b, t, c), residual)


class MLP(nn.Module):
    def __init__(self, d_model, use_b200_gemm):
        super().__init__()
        self.c_fc = B200Linear(d_model, 4 * d_model, use_b200_gemm=use_b200_gemm)
        self.c_proj = B200Linear(4 * d_model, d_model, use_b200_gemm=use_b200_gemm)

    def forward(self, x, residual=None):
        # BLUEFOG_B200_MLP_FUSION=0 keeps the GELU a kernel of its own between the two GEMMs
        if (self.c_fc.use_b200_gemm and x.is_cuda and x.dtype == torch.bfloat16
                and os.environ.get("BLUEFOG_B200_MLP_FUSION", "1") != "0"):
            from bluefog_b200.ops import gemm
            res2d = None if residual is None else residual.reshape(-1, residual.shape[-1])
            y = gemm.mlp_gelu(x.reshape(-1, x.shape[-1]), self.c_fc.weight, self.c_fc.bias, self.c_proj.weight,
                              self.c_proj.bias, res2d)
            return y.view(*x.shape[:-1], y.shape[-1])
        return self.c_proj(F.gelu(self.c_fc(x), approximate="tanh"), residual)


class GatedMLP(nn.Module):
    """``c_proj(act(gate) * up)`` with gate and up in one weight ``c_fc`` [2 inner, d_model]; no biases."""

    def __init__(self, d_model, use_b200_gemm, act, inner=None):
        super().__init__()
        self.act = act
        # two thirds of four times d_model, the parameters of the ungated block, on a multiple of 64
        inner = (8 * d_model // 3 + 63) // 64 * 64 if inner is None else inner
        self.c_fc = B200Linear(d_model, 2 * inner, bias=False, use_b200_gemm=use_b200_gemm)
        self.c_proj = B200Linear(inner, d_model, bias=False, use_b200_gemm=use_b200_gemm)

    def forward(self, x, residual=None):
        if self.c_fc.use_b200_gemm and x.dtype == self.c_fc.weight.dtype:
            return _gemm.gated_mlp(x, self.c_fc.weight, self.c_proj.weight, act=self.act, residual=residual)
        gate, up = self.c_fc(x).chunk(2, -1)
        gate = F.silu(gate) if self.act == "silu" else F.gelu(gate, approximate="tanh")
        return self.c_proj(gate * up, residual)


class Block(nn.Module):
    def __init__(self, d_model, n_head, use_b200_gemm, n_kv_head=None, mlp="gelu", use_b200_attention=False):
        super().__init__()
        self.ln_1 = LayerNorm(d_model)
        self.attn = Attention(d_model, n_head, use_b200_gemm, n_kv_head, use_b200_attention)
        self.ln_2 = LayerNorm(d_model)
        if mlp not in ("gelu", "swiglu", "geglu"):
            raise ValueError("mlp has to be 'gelu', 'swiglu' or 'geglu', got %r" % (mlp,))
        self.mlp = (MLP(d_model, use_b200_gemm) if mlp == "gelu"
                    else GatedMLP(d_model, use_b200_gemm, "silu" if mlp == "swiglu" else "gelu"))

    def forward(self, x, cu_seqlens=None, drop=None):
        if drop is not None:
            # drop(y, x, which): dropout of a sub-layer's output joined with the residual stream
            h, x = self.ln_1.with_residual(x)
            x = drop(self.attn(h, None, cu_seqlens), x, 0)
            h, x = self.ln_2.with_residual(x)
            return drop(self.mlp(h), x, 1)
        # the residual stream joins each sub-layer's output inside the last GEMM's epilogue
        # and its two gradients (through the LayerNorm, and past it) meet inside the LayerNorm backward kernel
        h, x = self.ln_1.with_residual(x)
        x = self.attn(h, x, cu_seqlens)
        h, x = self.ln_2.with_residual(x)
        return self.mlp(h, x)


class GPT2(nn.Module):
    def __init__(self, vocab_size=50257, n_positions=1024, d_model=768, n_layer=12, n_head=12,
                 use_b200_gemm=True, n_kv_head=None, mlp="gelu", dropout=0.0, use_b200_attention=False):
        super().__init__()
        if not 0.0 <= dropout < 1.0:
            raise ValueError("dropout has to lie in [0, 1), got %r" % (dropout,))
        self.wte = nn.Embedding(vocab_size, d_model)
        self.wpe = nn.Embedding(n_positions, d_model)
        self.h = nn.ModuleList([Block(d_model, n_head, use_b200_gemm, n_kv_head, mlp, use_b200_attention) for _ in range(n_layer)])
        self.ln_f = LayerNorm(d_model)
        self.use_b200_gemm = use_b200_gemm
        self.dropout = dropout
        if dropout > 0.0:
            # [seed, step]; part of the state, so that a resumed run goes on with the masks it would have drawn.  Ranks may
            # take it from one another by a broadcast: each draws masks of its own from it (rank_key).
            self.register_buffer("dropout_key", fused_dropout.new_key(torch.initial_seed() % 2 ** 62))
        self.apply(self._init)
        for name, p in self.named_parameters():
            if name.endswith("c_proj.weight"):
                nn.init.normal_(p, mean=0.0, std=0.02 / math.sqrt(2 * n_layer))

    @staticmethod
    def _init(m):
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)

    def forward(self, idx, targets=None, cu_seqlens=None):
        """Logits [b, t, vocab], or the mean cross-entropy when ``targets`` is given.  ``cu_seqlens``: boundaries of packed
        documents in the b * t tokens of ``idx`` (int32, see ``fused_attention``)."""
        b, t = idx.shape
        x = fused_embedding.token_position_embedding(idx, self.wte.weight, self.wpe.weight)   # wte[idx] + wpe[:t]
        key = None
        if self.dropout > 0.0 and self.training:
            key = fused_dropout.rank_key(self.dropout_key)      # the backward pass reads this step's key, the buffer goes on
            self.dropout_key[1] += 1
            x = fused_dropout.dropout_add(x, None, self.dropout, key)
        for i, block in enumerate(self.h):
            drop = None
            if key is not None:
                def drop(y, residual, which, site=2 * i + 1):
                    return fused_dropout.dropout_add(y, residual, self.dropout, key, site + which)
            x = block(x, cu_seqlens, drop)
        x = self.ln_f(x)
        w = self.wte.weight                        # tied output embedding, [vocab, d_model]
        vocab = w.shape[0]
        pad = (-vocab) % 64 if x.is_cuda else 0
        if pad:
            # 50257 output columns make every GEMM of the classifier (forward, both gradients) run with
            # odd leading dimensions; the product is taken against the matrix padded to a multiple of
            # 64 rows and the surplus logits are set to -inf, which leaves loss and gradients unchanged
            w = F.pad(w, (0, 0, 0, pad))
        x2 = x.reshape(b * t, x.shape[-1])
        logits = None
        if self.use_b200_gemm and x2.is_cuda and x2.dtype == torch.bfloat16 and w.dtype == torch.bfloat16:
            from bluefog_b200.ops import gemm
            if gemm.available():
                logits = gemm.linear(x2, w)
        if logits is None:
            logits = F.linear(x2, w)
        if pad:
            logits[:, vocab:] = float("-inf")
        if targets is None:
            return logits[:, :vocab].reshape(b, t, vocab)
        from bluefog_b200.ops.fused_ce import cross_entropy
        return cross_entropy(logits, targets.reshape(-1))


def gpt2_small(**kw):
    return GPT2(d_model=768, n_layer=12, n_head=12, **kw)


def gpt2_medium(**kw):
    return GPT2(d_model=1024, n_layer=24, n_head=16, **kw)
