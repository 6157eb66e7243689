"""Cases that measure the transformer-block operators of ``bluefog_b200.ops``: causal attention with grouped heads
over packed documents, the gated feed-forward block, and dropout joined with the residual stream.

``run`` computes a case in plain PyTorch operations (fp32 inside, one rounding at the end) while ``own`` is false, and
through this library's entry points while it is true; both take the state that ``prepare`` makes.  ``exact`` gives the
same outputs from the definitions in fp64.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # ---- attention -------------------------------------------------------------------------------------------
        # scoring one short prompt with GPT-2 small's heads: a launch-latency call
        dict(name="attn_fwd_short", op="attn", train=False, lengths="37", heads=12, kv_heads=12, dim=64, packed=True, dense=True),
        # evaluating GPT-2 medium on a full batch of the benchmark (8 x 1024 tokens), no gradients
        dict(name="attn_fwd_gpt2_medium", op="attn", train=False, lengths=",".join(["1024"] * 8), heads=16, kv_heads=16, dim=64,
             packed=True, dense=True),
        # the attention of one GPT-2 medium layer in the benchmark's training step
        dict(name="attn_train_gpt2_medium", op="attn", train=True, lengths=",".join(["1024"] * 8), heads=16, kv_heads=16, dim=64,
             packed=True, dense=True),
        # documents of very different lengths packed into one row, four query heads to a key head, some padding behind them
        dict(name="attn_train_packed", op="attn", train=True, lengths="1531,1,700,2999,64,129,0,1022,1500", heads=16, kv_heads=4,
             dim=64, packed=True, dense=False, padding=246),
        # one long document, wide heads, grouped
        dict(name="attn_train_long", op="attn", train=True, lengths="8192", heads=16, kv_heads=4, dim=128, packed=False, dense=True),
        # ---- gated feed-forward block ----------------------------------------------------------------------------
        # a handful of tokens through the block of a GPT-2 medium sized model: the weights are what is read
        dict(name="gated_fwd_few_rows", op="gated", train=False, rows=8, width=1024, inner=2752, act="silu", residual=True),
        # one layer of GPT-2 medium's training step with the gated block in the place of the GELU one
        dict(name="gated_train_gpt2_medium", op="gated", train=True, rows=8192, width=1024, inner=2752, act="silu", residual=True),
        # odd sizes and the GELU gate: a partial batch, widths that fill no tile
        dict(name="gated_train_odd", op="gated", train=True, rows=1537, width=776, inner=2056, act="gelu", residual=False),
        # a wide block on the largest batch
        dict(name="gated_train_wide", op="gated", train=True, rows=16384, width=2048, inner=5504, act="silu", residual=True),
        # ---- dropout ---------------------------------------------------------------------------------------------
        # the embedding dropout of a short prompt in training: a launch-latency call, odd row length
        dict(name="dropout_short", op="dropout", train=True, rows=37, width=771, type="fp32", p=0.1, residual=False),
        # residual dropout of one GPT-2 medium layer in the benchmark's training step
        dict(name="dropout_gpt2_medium", op="dropout", train=True, rows=8192, width=1024, type="bf16", p=0.1, residual=True),
        # the same on activations far larger than the cache
        dict(name="dropout_wide", op="dropout", train=True, rows=65536, width=2048, type="bf16", p=0.2, residual=True),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "gated", "dropout"])
    if op == "attn":
        kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
        heads = kv_heads * rng.choice([g for g in (1, 2, 4, 8) if kv_heads * g <= 16])
        dim = rng.choice([32, 64, 64, 80, 128, 128])
        train = rng.random() < 0.6
        packed = rng.random() < 0.6
        if rng.random() < 0.4:
            t, b = _log_between(rng, 1, 4096), _log_between(rng, 1, 8)
            b = max(1, min(b, 8192 // t))
            return dict(op="attn", train=train, lengths=",".join([str(t)] * b), heads=heads, kv_heads=kv_heads, dim=dim,
                        packed=packed, dense=True)
        docs = rng.randint(1, 12)
        lengths = [0 if rng.random() < 0.05 else _log_between(rng, 1, 4096 if docs <= 6 else 1500) for _ in range(docs)]
        lengths[rng.randrange(docs)] += 1
        return dict(op="attn", train=train, lengths=",".join(str(n) for n in lengths), heads=heads, kv_heads=kv_heads, dim=dim,
                    packed=packed, dense=False, padding=rng.choice([0, 0, rng.randint(1, 300)]))
    if op == "gated":
        return dict(op="gated", train=rng.random() < 0.6, rows=_log_between(rng, 1, 16384), width=8 * _log_between(rng, 8, 256),
                    inner=8 * _log_between(rng, 16, 688), act=rng.choice(["silu", "gelu"]), residual=rng.random() < 0.5)
    return dict(op="dropout", train=rng.random() < 0.6, rows=_log_between(rng, 1, 65536), width=_log_between(rng, 8, 2048),
                type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), p=rng.choice([0.05, 0.1, 0.2, 0.5]), residual=rng.random() < 0.7)


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    train = case["train"]
    s = dict(case=case)
    if case["op"] == "attn":
        lengths = _lengths(case)
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        tokens = sum(lengths) + case.get("padding", 0)
        lead = (len(lengths), lengths[0]) if case["dense"] else (tokens,)
        if case["packed"]:
            s["qkv"] = normal(*lead, (heads + 2 * kv_heads) * dim).requires_grad_(train)
        else:
            s["q"] = normal(*lead, heads, dim).requires_grad_(train)
            s["k"] = normal(*lead, kv_heads, dim).requires_grad_(train)
            s["v"] = normal(*lead, kv_heads, dim).requires_grad_(train)
        if not case["dense"]:
            s["cu_seqlens"] = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
        if train:
            s["dout"] = normal(*lead, heads, dim)
    elif case["op"] == "gated":
        rows, width, inner = case["rows"], case["width"], case["inner"]
        s["x"] = normal(rows, width).requires_grad_(train)
        s["w_gate_up"] = normal(2 * inner, width, std=1.0 / math.sqrt(width)).requires_grad_(train)
        s["w_down"] = normal(width, inner, std=1.0 / math.sqrt(inner)).requires_grad_(train)
        s["residual"] = normal(rows, width).requires_grad_(train) if case["residual"] else None
        if train:
            s["dout"] = normal(rows, width)
    else:
        dtype = _TYPES[case["type"]]
        shape = (case["rows"], case["width"])
        s["x"] = normal(*shape, dtype=dtype).requires_grad_(train)
        s["residual"] = normal(*shape, dtype=dtype).requires_grad_(train) if case["residual"] else None
        s["key"] = torch.tensor([seed * 0x9E3779B1 + 12345, 3 + seed % 1000], dtype=torch.int64, device="cuda")
        if train:
            s["dout"] = normal(*shape, dtype=dtype)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------

def _plain_attention(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["packed"]:
        q, k, v = s["qkv"].split([heads * dim, kv_heads * dim, kv_heads * dim], dim=-1)
    else:
        q, k, v = s["q"], s["k"], s["v"]
    group = heads // kv_heads
    q = q.float().reshape(-1, kv_heads, group, dim)
    k, v = (z.float().reshape(-1, kv_heads, dim) for z in (k, v))
    tokens = q.shape[0]
    if case["dense"]:
        b, t = s["dout"].shape[:2] if case["train"] else s["qkv" if case["packed"] else "q"].shape[:2]
        q, k, v = q.view(b, t, kv_heads, group, dim), k.view(b, t, kv_heads, dim), v.view(b, t, kv_heads, dim)
    else:
        # the documents side by side, each padded to the longest
        cu = s["cu_seqlens"].long()
        t = max(_lengths(case))
        pos = torch.arange(t, device=cu.device)
        inside = pos < (cu[1:] - cu[:-1])[:, None]
        row = (cu[:-1, None] + pos).clamp(max=tokens - 1)
        q = q[row] * inside[:, :, None, None, None]
        k, v = (z[row] * inside[:, :, None, None] for z in (k, v))
    scores = torch.einsum("bikgd,bjkd->bkgij", q, k) * (1.0 / math.sqrt(dim))
    scores = scores.masked_fill(torch.ones(t, t, dtype=torch.bool, device=q.device).triu(1), -math.inf)
    e = (scores - scores.amax(-1, keepdim=True).detach()).exp()
    out = torch.einsum("bkgij,bjkd->bikgd", e / e.sum(-1, keepdim=True), v).reshape(q.shape[0], t, heads, dim)
    if not case["dense"]:
        out = torch.zeros(tokens, heads, dim, device=q.device).index_put((row[inside],), out[inside])
    out = out.to(torch.bfloat16)
    if not case["train"]:
        return [out]
    leaves = [s["qkv"]] if case["packed"] else [s["q"], s["k"], s["v"]]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def _plain_gated(s):
    case = s["case"]
    gate, up = (s["x"].float() @ s["w_gate_up"].float().t()).chunk(2, dim=1)
    if case["act"] == "silu":
        gate = gate / (1 + (-gate).exp())
    else:
        gate = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    out = (gate * up) @ s["w_down"].float().t()
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = out.to(torch.bfloat16)
    if not case["train"]:
        return [out]
    leaves = [s["x"], s["w_gate_up"], s["w_down"]] + ([s["residual"]] if s["residual"] is not None else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def _plain_round(c0, c1, c2, c3, k0, k1):
    # one round of Philox4x32; 64-bit products wrap, which leaves their low and high words as they should be
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    return ((b >> 32) & 0xFFFFFFFF) ^ c1 ^ k0, b & 0xFFFFFFFF, ((a >> 32) & 0xFFFFFFFF) ^ c3 ^ k1, a & 0xFFFFFFFF


def _plain_keep(key, count, threshold):
    seed, step = key[0], key[1]
    index = torch.arange((count + 7) // 8, device=key.device)
    c = (index & 0xFFFFFFFF, index >> 32, (step & 0xFFFFFFFF).expand_as(index), ((step >> 32) & 0xFFFFFFFF).expand_as(index))
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for r in range(10):
        c = _plain_round(*c, (k0 + r * 0x9E3779B9) & 0xFFFFFFFF, (k1 + r * 0xBB67AE85) & 0xFFFFFFFF)
    words = torch.stack(c, dim=1)
    return torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:count] >= threshold


def _plain_dropout(s):
    case = s["case"]
    x = s["x"]
    threshold = round(case["p"] * 65536)
    keep = _plain_keep(s["key"], x.numel(), threshold).view(x.shape)
    out = torch.where(keep, x.float() * (65536.0 / (65536 - threshold)), 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = out.to(x.dtype)
    if not case["train"]:
        return [out]
    leaves = [x] + ([s["residual"]] if s["residual"] is not None else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


# ---- the library's entry points ----------------------------------------------------------------------------------

def _own_attention(s):
    from bluefog_b200.ops import fused_attention
    case = s["case"]
    if case["packed"]:
        leaves = [s["qkv"]]
        out = fused_attention.causal_self_attention(s["qkv"], case["heads"], case["kv_heads"], cu_seqlens=s.get("cu_seqlens"))
    else:
        leaves = [s["q"], s["k"], s["v"]]
        out = fused_attention.causal_attention(*leaves, cu_seqlens=s.get("cu_seqlens"))
    if not case["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def _own_gated(s):
    from bluefog_b200.ops import gemm
    out = gemm.gated_mlp(s["x"], s["w_gate_up"], s["w_down"], act=s["case"]["act"], residual=s["residual"])
    if not s["case"]["train"]:
        return [out]
    leaves = [s["x"], s["w_gate_up"], s["w_down"]] + ([s["residual"]] if s["residual"] is not None else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def _own_dropout(s):
    from bluefog_b200.ops import fused_dropout
    out = fused_dropout.dropout_add(s["x"], s["residual"], s["case"]["p"], s["key"])
    if not s["case"]["train"]:
        return [out]
    leaves = [s["x"]] + ([s["residual"]] if s["residual"] is not None else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attention, "gated": _own_gated, "dropout": _own_dropout}[op](state)
    return {"attn": _plain_attention, "gated": _plain_gated, "dropout": _plain_dropout}[op](state)


def work(case):
    train = case["train"]
    if case["op"] == "attn":
        lengths = _lengths(case)
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        tokens = sum(lengths) + case.get("padding", 0)
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        # forward: two products; backward: the scores once more and four gradients' products
        flops = (14 if train else 4) * dim * heads * pairs
        q, kv = 2 * tokens * heads * dim, 2 * tokens * kv_heads * dim
        return {"bytes": (2 * q + 2 * kv) + ((2 * q + 2 * kv) if train else 0), "flops": flops}
    rows, width = case["rows"], case["width"]
    if case["op"] == "gated":
        inner = case["inner"]
        weights = 2 * 3 * width * inner
        x = 2 * rows * width
        moved = weights + x * (3 if case["residual"] else 2)
        if train:
            moved += weights + 2 * x
        return {"bytes": moved, "flops": (18 if train else 6) * rows * width * inner}
    size = 4 if case["type"] == "fp32" else 2
    streams = 2 + (1 if case["residual"] else 0) + (2 if train else 0)
    return {"bytes": streams * size * rows * width, "flops": 0}


# ---- the definitions in fp64 -------------------------------------------------------------------------------------

def _exact_attention(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["packed"]:
        flat = s["qkv"].detach().double().flatten(0, -2)
        q = flat[:, :heads * dim].reshape(-1, heads, dim)
        k = flat[:, heads * dim:(heads + kv_heads) * dim].reshape(-1, kv_heads, dim)
        v = flat[:, (heads + kv_heads) * dim:].reshape(-1, kv_heads, dim)
        lead = s["qkv"].shape[:-1]
    else:
        q, k, v = (s[n].detach().double().reshape(-1, s[n].shape[-2], dim) for n in "qkv")
        lead = s["q"].shape[:-2]
    out, dq, dk, dv = (torch.zeros_like(z) for z in (q, q, k, v))
    dout = s["dout"].double().reshape(q.shape) if case["train"] else None
    start = 0
    for n in _lengths(case):
        rows = slice(start, start + n)
        start += n
        for h in range(heads if n else 0):
            c = h * kv_heads // heads
            qh, kh, vh = q[rows, h], k[rows, c], v[rows, c]
            p = torch.softmax((qh @ kh.t() / dim ** 0.5).tril() + torch.full((n, n), -math.inf, device=q.device, dtype=q.dtype).triu(1), 1)
            out[rows, h] = p @ vh
            if dout is not None:
                do = dout[rows, h]
                dp = do @ vh.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / dim ** 0.5
                dv[rows, c] += p.t() @ do
                dq[rows, h] = ds @ kh
                dk[rows, c] += ds.t() @ qh
    out = out.reshape(*lead, heads, dim)
    if dout is None:
        return [out]
    if case["packed"]:
        return [out, torch.cat([z.flatten(1) for z in (dq, dk, dv)], 1).reshape(*lead, -1)]
    return [out, dq.reshape(*lead, heads, dim), dk.reshape(*lead, kv_heads, dim), dv.reshape(*lead, kv_heads, dim)]


def _exact_gated(s):
    case = s["case"]
    inner = case["inner"]
    x, wd = s["x"].detach().double(), s["w_down"].detach().double()
    wg, wu = s["w_gate_up"].detach().double()[:inner], s["w_gate_up"].detach().double()[inner:]
    g, u = x @ wg.t(), x @ wu.t()
    if case["act"] == "silu":
        sig = torch.sigmoid(g)
        a, da = g * sig, sig + g * sig * (1 - sig)
    else:
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (g + 0.044715 * g ** 3))
        a, da = 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th ** 2) * c * (1 + 3 * 0.044715 * g ** 2)
    h = a * u
    out = h @ wd.t()
    if case["residual"]:
        out = out + s["residual"].detach().double()
    if not case["train"]:
        return [out]
    dy = s["dout"].double()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    grads = [dg @ wg + du @ wu, torch.cat([dg.t() @ x, du.t() @ x]), dy.t() @ h]
    return [out, *grads] + ([dy] if case["residual"] else [])


def _exact_dropout(s):
    case = s["case"]
    seed, step = (np.uint64(int(v) % 2 ** 64) for v in s["key"].cpu())
    n = case["rows"] * case["width"]
    low, word = np.uint64(0xFFFFFFFF), np.uint64(32)
    index = np.arange((n + 7) // 8, dtype=np.uint64)
    x0, x1 = index & low, index >> word
    x2, x3 = np.full_like(index, step & low), np.full_like(index, step >> word)
    a, b = int(seed & low), int(seed >> word)
    for _ in range(10):
        m0, m1 = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (m1 >> word) ^ x1 ^ np.uint64(a), m1 & low, (m0 >> word) ^ x3 ^ np.uint64(b), m0 & low
        a, b = (a + 0x9E3779B9) % 2 ** 32, (b + 0xBB67AE85) % 2 ** 32
    bits = np.empty((index.size, 8), dtype=np.uint16)
    for i, w in enumerate((x0, x1, x2, x3)):
        bits[:, 2 * i] = (w & np.uint64(0xFFFF)).astype(np.uint16)
        bits[:, 2 * i + 1] = (w >> np.uint64(16)).astype(np.uint16)
    threshold = round(case["p"] * 65536)
    kept = torch.from_numpy(bits.reshape(-1)[:n] >= threshold).cuda().reshape(case["rows"], case["width"])
    factor = kept.double() * 65536 / (65536 - threshold)
    out = s["x"].detach().double() * factor
    if case["residual"]:
        out = out + s["residual"].detach().double()
    if not case["train"]:
        return [out]
    dy = s["dout"].double()
    return [out, dy * factor] + ([dy] if case["residual"] else [])


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attention, "gated": _exact_gated, "dropout": _exact_dropout}[case["op"]](s)
