"""Attention, gated block and dropout together, as GPT-2 uses them: the bf16 kernels against the same weights, masks and
documents evaluated in fp32 with PyTorch's operators.

Bound on the norm of a difference: every operator rounds its result and some of its operands to bf16, each rounding is
off by at most 2^-8 of the value and independent of the others, and between the embedding and the loss, and back, a value
passes about 16 of them per layer; two layers and the classifier give sqrt(2 * 2 * 16 + 8) * 2^-8 = 0.033.  Twice that is
allowed, since LayerNorm and the residual stream weigh them unevenly."""
import math
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
BOUND = 2 * math.sqrt(2 * 2 * 16 + 8) * 2.0 ** -8
OPTIONS = [dict(use_b200_attention=True), dict(n_kv_head=2, mlp="swiglu", use_b200_attention=True),
           dict(n_kv_head=1, mlp="geglu", dropout=0.2, use_b200_attention=True)]


def _models(**kw):
    from bluefog_b200.models import gpt2
    torch.manual_seed(0)
    args = dict(vocab_size=1001, n_positions=160, d_model=256, n_layer=2, n_head=4, **kw)
    ref = gpt2.GPT2(**args).cuda()
    with torch.no_grad():
        for p in ref.parameters():                                    # larger than at the start of a training, so that
            p.mul_(3 if p.dim() == 2 else 1)                          # attention and gates are not all but flat
            p.copy_(p.to(torch.bfloat16))
    fast = gpt2.GPT2(**args).cuda()
    fast.load_state_dict(ref.state_dict())
    return ref, fast.to(torch.bfloat16)


def _near(a, b, what):
    off = ((a.float() - b).norm() / b.norm()).item()
    assert off <= BOUND, (what, off)


@pytest.mark.parametrize("kw", OPTIONS)
@pytest.mark.parametrize("packed", [False, True])
def test_logits_loss_and_gradients(kw, packed):
    ref, fast = _models(**kw)
    x, y = (torch.randint(0, 1001, (3, 150), device="cuda") for _ in range(2))
    cu = torch.tensor([0, 70, 71, 300, 450], dtype=torch.int32, device="cuda") if packed else None
    _near(fast.eval()(x, cu_seqlens=cu), ref.eval()(x, cu_seqlens=cu), "logits")
    loss, want = fast.train()(x, y, cu), ref.train()(x, y, cu)
    assert abs(loss.item() - want.item()) <= BOUND * abs(want.item())
    loss.backward()
    want.backward()
    for (name, p), q in zip(fast.named_parameters(), ref.parameters()):
        if q.grad.norm() > 1e-6:                                      # key biases: zero but for rounding
            _near(p.grad, q.grad, name) if "c_attn.bias" not in name else None
    if "dropout" in kw:
        assert fast.dropout_key.tolist() == ref.dropout_key.tolist() and fast.dropout_key.tolist()[1] == 1


def test_captured_training_step_repeats_the_eager_one():
    """Forward and backward in one graph: replay k draws the masks of eager step k and gives its gradients, bit for bit."""
    _, model = _models(n_kv_head=2, mlp="swiglu", dropout=0.1, use_b200_attention=True)
    x, y = (torch.randint(0, 1001, (2, 130), device="cuda") for _ in range(2))
    params = list(model.parameters())

    def step():
        loss = model(x, y)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    names = [n for n, _ in model.named_parameters()]
    eager = [step() for _ in range(3)]
    again = [step() for _ in range(1)]
    assert not torch.equal(eager[0][0], eager[1][0]) and not torch.equal(again[0][0], eager[2][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    model.dropout_key[1] = 0
    for k in range(3):
        graph.replay()
        # the loss adds its rows with atomics: 260 fp32 terms in any order
        assert abs(got[0].item() - eager[k][0].item()) <= 260 * 2.0 ** -24 * abs(eager[k][0].item())
        for n, a, b in zip(names, got[1:], eager[k][1:]):
            if n.startswith("wte") or n.startswith("wpe") or "bias" in n or ".ln_" in n or n.startswith("ln_"):
                # sums that other kernels of the library take with atomics
                torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-3 * b.float().abs().max().item())
            else:
                assert torch.equal(a, b), n


_FIRST_CALL = """
import torch
from bluefog_b200 import _C
from bluefog_b200.ops import fused_attention as fa, gemm
torch.manual_seed(0)
mk = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
qkv, wgu, wd, dy = mk(200, 3 * 128), mk(2 * 136, 128), mk(64, 136), mk(200, 64)
cu = torch.tensor([0, 77, 200], dtype=torch.int32, device="cuda")

def step(leaves):
    out = fa.causal_self_attention(leaves[0], 2, cu_seqlens=cu)
    y = gemm.gated_mlp(out.view(200, 128), *leaves[1:])
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

leaves = [t.clone().requires_grad_(True) for t in (qkv, wgu, wd)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step(leaves)
fa.check_sequences()
assert _C.gemm_status() == 0
want = step([t.clone().requires_grad_(True) for t in (qkv, wgu, wd)])
for _ in range(2):
    graph.replay()
assert all(torch.equal(a, b) for a, b in zip(got, want))
# what one call reports, a replay does not take back
fa.causal_self_attention(qkv, 2, cu_seqlens=torch.tensor([0, 150, 120], dtype=torch.int32, device="cuda"))
graph.replay()
try:
    fa.check_sequences()
except IndexError:
    print("reported")
"""


def test_first_calls_of_a_process_in_a_capture():
    run = subprocess.run([sys.executable, "-c", _FIRST_CALL], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "reported" in run.stdout, run.stdout + run.stderr
