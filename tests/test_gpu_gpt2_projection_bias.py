"""The bias of GPT-2's joint q, k, v projection: the gradients of its query and value parts through ``causal_self_attention``, and that
of the key part, which is zero but for rounding (a constant added to every key shifts a row's scores alike).

Bound as for the other gradients of this model: sixteen roundings of 2^-8 per layer and direction, two layers, eight in the
classifier, twice that."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BOUND = 2 * math.sqrt(2 * 2 * 16 + 8) * 2.0 ** -8


@pytest.mark.parametrize("n_kv_head", [4, 2, 1])
@pytest.mark.parametrize("packed", [False, True])
def test_bias_of_the_joint_projection(n_kv_head, packed):
    from bluefog_b200.models import gpt2
    torch.manual_seed(0)
    args = dict(vocab_size=1001, n_positions=160, d_model=256, n_layer=2, n_head=4, n_kv_head=n_kv_head, use_b200_attention=True)
    ref = gpt2.GPT2(**args).cuda()
    with torch.no_grad():
        for p in ref.parameters():
            p.mul_(3 if p.dim() == 2 else 1)                          # attention that is not all but flat
            p.copy_(p.to(torch.bfloat16))
    fast = gpt2.GPT2(**args).cuda()
    fast.load_state_dict(ref.state_dict())
    fast.to(torch.bfloat16)
    x, y = (torch.randint(0, 1001, (3, 150), device="cuda") for _ in range(2))
    cu = torch.tensor([0, 70, 71, 300, 450], dtype=torch.int32, device="cuda") if packed else None
    fast(x, y, cu).backward()
    ref(x, y, cu).backward()
    kv = 64 * n_kv_head
    for a, b in zip(fast.h, ref.h):
        q, k, v = a.attn.c_attn.bias.grad.float().split([256, kv, kv])
        want_q, _, want_v = b.attn.c_attn.bias.grad.split([256, kv, kv])
        for got, want in ((q, want_q), (v, want_v)):
            assert want.norm() > 1e-6
            assert ((got - want).norm() / want.norm()).item() <= BOUND
        assert k.norm() <= BOUND * q.norm()
