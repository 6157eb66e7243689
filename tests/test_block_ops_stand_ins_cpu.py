"""Fake tensors, which claim to lie on a GPU and have no memory, are refused before anything is launched or a device is asked for."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from bluefog_b200 import _C


def test_fake_tensors_are_refused():
    with FakeTensorMode():
        t = torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda")
        key = torch.empty(2, dtype=torch.int64, device="cuda")
        cu = torch.empty(2, dtype=torch.int32, device="cuda")
        for call in (lambda: _C.causal_attention(t, t, t, None, 0.1), lambda: _C.causal_attention(t, t, t, cu, 0.1),
                     lambda: _C.causal_self_attention(t.flatten(1).repeat(1, 3), 2, 2, None, 0.1),
                     lambda: _C.dropout_add(t, None, 100, 1.0, key, 0), lambda: _C.dropout_add(t, t, 100, 1.0, key, 0)):
            with pytest.raises(NotImplementedError, match="plain tensors"):
                call()
        assert _C.gated_mlp(t[:, 0], t[:, 0], t[:, 0, :4], 3, None) is None       # PyTorch's operators take it
