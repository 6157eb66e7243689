"""``check_sequences`` sees what calls on any stream reported, and loses none of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _bad(tokens=200):
    from bluefog_b200.ops import fused_attention as fa
    qkv = torch.zeros(tokens, 3 * 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 150, 120], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return lambda: fa.causal_self_attention(qkv, 1, cu_seqlens=cu)


def test_a_report_from_another_stream():
    from bluefog_b200.ops import fused_attention as fa
    call = _bad()
    call()                                                            # loading a kernel for the first time waits for the device
    with pytest.raises(IndexError):
        fa.check_sequences()
    x = torch.randn(4096, 4096, device="cuda")
    x = x @ x * 1e-3
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(40):                                           # some milliseconds in front of the call
            x = x @ x * 1e-3
        call()
    with pytest.raises(IndexError):
        fa.check_sequences()
    torch.cuda.synchronize()
    fa.check_sequences()                                              # reported once


@pytest.mark.parametrize("first", [128, 1, -3])
def test_boundaries_that_do_not_start_at_zero(first):
    """The kernels take the first boundary as 0; that it is another one is reported, as the CPU path does."""
    from bluefog_b200.ops import fused_attention as fa
    qkv = torch.zeros(256, 3 * 64, dtype=torch.bfloat16, device="cuda")
    fa.causal_self_attention(qkv, 1, cu_seqlens=torch.tensor([first, 256], dtype=torch.int32, device="cuda"))
    with pytest.raises(IndexError, match="start at 0"):
        fa.check_sequences()
    fa.causal_self_attention(qkv, 1, cu_seqlens=torch.tensor([0, 256], dtype=torch.int32, device="cuda"))
    fa.check_sequences()
