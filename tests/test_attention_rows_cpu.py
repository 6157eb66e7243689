"""Which memory the attention kernels walk over, for every way a tensor can lie: ``_C.attention_spacing`` gives the strides that a
launch would get, or nothing where the operator makes a copy first.  What is accepted has to be where the tensor's rows are."""
import itertools

import pytest
import torch

from bluefog_b200 import _C


def _tensor(*shape):
    return torch.arange(torch.Size(shape).numel(), dtype=torch.float32).to(torch.bfloat16).view(shape)


def _check(t, side_by_side=False):
    """Whether t is accepted; if so, its rows lie at the spacing that is given, in the order of its leading dimensions."""
    spacing = _C.attention_spacing(t, side_by_side)
    if spacing is None:
        return False
    lead = t.dim() - (1 if side_by_side else 2)
    heads = 1 if side_by_side else t.shape[-2]
    head_stride = 0 if side_by_side else spacing[1]
    assert t.stride(-1) == 1
    for row, index in enumerate(itertools.product(*(range(n) for n in t.shape[:lead]))):
        for h in range(heads):
            at = sum(i * s for i, s in zip(index, t.stride())) + (0 if side_by_side else h * t.stride(-2))
            assert row * spacing[0] + h * head_stride == at, (tuple(t.shape), t.stride(), spacing)
    return True


def _gradient(shape, reduce):
    """The gradient that autograd hands to a node whose result of this shape goes through ``reduce``."""
    seen = []
    x = _tensor(*shape).requires_grad_(True)
    y = x * 1
    y.register_hook(seen.append)
    z = reduce(y)
    z.backward(torch.ones_like(z))
    return seen[0]


@pytest.mark.parametrize("shape,reduce,accepted", [
    ((6, 3, 16), lambda y: y.sum(0), False),                           # packed documents, summed over the tokens
    ((2, 6, 3, 16), lambda y: y.sum(1), False),                        # a batch, summed over the tokens
    ((2, 6, 3, 16), lambda y: y.flatten(-2).sum(1), False),
    ((2, 6, 3, 16), lambda y: y.sum(0), False),                        # over the batch
    ((2, 6, 3, 16), lambda y: y.sum((0, 1)), False),
    ((2, 6, 3, 16), lambda y: y.sum(2), False),                        # over the heads
    ((2, 6, 3, 16), lambda y: y.sum(), False),
    ((1, 6, 3, 16), lambda y: y.sum(1), False),
    ((6, 1, 3, 16), lambda y: y.sum(0), False),
    ((6, 1, 3, 16), lambda y: y.sum(1), True),                         # one token per sequence: nothing is broadcast
    ((2, 6, 3, 16), lambda y: y * 2, True),
    ((2, 6, 3, 16), lambda y: y[:, 2:5], True),                        # a padded gradient is dense
])
def test_gradients_of_sums(shape, reduce, accepted):
    g = _gradient(shape, reduce)
    assert g.shape == shape and _check(g) == accepted, (g.stride(), _C.attention_spacing(g))


@pytest.mark.parametrize("t,accepted", [
    (_tensor(1, 3, 16).expand(6, 3, 16), False),
    (_tensor(2, 1, 3, 16).expand(2, 6, 3, 16), False),
    (_tensor(1, 6, 3, 16).expand(2, 6, 3, 16), False),
    (_tensor(6, 1, 16).expand(6, 3, 16), False),
    (_tensor(6, 3, 1).expand(6, 3, 16), False),
    (_tensor(6, 3, 16), True),
    (_tensor(2, 6, 3, 16), True),
    (_tensor(2, 6, 3, 16)[:, :4], False),                              # gaps between the sequences
    (_tensor(2, 6, 3, 16)[:, ::2], True),                              # every other token, all of them evenly spaced
    (_tensor(2, 6, 3, 16).transpose(0, 1), False),
    (_tensor(2, 3, 6, 16).transpose(1, 2), False),                     # heads outside the tokens
    (_tensor(6, 5, 16)[:, 1:4], True),
    (_tensor(6, 3, 24)[..., 8:], True),
    (_tensor(6, 3, 24)[..., 4:20], False),                             # 8-byte offset
    (_tensor(6, 3, 20)[..., :16], False),                              # spacing of 40 bytes
    (_tensor(1, 1, 1, 16), True),
    (_tensor(4, 1, 1, 16).expand(4, 1, 1, 16), True),
    (_tensor(96).as_strided((4, 2, 16), (16, 16, 1)), False),          # rows that overlap
])
def test_views(t, accepted):
    assert _check(t) == accepted, (t.stride(), _C.attention_spacing(t))


@pytest.mark.parametrize("t,accepted", [
    (_tensor(1, 48).expand(6, 48), False),
    (_tensor(2, 1, 48).expand(2, 6, 48), False),
    (_tensor(1, 6, 48).expand(2, 6, 48), False),
    (_tensor(1, 1, 48).expand(2, 6, 48), False),
    (_tensor(6, 1).expand(6, 48), False),
    (_tensor(6, 48), True),
    (_tensor(2, 6, 48), True),
    (_tensor(2, 6, 64)[..., 8:56], True),
    (_tensor(2, 6, 48)[:, 1:4], False),
    (_tensor(2, 6, 48).transpose(0, 1), False),
    (_tensor(6, 1, 48).expand(6, 1, 48), True),
    (_tensor(6, 52)[:, :48], False),
])
def test_views_of_a_joint_projection(t, accepted):
    assert _check(t, True) == accepted, (t.stride(), _C.attention_spacing(t, True))
