"""Which calls the attention kernels take, by sizes alone: grids and offsets have 31 bits."""
import math

import pytest


def _tiles(lead, batch):
    tokens = math.prod(lead)
    return tokens // lead[-1] * -(-lead[-1] // 128) if batch is None else tokens // 128 + batch + 1


@pytest.mark.parametrize("lead", [(1,), (130,), (8, 1024), (2 ** 26, 1), (2 ** 26 + 1, 1), (2 ** 19, 129), (2 ** 30,), (2 ** 31 - 257,), (2 ** 31 - 256,), (2 ** 32,)])
@pytest.mark.parametrize("heads", [1, 3, 8, 16])
@pytest.mark.parametrize("batch", [None, 1, 2 ** 25, 2 ** 26, 2 ** 30])
def test_limits(lead, heads, batch):
    from bluefog_b200.ops import fused_attention as fa
    # both kinds of blocks of the backward pass in one grid; TMA coordinates of the rows
    fits = _tiles(lead, batch) * heads * 2 < 2 ** 31 and math.prod(lead) < 2 ** 31 - 256
    assert fa._fits(lead, heads, batch) == fits
