"""Dropout of ranks that start from one another's state."""
import pytest
import torch

from conftest import run_ranks


def test_ranks_draw_masks_of_their_own():
    run_ranks("dropout_masks", 3)


class _Rank:
    def __init__(self, rank):
        self.rank, self.is_initialized = lambda: rank, lambda: rank is not None


@pytest.mark.parametrize("seed", [0, 7, -1, 2 ** 63 - 1, -2 ** 63])
def test_rank_keys_wrap(seed, monkeypatch):
    from bluefog_b200.ops import fused_dropout
    key = fused_dropout.new_key(seed)
    key[1] = 5
    for rank in (None, 0, 1, 2, 1023):
        monkeypatch.setattr(fused_dropout, "_b", _Rank(rank))
        got = fused_dropout.rank_key(key)
        assert [v % 2 ** 64 for v in got.tolist()] == [(seed + (rank or 0) * 0x9E3779B97F4A7C15) % 2 ** 64, 5]
        assert key.tolist() == [seed, 5] and got.data_ptr() != key.data_ptr()
