"""Moves that are no whole numbers are refused, not cut to some."""
import numpy as np
import pytest
import torch

from test_cache_moves import DEVICES, caches, expect, raw, same
from vllm_sly_radiance_b200.engine.cache_moves import CacheMover


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("blocks,slots", [
    ([(1.5, 2)], []), ([(1.0, 2)], []), (np.array([[1, 2, 3.7]]), []), ([], [(1, 2.9)]), ([("1", "2")], []),
    ([(True, False)], []), ([(1, None)], []), ([(1 << 70, 2)], []), ([(1, 2), (3,)], [])])
def test_refused_types(device, blocks, slots):
    c = caches(device)
    want = raw(c)
    with pytest.raises(ValueError):
        CacheMover(c).copy(blocks, slots)
    assert same(c, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("make", [np.array, np.int32, np.uint8, torch.tensor, tuple, lambda m: np.array(m)[:, ::-1][:, ::-1]])
def test_whole_numbers_of_any_kind(device, make):
    c = caches(device)
    want = expect(*raw(c), [(1, 2, 5), (3, 4, 16)], [(0, 5)])
    CacheMover(c).copy(make([(1, 2, 5), (3, 4, 16)]), make([(0, 5)]))
    CacheMover(c).copy([], ())
    CacheMover(c).copy(np.empty((0, 2)), np.zeros((0, 2), np.int64))
    assert same(c, want)
