"""Ranks and slices that the multi-adapter projection's first tests leave out, with their formula and tolerance
(test_lora_gpu): ranks that 4 or 8 do not divide, and more rank rows than one matrix instruction takes."""
import numpy as np
import pytest

from test_lora_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("R", [1, 2, 3, 5, 12, 20, 50, 67, 131])
@pytest.mark.parametrize("fp8", [False, True])
def test_ranks_of_any_size(tile_rows, R, fp8):
    T = 150
    slots = np.random.default_rng(R).integers(-1, 3, T)
    check(*make(T, 192, [72, 16, 40], R, 3, fp8, seed=R, ranks=[R, max(1, R - 1), (R + 1) // 2]), slots=slots, tile_rows=tile_rows)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("R,sizes", [(128, [136, 64, 64]), (256, [80, 24]), (200, [40, 40]), (72, [16] * 8), (100, [24, 24, 24])])
@pytest.mark.parametrize("Kd", [264, 131])
def test_more_rank_rows_than_one_instruction(tile_rows, R, sizes, Kd):
    """Groups of whole slices: several CTAs, and a last group with fewer slices than the others."""
    T = 140
    slots = np.random.default_rng(R).integers(-1, 2, T)
    for fp8 in (False, True):
        check(*make(T, Kd, sizes, R, 2, fp8, seed=R, ranks=[R, R - 3]), slots=slots, tile_rows=tile_rows)
