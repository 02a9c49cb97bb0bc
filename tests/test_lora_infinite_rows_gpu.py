"""Rows of x that hold an infinity, for ranks that do not fill the 16 that a matrix instruction takes."""
import numpy as np
import pytest
import torch

from test_lora_gpu import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("R,ranks", [(8, [1, 5]), (16, [3, 16]), (40, [17, 40])])
def test_infinite_row_of_x(tile_rows, R, ranks):
    """A row of x with an infinity, matrices without a zero: infinities of the products' signs for every rank, not NaN
    from what the tile holds beyond the adapter's rank."""
    g = torch.Generator().manual_seed(R)
    T, Kd = 20, 96
    a = torch.rand(2, 1, R, Kd, generator=g).add(0.5).to(torch.bfloat16)
    b = torch.rand(2, 24, R, generator=g).add(0.5).to(torch.bfloat16)
    b[:, 1::2] *= -1
    x, y = torch.randn(T, Kd, generator=g).to(torch.bfloat16), torch.randn(T, 24, generator=g).to(torch.bfloat16)
    x[3, 7], x[4, 90] = float("inf"), float("-inf")
    slots = np.arange(T) % 2
    got = run(y, x, a, b, torch.ones(2), torch.tensor(ranks, dtype=torch.int32), [0, 24], slots, tile_rows=tile_rows)
    sign = torch.tensor([1.0, -1.0] * 12, dtype=torch.float64)
    assert torch.equal(got[3], sign * float("inf")) and torch.equal(got[4], -sign * float("inf"))
    assert torch.isfinite(got[[i for i in range(T) if i not in (3, 4)]]).all()
