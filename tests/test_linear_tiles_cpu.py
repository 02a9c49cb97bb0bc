"""Which kernel a product of linear_fused takes: the rule on a card of 148 SMs, for the sizes that the GPU tests run."""
import pytest

from vllm_sly_radiance_b200.ops import _ext

# tile rows, CTA pairs, CTAs that share K <- tokens, slots, experts, K, N, act
TILES = [
    ((16, False, 8), (1, 8, 32, 2048, 256, "none")),
    ((16, False, 4), (1, 8, 32, 1024, 512, "none")),
    ((16, False, 2), (1, 8, 32, 512, 256, "swiglu")),
    ((16, False, 1), (24, 8, 32, 1100 // 8 * 8, 514, "none")),
    ((32, False, 1), (256, 4, 64, 1096, 1030, "none")),
    # 64 rows: several items a CTA, more k blocks than the ring has stages, odd widths
    ((64, False, 1), (512, 3, 64, 200, 1034, "swiglu")),
    ((64, False, 1), (640, 3, 64, 1096, 330, "none")),
    ((64, False, 1), (640, 3, 64, 1096, 1040, "swiglu")),
    # CTA pairs on experts' rows: several items a pair, tiles of 1 to 256 rows
    ((256, True, 1), (2048, 8, 64, 1096, 520, "swiglu")),
    ((256, True, 1), (2048, 8, 64, 136, 516, "none")),
    ((256, True, 1), (1024, 4, 8, 1096, 2560, "none")),
    ((256, True, 1), (1500, 2, 6, 200, 5134, "swiglu")),
    # one weight: every height that pairs take
    ((64, True, 1), (64, 1, 1, 264, 20002, "none")),
    ((64, True, 1), (500, 1, 1, 1032, 2060, "swiglu")),
    ((96, True, 1), (300, 1, 1, 1096, 4000, "none")),
    ((96, True, 1), (700, 1, 1, 264, 2050, "none")),
    ((128, True, 1), (1000, 1, 1, 1096, 2050, "none")),
    ((160, True, 1), (2000, 1, 1, 136, 1030, "none")),
    ((192, True, 1), (1500, 1, 1, 200, 4000, "swiglu")),
    ((224, True, 1), (400, 1, 1, 200, 8200, "swiglu")),
    ((256, True, 1), (4096, 1, 1, 512, 2048, "none")),
    ((256, True, 1), (4096, 1, 1, 1032, 1024, "swiglu")),
]


def tiles(T, k, E, Kd, N, act, sms=148):
    sw = act == "swiglu"
    return _ext.ext().linear_fused_tiles(T * k, E, N // 2 if sw else N, Kd, sw, sms)


@pytest.mark.skipif(not _ext.available(), reason="the extension is not built")
@pytest.mark.parametrize("want,case", TILES)
def test_rule(want, case):
    assert tiles(*case) == want


@pytest.mark.skipif(not _ext.available(), reason="the extension is not built")
def test_rule_over_all_sizes():
    """Tiles fit their kernel, pairs' rows are whole 32s, a split leaves every CTA four 64-blocks of K."""
    heights = set()
    for T in (1, 2, 15, 31, 63, 130, 500, 1100, 4096, 20000):
        for E in (1, 2, 7, 64, 1024):
            for Kd in (8, 200, 1000, 5120):
                for N in (2, 130, 1030, 8704):
                    for act in ("none", "swiglu"):
                        tile, pair, splits = tiles(T, min(E, 8), E, Kd, N, act)
                        heights.add((tile, pair))
                        assert tile in ((64, 96, 128, 160, 192, 224, 256) if pair else (16, 32, 64))
                        assert splits in (1, 2, 4, 8) and (splits == 1 or (tile == 16 and (Kd + 63) // 64 >= 4 * splits))
    assert {(16, False), (32, False), (64, False), (64, True), (128, True), (256, True)} <= heights
    for bad in ((0, 1, 8, 8, False, 148), (8, 0, 8, 8, False, 148), (8, 1, 8, 8, False, 1)):
        with pytest.raises(ValueError):
            _ext.ext().linear_fused_tiles(*bad)
