"""The router's choice where 32 bits cannot tell candidates apart, and its weights where 32 bits cannot hold the scores."""
import math

import pytest
import torch

from test_moe_router_cpu import SMALL_SIGMOIDS, check_masked_rows, check_small_sigmoids, check_small_softmax, close
from vllm_sly_radiance_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


@pytest.mark.parametrize("std", [2e-5, 1e-4])
def test_groups_whose_best_two_cancel(std):
    """Biases of +64 and -64: a group's value is about 1, its two terms are rounded to steps of 2^-17."""
    logits = torch.randn(2000, 8, device=DEV, generator=gen(0)) * std
    bias = torch.tensor([64.0, -64.0] * 4, device=DEV)
    ids, _ = K.moe_route(logits, 2, score="sigmoid", bias=bias, groups=4, top_groups=1)
    s = torch.sigmoid(logits.double())
    best = (s[:, ::2] + s[:, 1::2]).argmax(1)              # values in 64 bits, the bias gone
    assert torch.equal(ids, torch.stack([2 * best, 2 * best + 1], 1))


def test_softmax_sum_that_loses_every_addition():
    """1024 experts: expert 0 has e = 1, 36 others 0.98 * 2^-24 each, so that 32-bit additions one after the other leave 1.
    With the bias, expert 0 is worth -35.3 * 2^-24 and expert 40 -33.5 * 2^-24; without the lost terms' 0 it would win."""
    u = 2.0 ** -24
    l = torch.full((1, 1024), -torch.inf)
    l[0, 0] = 0.0
    small = math.log(0.98 * u)
    l[0, 1:32] = small
    for lane in (1, 2, 4, 8, 16):
        l[0, 32 * lane] = small
    bias = torch.full((1024,), -8.0)
    bias[0], bias[40] = -1.0, -33.5 * u
    s = torch.softmax(l.double(), 1) + bias.double()
    assert int(s.argmax()) == 40
    ids, _ = K.moe_route(l.to(DEV), 1, bias=bias.to(DEV))
    assert ids.tolist() == [[40]]


def test_bias_that_is_no_number():
    """An expert whose bias is NaN ranks last, and adds nothing to its group's value."""
    logits = torch.randn(50, 64, device=DEV, generator=gen(1))
    bias = torch.randn(64, device=DEV, generator=gen(2)) * 0.1
    bias[3], bias[17], bias[18], bias[40] = torch.nan, torch.nan, torch.nan, torch.nan
    for kw in ({}, {"groups": 8, "top_groups": 3}):
        got = K.moe_route(logits, 6, score="sigmoid", bias=bias, **kw)
        want = K.moe_route(logits.cpu(), 6, score="sigmoid", bias=bias.cpu(), **kw)
        assert torch.equal(got[0].cpu(), want[0])
        assert (got[1].cpu() - want[1]).abs().max() < 2.0 ** -19


@pytest.mark.parametrize("logits", SMALL_SIGMOIDS)
def test_sigmoid_scores_below_32_bits(logits):
    check_small_sigmoids(logits, DEV)


def test_softmax_scores_below_32_bits():
    check_small_softmax(DEV)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_rows_keep_weights_of_zero(score):
    check_masked_rows(score, DEV)


@pytest.mark.parametrize("E,groups,tops,k", [(680, 17, 3, 8), (1023, 3, 2, 32), (1020, 5, 2, 7), (999, 9, 4, 16), (1023, 31, 5, 9)])
@pytest.mark.parametrize("score,biased", [("softmax", False), ("sigmoid", True), ("softmax", True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_groups_of_many_experts(E, groups, tops, k, score, biased, dtype):
    """More than 32 experts for a lane: numbers of groups just above a power of two."""
    logits = (torch.randn(21, E, device=DEV, generator=gen(E)) * 2).to(dtype)
    bias = torch.randn(E, device=DEV, generator=gen(k)) * 0.1 if biased else None
    kw = dict(score=score, groups=groups, top_groups=tops)
    got = K.moe_route(logits, k, bias=bias, **kw)
    want = K.moe_route(logits.cpu(), k, bias=None if bias is None else bias.cpu(), **kw)
    assert torch.equal(got[0].cpu(), want[0])
    close(got[1], want[1].double())
