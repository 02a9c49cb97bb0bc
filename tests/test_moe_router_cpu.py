"""The router's weights where 32 bits cannot hold the scores, on the CPU; the GPU tests run the same cases."""
import pytest
import torch

from vllm_sly_radiance_b200.ops import kernels as K

SMALL_SIGMOIDS = [[-100.0, -101.0, -103.5, -140.0, -99.25, -250.0],
                  [-100.0, -101.0, -60.0, -90.0, -75.0, -300.0],
                  [-95.0, 0.5, -92.125, -3.0, -torch.inf, -88.0],
                  [-700.0, -701.0, -702.0, -710.0, -705.0, -torch.inf],
                  [-90000.0, -90001.0, -90002.0, -90010.0, -90003.0, -99999.0]]


def close(got, want):
    """exp, its argument, sum and quotient in 32 bits: below 2^-19 of the weight; the smallest numbers by their steps of 2^-149."""
    d = (got.double().cpu() - want).abs()
    assert bool((d <= want.abs() * 2.0 ** -19 + 1e-44).all()), (got.tolist(), want.tolist())


def check_small_sigmoids(logits, device):
    """sigmoid(l) = e^min(l, 0) / (1 + e^-|l|); divided by their sum only ratios remain."""
    l = torch.tensor([logits])
    for bias in (None, torch.zeros(6, device=device)):
        ids, w = K.moe_route(l.to(device), 5, score="sigmoid", bias=bias, scale=2.5)
        x = l.double()[0][ids.cpu()[0]]
        e = torch.exp(x.clamp(max=0) - x.clamp(max=0).max()) / (1 + torch.exp(-x.abs()))
        close(w[0], 2.5 * e / e.sum())


def check_small_softmax(device):
    """The bias picks experts whose share of the softmax 32 bits do not hold, nor 64."""
    l = torch.tensor([[200.0, 3.0, 1.0, 2.5, -torch.inf, 0.0], [900.0, 3.0, 1.0, 2.5, -2.0, 0.0]])
    bias = torch.tensor([-8.0, 1.0, 2.0, 3.0, 0.0, 0.0])
    ids, w = K.moe_route(l.to(device), 3, bias=bias.to(device))
    assert ids.tolist() == [[3, 2, 1]] * 2
    close(w, torch.softmax(torch.tensor([[2.5, 1.0, 3.0]] * 2).double(), 1))


def check_masked_rows(score, device):
    l = torch.full((1, 16), -torch.inf, device=device)
    for bias in (None, torch.zeros(16, device=device)):
        ids, w = K.moe_route(l, 4, score=score, bias=bias)
        assert w.tolist() == [[0.0] * 4] and len(set(ids[0].tolist())) == 4


@pytest.mark.parametrize("logits", SMALL_SIGMOIDS)
def test_sigmoid_scores_below_32_bits(logits):
    check_small_sigmoids(logits, "cpu")


def test_softmax_scores_below_32_bits():
    check_small_softmax("cpu")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_rows_keep_weights_of_zero(score):
    check_masked_rows(score, "cpu")
