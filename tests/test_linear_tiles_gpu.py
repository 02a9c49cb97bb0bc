"""linear_fused on every kernel that its rule can pick (test_linear_tiles_cpu.py pins which), against 64 bits: single CTAs and
CTA pairs, several items a CTA, more k blocks than the ring has stages, rows in order and by token."""
import pytest
import torch

import moe_oracle as M
from test_linear_tiles_cpu import TILES, tiles
from vllm_sly_radiance_b200.models.layers import LinearBank
from vllm_sly_radiance_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def bf16(g, *shape, std=1.0):
    return randn(g, *shape, std=std).to(torch.bfloat16)


def check(got, x, bank, rows, starts, scale, residual):
    """Rows of one expert after another against moe_oracle.linear's value and bound, its products by matrix."""
    K_ = x.shape[1]
    for e, (a, b) in enumerate(zip(starts, starts[1:])):
        for r0 in range(a, b, 1024):
            r = slice(r0, min(b, r0 + 1024))
            xe, w = x[rows[r]].double(), bank.weight[e].double()
            y = xe @ w.t()
            err = (xe.abs() @ w.abs().t()) * (K_ * 2.0 ** -23)
            if bank.bias is not None:
                y = y + bank.bias[e].double()
                err = err + y.abs() * 2.0 ** -24
            if bank.act == "swiglu":
                n = y.shape[1] // 2
                g, u, eg, eu = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
                s = g * torch.sigmoid(g)
                y = s * u
                err = 1.1 * eg * (u.abs() + eu) + s.abs() * eu + 2.0 ** -19 * y.abs()
            if scale is not None:
                y, err = y * scale[r].double()[:, None], err * scale[r].double().abs()[:, None]
                err = err + 2.0 ** -24 * y.abs()
            if residual is not None:
                y = y + residual[r].double()
            err = err + 2.0 ** -23 * y.abs()
            M.near(got[r], y, err + M.BF16 * (y.abs() + err) + 1e-38)


def popular_ids(g, T, E, k):
    """Experts of very different popularity: tiles from one row to whole ones."""
    return torch.topk(randn(g, T, E) * 1.5 + randn(g, E, std=0.7), min(k, E), dim=1).indices


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("want,case", TILES)
def test_every_tile(want, case, by_token, rest):
    T, k, E, Kd, N, act = case
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if sms == 148:
        assert tiles(*case) == want
    g = gen(T + 3 * E + Kd)
    ids = popular_ids(g, T, E, k) if E > 1 else torch.zeros(T, 1, dtype=torch.long, device=DEV)
    plan = K.moe_plan(ids, E)
    bank = LinearBank(bf16(g, E, N, Kd, std=Kd ** -0.5), bf16(g, E, N, std=0.3) if rest else None, act=act)
    R = T * k
    x = bf16(g, T if by_token else R, Kd + 8)[:, :Kd]                # rows apart
    scale = torch.rand(R, device=DEV, generator=g) * 2 if rest else None
    residual = bf16(g, R, bank.width) if rest else None
    rows = plan.order.long() // k if by_token else torch.arange(R, device=DEV)
    first = K.linear_fused(x, bank, plan=plan, by_token=by_token, scale=scale, residual=residual)
    assert K.check_status(DEV) == 0
    check(first, x, bank, rows, plan.starts.tolist(), scale, residual)
    for _ in range(4):                                               # one order of sums, whatever meets in time
        assert torch.equal(K.linear_fused(x, bank, plan=plan, by_token=by_token, scale=scale, residual=residual), first)
    if E == 1 and not by_token:
        assert torch.equal(K.linear_fused(x, bank, scale=scale, residual=residual), first)
    assert K.check_status(DEV) == 0


@pytest.mark.parametrize("act,Kd,N", [("swiglu", 1096, 520), ("none", 136, 516)])
def test_a_rank_of_the_experts_on_pairs(act, Kd, N):
    """Half of the experts are another rank's: rows behind the last one stay as they were."""
    g = gen(3)
    T, k, E, n = 2048, 8, 64, 32
    plan = K.moe_plan(popular_ids(g, T, E, k), n, first=16)
    assert tiles(T, k, n, Kd, N, act)[1]
    bank = LinearBank(bf16(g, n, N, Kd, std=Kd ** -0.5), act=act)
    x = bf16(g, T, Kd)
    out = torch.full((T * k, bank.width), 7.0, dtype=torch.bfloat16, device=DEV)
    K.linear_fused(x, bank, plan=plan, by_token=True, out=out)
    starts = plan.starts.tolist()
    assert bool((out[starts[-1]:] == 7).all())
    check(out, x, bank, plan.order.long().clamp(min=0) // k, starts, None, None)
    assert K.check_status(DEV) == 0


def test_pairs_in_a_graph_beside_another_stream():
    """A captured call by token on pairs and eager ones on another stream at the same time."""
    g = gen(4)
    T, k, E, Kd, N = 2048, 8, 64, 520, 512
    plan = K.moe_plan(popular_ids(g, T, E, k), E)
    bank = LinearBank(bf16(g, E, N, Kd, std=Kd ** -0.5), act="swiglu")
    x, other = bf16(g, T, Kd), bf16(g, T, Kd)
    want, want_other = (K.linear_fused(v, bank, plan=plan, by_token=True) for v in (x, other))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.linear_fused(x, bank, plan=plan, by_token=True)
    side = torch.cuda.Stream()
    for _ in range(5):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            got = K.linear_fused(other, bank, plan=plan, by_token=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got, want_other)
    assert K.check_status(DEV) == 0
