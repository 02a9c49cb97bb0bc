"""Mixture-of-experts operators on the CPU: the oracle path against 64-bit definitions, and what the entry points refuse."""
import pytest
import torch

import moe_oracle as M
from vllm_sly_radiance_b200.models.layers import LinearBank
from vllm_sly_radiance_b200.ops import kernels as K

ROUTES = [
    # T, E, k, score, bias, groups, top_groups, renorm, scale
    (5, 16, 4, "softmax", False, 1, 1, True, 1.0),
    (3, 60, 6, "sigmoid", True, 1, 1, True, 2.5),
    (4, 32, 4, "sigmoid", True, 8, 3, True, 1.0),
    (4, 32, 4, "softmax", False, 4, 2, False, 16.0),
    (2, 8, 8, "softmax", True, 1, 1, False, 1.0),
    (1, 1, 1, "softmax", False, 1, 1, True, 1.0),
]


@pytest.mark.parametrize("T,E,k,score,biased,groups,tops,renorm,scale", ROUTES)
def test_route_definition(T, E, k, score, biased, groups, tops, renorm, scale):
    g = torch.Generator().manual_seed(T * E)
    logits = torch.randn(T, E, generator=g) * 2
    bias = torch.randn(E, generator=g) * 0.2 if biased else None
    ids, w = K.moe_route(logits, k, score=score, bias=bias, groups=groups, top_groups=tops, renormalize=renorm, scale=scale)
    want_ids, want_w = M.route(logits, k, score, bias, groups, tops, renorm, scale)
    assert ids.tolist() == want_ids.tolist() and ids.dtype == torch.int64
    M.near(w, want_w, want_w.abs() * 2.0 ** -22)


def test_route_ties_and_masks():
    logits = torch.zeros(1, 8)
    ids, w = K.moe_route(logits, 3)
    assert ids.tolist() == [[0, 1, 2]] and torch.allclose(w, torch.full((1, 3), 1 / 3))
    logits = torch.full((2, 8), -torch.inf)
    logits[0, 5] = 1.0
    ids, w = K.moe_route(logits, 2)
    assert ids[0, 0] == 5 and w[0].tolist() == [1.0, 0.0] and w[1].tolist() == [0.0, 0.0]
    logits = torch.randn(2, 8)
    logits[1, 3] = torch.nan
    ids, w = K.moe_route(logits, 4, groups=2, top_groups=1)
    assert w[1].isnan().all() and not w[0].isnan().any()
    assert len(set(ids[1].tolist())) == 4


def test_plan_definition():
    g = torch.Generator().manual_seed(0)
    for T, k, E, first, n in [(7, 3, 10, 0, 10), (9, 2, 12, 4, 4), (1, 1, 3, 2, 1), (0, 2, 4, 0, 4), (5, 2, 6, 6, 2)]:
        ids = torch.randint(-1, E, (T, k), generator=g)
        p = K.moe_plan(ids, n, first=first)
        order, pos, counts = M.plan(ids, n, first)
        assert p.order.tolist() == order and p.pos.tolist() == pos and p.counts.tolist() == counts
        assert p.starts.tolist() == [sum(counts[:i]) for i in range(n + 1)]


def test_plan_items_are_the_grouped_products():
    ids = torch.randint(0, 6, (40, 2), generator=torch.Generator().manual_seed(1))
    p = K.moe_plan(ids, 6, tile=16)
    items = [i for i in p.items.tolist() if i[2]]
    rows = [(e, r) for e, r0, n in items for r in range(r0, r0 + n)]
    assert rows == [(e, r) for e in range(6) for r in range(int(p.starts[e]), int(p.starts[e + 1]))]


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("by_token", [False, True])
def test_linear_definition(act, by_token):
    g = torch.Generator().manual_seed(3)
    T, k, E, N, Kd = 6, 2, 5, 14, 24
    ids = torch.randint(0, E, (T, k), generator=g)
    p = K.moe_plan(ids, E)
    w = (torch.randn(E, N, Kd, generator=g) * 0.3).to(torch.bfloat16)
    b = (torch.randn(E, N, generator=g) * 0.3).to(torch.bfloat16)
    x = torch.randn(T if by_token else T * k, Kd, generator=g).to(torch.bfloat16)
    scale = torch.rand(T * k, generator=g)
    res = torch.randn(T * k, N // 2 if act == "swiglu" else N, generator=g).to(torch.bfloat16)
    got = K.linear_fused(x, LinearBank(w, b, act=act), plan=p, by_token=by_token, scale=scale, residual=res)
    rows = p.order.long() // k if by_token else torch.arange(T * k)
    M.near(got, *M.linear(x, w, b, act, rows, ids.flatten()[p.order.long()], scale, res))


def test_combine_definition():
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, 4, (5, 3), generator=g)
    p = K.moe_plan(ids, 4)
    rows = torch.randn(15, 10, generator=g).to(torch.bfloat16)
    w, sh, gate = torch.rand(5, 3, generator=g), torch.randn(5, 10, generator=g).to(torch.bfloat16), torch.randn(5, generator=g)
    M.near(K.moe_combine(rows, p, w), *M.combine(rows, p.pos, w))
    M.near(K.moe_combine(rows, p, w, shared=sh, gate=gate), *M.combine(rows, p.pos, w, sh, gate))


def refusals(dev):
    """(call, ...) that must raise ValueError on `dev`."""
    f = torch.zeros(4, 16, device=dev)
    ids = torch.zeros(4, 2, dtype=torch.long, device=dev)
    plan = K.moe_plan(ids, 3)
    w = torch.zeros(3, 8, 16, dtype=torch.bfloat16, device=dev)
    x = torch.zeros(8, 16, dtype=torch.bfloat16, device=dev)
    bank, one = LinearBank(w), LinearBank(w[0].contiguous())
    rows = torch.zeros(8, 8, dtype=torch.bfloat16, device=dev)
    wt = torch.zeros(4, 2, device=dev)
    return [
        lambda: K.moe_route(f, 0), lambda: K.moe_route(f, 17), lambda: K.moe_route(f, 2, score="relu"),
        lambda: K.moe_route(f, 2, groups=3), lambda: K.moe_route(f, 9, groups=2, top_groups=1),
        lambda: K.moe_route(f, 2, groups=2, top_groups=3), lambda: K.moe_route(f[0], 2), lambda: K.moe_route(f.long(), 2),
        lambda: K.moe_route(f, 2, bias=torch.zeros(4, device=dev)),
        lambda: K.moe_route(f, 2, bias=torch.zeros(16, dtype=torch.bfloat16, device=dev)),
        lambda: K.moe_route(f, 2, bias=torch.zeros(16, device=dev), groups=16, top_groups=4),
        lambda: K.moe_plan(ids[0], 3), lambda: K.moe_plan(ids.float(), 3), lambda: K.moe_plan(ids, 0),
        lambda: K.moe_plan(ids, 1025), lambda: K.moe_plan(ids, 3, first=-1),
        lambda: K.moe_gather(x, plan),
        lambda: K.moe_combine(rows[:7], plan, wt), lambda: K.moe_combine(rows.float(), plan, wt),
        lambda: K.moe_combine(rows, plan, wt[:3]), lambda: K.moe_combine(rows, plan, wt.double()),
        lambda: K.moe_combine(rows, plan, wt, shared=rows), lambda: K.moe_combine(rows, plan, wt, gate=wt[:, 0]),
        lambda: K.linear_fused(x, bank), lambda: K.linear_fused(x, one, by_token=True),
        lambda: K.linear_fused(x[:4], bank, plan=plan), lambda: K.linear_fused(x, bank, plan=plan, by_token=True),
        lambda: K.linear_fused(x.float(), bank, plan=plan), lambda: K.linear_fused(x[:, :8], bank, plan=plan),
        lambda: K.linear_fused(x, LinearBank(w[:2].contiguous()), plan=plan),
        lambda: K.linear_fused(x, bank, plan=plan, scale=torch.zeros(7, device=dev)),
        lambda: K.linear_fused(x, bank, plan=plan, residual=rows[:7]),
        lambda: K.linear_fused(x, bank, plan=plan, out=rows.float()),
        lambda: LinearBank(w.float()), lambda: LinearBank(w[:, :, :12].contiguous()), lambda: LinearBank(w[:, :, :8]),
        lambda: LinearBank(w[:, :7].contiguous(), act="swiglu"), lambda: LinearBank(w, act="gelu"),
        lambda: LinearBank(w, torch.zeros(3, 7, dtype=torch.bfloat16, device=dev)),
        lambda: LinearBank(torch.zeros(1025, 1, 8, dtype=torch.bfloat16, device=dev)),
    ]


@pytest.mark.parametrize("i", range(len(refusals("cpu"))))
def test_refusals(i):
    with pytest.raises(ValueError):
        refusals("cpu")[i]()
