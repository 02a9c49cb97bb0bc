"""Mixture-of-experts kernels against 64-bit definitions (tolerances derived in moe_oracle.py)."""
import pytest
import torch

import moe_oracle as M
from test_moe_ops_cpu import refusals
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


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("i", range(len(refusals("cpu"))))
def test_refusals(i):
    with pytest.raises(ValueError):
        refusals(DEV)[i]()


def test_refuses_other_devices_and_strides():
    g = gen(0)
    bank = LinearBank(bf16(g, 16, 24))
    x = bf16(g, 4, 24)
    with pytest.raises(ValueError):
        K.linear_fused(x, LinearBank(bank.weight.cpu()))
    with pytest.raises(ValueError):
        K.linear_fused(x.expand(4, 24)[:1].expand(4, 24), bank)           # rows on top of one another
    with pytest.raises(ValueError):
        K.linear_fused(bf16(g, 4, 28)[:, :24], bank)                      # a row stride off 16 bytes
    buf = bf16(g, 4, 24)
    with pytest.raises(ValueError):
        K.linear_fused(buf, LinearBank(bf16(g, 24, 24)), out=buf)         # in place of x
    with pytest.raises(ValueError):
        K.moe_route(randn(g, 16, 4).t(), 2)


# ---------------------------------------------------------------------------------------------
# route
# ---------------------------------------------------------------------------------------------
# exp, sum and quotient in 32 bits: below 2^-19 of the weight
def check_route(logits, k, **kw):
    ids, w = K.moe_route(logits, k, **kw)
    names = {"renormalize": "renorm"}
    want_ids, want_w = M.route(logits, k, **{names.get(n, n): v for n, v in kw.items()})
    assert ids.tolist() == want_ids.tolist()
    M.near(w.cpu(), want_w, want_w.abs() * 2.0 ** -19)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", [(1, 256, 8), (9, 60, 4), (33, 8, 8), (5, 1, 1), (7, 1024, 32), (3, 33, 5), (64, 512, 10),
                                   (2, 129, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route(T, E, k, dtype, score, biased):
    g = gen(T * E + k)
    logits = (randn(g, T, E) * 2).to(dtype)
    bias = randn(g, E, std=0.1) if biased else None
    check_route(logits, k, score=score, bias=bias)
    check_route(logits, k, score=score, bias=bias, renormalize=False, scale=2.5)


@pytest.mark.parametrize("E,groups,tops,k", [(256, 8, 4, 8), (160, 8, 3, 6), (60, 3, 2, 4), (64, 32, 5, 7), (35, 5, 2, 3),
                                             (1024, 16, 2, 32), (20, 10, 4, 8)])
@pytest.mark.parametrize("score,biased", [("softmax", False), ("sigmoid", True), ("softmax", True)])
def test_route_groups(E, groups, tops, k, score, biased):
    g = gen(E + groups)
    logits = randn(g, 40, E) * 2
    bias = randn(g, E, std=0.1) if biased else None
    check_route(logits, k, score=score, bias=bias, groups=groups, top_groups=tops)


def test_route_tells_near_candidates_apart():
    """Scores whose 32-bit roundings meet: the order is that of 64 bits."""
    g = gen(5)
    logits = randn(g, 300, 64)
    # the bias levels every expert of the first row to nearly one value
    bias = (1 - torch.sigmoid(logits[0].double())).float()
    check_route(logits[:1].repeat(20, 1) + randn(g, 20, 64, std=1e-7), 8, score="sigmoid", bias=bias)
    check_route(logits[:1].repeat(20, 1) + randn(g, 20, 64, std=1e-7), 8, score="sigmoid", bias=bias, groups=8, top_groups=3)
    # thousands of tokens: some always meet
    logits, bias = randn(g, 3000, 64) * 1.5, randn(g, 64, std=0.1)
    s = torch.sigmoid(logits.double()) + bias.double()
    want = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(K.moe_route(logits, 8, score="sigmoid", bias=bias)[0], want)


def test_route_ties_and_masks():
    ids, w = K.moe_route(torch.zeros(2, 70, device=DEV), 5)
    assert ids.tolist() == [[0, 1, 2, 3, 4]] * 2 and (w - 0.2).abs().max() < 1e-6
    l = torch.full((4, 48), -torch.inf, device=DEV)
    l[0, 37] = 3.0
    l[2] = torch.linspace(-1, 1, 48)
    l[2, 9] = torch.nan
    l[3] = torch.finfo(torch.float32).min
    l[3, 11] = 0
    for kw in [{}, {"groups": 4, "top_groups": 2}, {"renormalize": False}, {"bias": torch.zeros(48, device=DEV)},
               {"bias": torch.zeros(48, device=DEV), "groups": 4, "top_groups": 2}]:
        ids, w = K.moe_route(l, 6, **kw)
        assert ids[0, 0] == 37 and w[0].tolist() == [1, 0, 0, 0, 0, 0]
        assert w[1].tolist() == [0] * 6
        assert w[2].isnan().all()
        assert ids[3, 0] == 11 and w[3].tolist() == [1, 0, 0, 0, 0, 0]
        assert all(len(set(r)) == 6 and min(r) >= 0 and max(r) < 48 for r in ids.tolist())
    ids, w = K.moe_route(l, 6, score="sigmoid", scale=2.0)
    assert w[1].tolist() == [0] * 6 and ids[0, 0] == 37 and w[0, 0] == 2.0
    l[1, 4] = torch.inf
    assert K.moe_route(l, 6)[1][1].isnan().all() and K.moe_route(l, 6)[0][1, 0] == 4


def test_route_strides():
    g = gen(8)
    big = randn(g, 20, 257)
    for v in (big[:, :256], big[:, 1:], big[::2, :256], big[:1, :256]):
        got, want = K.moe_route(v, 8), K.moe_route(v.contiguous(), 8)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert K.moe_route(big[:0], 8)[0].shape == (0, 8)


# ---------------------------------------------------------------------------------------------
# plan, gather
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,E,first,n", [(1, 8, 256, 0, 256), (0, 3, 5, 0, 5), (64, 8, 256, 0, 256), (37, 3, 10, 4, 3),
                                           (300, 5, 1024, 0, 1024), (1500, 8, 64, 32, 32), (9000, 8, 256, 0, 256),
                                           (4099, 7, 60, 0, 60), (3, 1, 1, 0, 1), (20, 2, 8, 8, 4)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_plan(T, k, E, first, n, dtype):
    ids = torch.randint(-1, E, (T, k), device=DEV, generator=gen(T + k)).to(dtype)
    p = K.moe_plan(ids, n, first=first, tile=16)
    order, pos, counts = M.plan(ids.cpu(), n, first)
    assert p.order.tolist() == order and p.pos.tolist() == pos and p.counts.tolist() == counts
    assert p.starts.tolist() == [0] + torch.tensor(counts).cumsum(0).tolist()
    want = [[e, s + i, min(16, c - i)] for e, (s, c) in enumerate(zip(p.starts.tolist(), counts)) for i in range(0, c, 16)]
    items = p.items.tolist()
    assert items[:len(want)] == want and all(i == [0, 0, 0] for i in items[len(want):])


def test_plan_one_expert_and_strides():
    ids = torch.full((700, 6), 3, device=DEV)
    p = K.moe_plan(ids[:, ::2], 5)
    assert p.order.tolist() == list(range(2100)) and p.counts.tolist() == [0, 0, 0, 2100, 0]


@pytest.mark.parametrize("K_", [16, 96, 2048])
def test_gather(K_):
    g = gen(K_)
    x = bf16(g, 13, K_)
    ids = torch.randint(0, 7, (13, 3), device=DEV, generator=g)
    p = K.moe_plan(ids, 5)
    n = int(p.starts[-1])
    t = p.order[:n].long() // 3
    assert torch.equal(K.moe_gather(x, p)[:n], x[t])
    q, s = K.quant_fp8(x)
    gq, gs = K.moe_gather((q, s), p)
    assert torch.equal(gq[:n].view(torch.uint8), q.view(torch.uint8)[t]) and torch.equal(gs[:n], s[t])


# ---------------------------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------------------------
def grouped(T, k, E, Kd, N, act, by_token, seed=0, bias=True, ids=None, first=0, n=None):
    g = gen(seed + T * 7 + E)
    if ids is None:
        ids = torch.randint(0, E, (T, k), device=DEV, generator=g)
    n = n or E
    p = K.moe_plan(ids, n, first=first)
    w = bf16(g, n, N, Kd, std=Kd ** -0.5)
    b = bf16(g, n, N, std=0.3) if bias else None
    x = bf16(g, T if by_token else T * k, Kd)
    bank = LinearBank(w, b, act=act)
    R = int(p.starts[-1])
    order = p.order[:R].long()
    rows = order // k if by_token else torch.arange(R, device=DEV)
    return x, bank, p, rows, ids.flatten()[order] - first


def check_grouped(*a, scale=False, residual=False, **kw):
    x, bank, p, rows, experts = grouped(*a, **kw)
    g = gen(99)
    total, R = p.order.numel(), len(rows)
    s = torch.rand(total, device=DEV, generator=g) if scale else None
    r = bf16(g, total, bank.width) if residual else None
    out = torch.full((total, bank.width), 7.0, dtype=torch.bfloat16, device=DEV)
    got = K.linear_fused(x, bank, plan=p, by_token=kw.get("by_token", a[6]), scale=s, residual=r, out=out)
    assert K.check_status(DEV) == 0
    assert got.data_ptr() == out.data_ptr() and bool((out[R:] == 7).all())         # rows behind the last: as they were
    for a0 in range(0, R, 512):
        i = slice(a0, min(R, a0 + 512))
        M.near(got[i], *M.linear(x, bank.weight, bank.bias, bank.act, rows[i], experts[i], None if s is None else s[i],
                                 None if r is None else r[i]))


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("T,k,E,Kd,N", [
    (1, 2, 8, 64, 128),          # a cluster shares K where there is enough of it
    (1, 8, 32, 2048, 256),
    (3, 2, 4, 512, 2048),
    (1, 1, 1, 8, 2),             # the smallest weights
    (5, 3, 10, 200, 154),        # sizes that no tile divides
    (64, 8, 64, 128, 192),       # 8 rows an expert: 16-row tiles, several an expert
    (70, 4, 16, 72, 130),        # 64-row tiles
    (200, 4, 16, 136, 66),       # 128-row tiles
    (700, 2, 6, 320, 260),       # 256-row tiles
    (33, 1, 300, 64, 64),        # most experts without a row
])
def test_linear_grouped(act, by_token, T, k, E, Kd, N):
    check_grouped(T, k, E, Kd, N, act, by_token)


@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_linear_foreign_and_uneven_experts(act):
    g = gen(1)
    # another rank's experts and none at all; one expert with nearly every row
    ids = torch.randint(-1, 12, (90, 3), device=DEV, generator=g)
    check_grouped(90, 3, 12, 64, 96, act, True, ids=ids, first=4, n=4)
    check_grouped(90, 3, 12, 64, 96, act, False, ids=ids, first=12, n=4)          # no row
    ids = torch.where(torch.rand(500, 2, device=DEV, generator=g) < 0.95, 5, torch.randint(0, 40, (500, 2), device=DEV, generator=g))
    check_grouped(500, 2, 40, 128, 160, act, True, ids=ids, scale=True, residual=True)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 64, 65, 129, 255, 257, 700])
@pytest.mark.parametrize("act,Kd,N", [("none", 512, 320), ("swiglu", 328, 200)])
def test_linear_dense(rows, act, Kd, N):
    g = gen(rows)
    x, w, b = bf16(g, rows, Kd), bf16(g, N, Kd, std=Kd ** -0.5), bf16(g, N)
    bank = LinearBank(w, b, act=act)
    s, r = torch.rand(rows, device=DEV, generator=g) * 2, bf16(g, rows, bank.width)
    z = torch.zeros(rows, dtype=torch.long, device=DEV)
    i = torch.arange(rows, device=DEV)
    M.near(K.linear_fused(x, bank), *M.linear(x, w[None], b[None], act, i, z))
    want = M.linear(x, w[None], b[None], act, i, z, s, r)
    M.near(K.linear_fused(x, bank, scale=s, residual=r), *want)
    assert K.linear_fused(x, bank, scale=s, residual=r, out=r).data_ptr() == r.data_ptr()          # in place
    M.near(r, *want)
    assert K.check_status(DEV) == 0


def test_linear_strides_and_empty():
    g = gen(2)
    w = bf16(g, 136, 64, std=0.125)
    bank = LinearBank(w)
    big = bf16(g, 50, 200)
    want = K.linear_fused(big[:, 8:72].contiguous(), bank)
    assert torch.equal(K.linear_fused(big[:, 8:72], bank), want)
    assert torch.equal(K.linear_fused(big[::2, 8:72], bank), want[::2])
    for ld in (136, 137, 152):                           # rows of out on 16 bytes and off them
        out = torch.full((50, ld), 3.0, dtype=torch.bfloat16, device=DEV)
        K.linear_fused(big[:, 8:72], bank, out=out[:, :136], residual=want)
        assert torch.equal(out[:, :136], K.linear_fused(big[:, 8:72], bank, residual=want)) and bool((out[:, 136:] == 3).all())
    assert K.linear_fused(big[:0, :64], bank).shape == (0, 136)
    p = K.moe_plan(torch.zeros(0, 4, dtype=torch.long, device=DEV), 1)
    assert K.linear_fused(big[:0, :64], bank, plan=p, by_token=True).shape == (0, 136)


def test_linear_infinities_stay_in_their_row():
    g = gen(3)
    ids = torch.randint(0, 4, (40, 2), device=DEV, generator=g)
    p = K.moe_plan(ids, 4)
    bank = LinearBank(bf16(g, 4, 128, 64, std=0.1), act="swiglu")
    x = bf16(g, 40, 64)
    want = K.linear_fused(x, bank, plan=p, by_token=True)
    x[7] = torch.inf
    x[30, 5] = torch.nan
    got = K.linear_fused(x, bank, plan=p, by_token=True)
    t = p.order.long() // 2
    keep = (t != 7) & (t != 30)
    assert torch.equal(got[keep], want[keep]) and not got[~keep].isfinite().all(1).any()


def test_linear_is_the_same_every_time():
    a = grouped(64, 8, 64, 512, 256, "none", True)
    first = K.linear_fused(a[0], a[1], plan=a[2], by_token=True)
    for _ in range(5):
        assert torch.equal(K.linear_fused(a[0], a[1], plan=a[2], by_token=True), first)


# ---------------------------------------------------------------------------------------------
# combine
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,H", [(1, 8, 2048), (5, 3, 10), (17, 1, 8), (30, 11, 264), (4, 16, 7)])
@pytest.mark.parametrize("shared", [False, True])
def test_combine(T, k, H, shared):
    g = gen(T * k + H)
    ids = torch.randint(-1, 9, (T, k), device=DEV, generator=g)
    p = K.moe_plan(ids, 9)
    rows = bf16(g, T * k, H)
    n = int(p.starts[-1])
    rows[n:] = torch.nan                                  # rows that belong to nothing
    w = torch.rand(T, k, device=DEV, generator=g)
    w[ids < 0] = torch.nan                                # weights of none
    if not shared:
        M.near(K.moe_combine(rows, p, w), *M.combine(rows, p.pos, w))
        return
    sh, gate = bf16(g, T, 2 * H)[:, H:], randn(g, T, 3)[:, 1] * 4
    M.near(K.moe_combine(rows, p, w, shared=sh), *M.combine(rows, p.pos, w, sh))
    M.near(K.moe_combine(rows, p, w, shared=sh, gate=gate), *M.combine(rows, p.pos, w, sh, gate))
    assert K.check_status(DEV) == 0


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def block(g, E, H, I):
    return (LinearBank(bf16(g, E, 2 * I, H, std=H ** -0.5), act="swiglu"), LinearBank(bf16(g, E, H, I, std=I ** -0.5)),
            bf16(g, E, H, std=H ** -0.5))


def layer(x, up, down, router, k):
    ids, w = K.moe_route(x.float() @ router.float().t(), k)
    p = K.moe_plan(ids, up.E)
    return K.moe_combine(K.linear_fused(K.linear_fused(x, up, plan=p, by_token=True), down, plan=p), p, w)


def layer_oracle(x, up, down, router, k):
    """In 64 bits, but for the expert rows' rounding to bf16 between the products."""
    ids, w = M.route(x.float() @ router.float().t(), k)
    ids, w = ids.to(DEV), w.to(DEV)
    out = torch.zeros(x.shape, dtype=torch.double, device=DEV)
    for j in range(k):
        gu = torch.einsum("th,tnh->tn", x.double(), up.weight.double()[ids[:, j]])
        n = gu.shape[1] // 2
        a = gu[:, :n] * torch.sigmoid(gu[:, :n]) * gu[:, n:]
        out += w[:, j:j + 1] * torch.einsum("ti,thi->th", a, down.weight.double()[ids[:, j]])
    return out


@pytest.mark.parametrize("T", [1, 6, 50, 333])
def test_layer(T):
    g = gen(T)
    up, down, router = block(g, 16, 256, 128)
    x = bf16(g, T, 256)
    got, want = layer(x, up, down, router, 4), layer_oracle(x, up, down, router, 4)
    # three roundings to bf16 (activations, expert rows, result), each of independent sign: in the 2-norm at most their sum
    assert (got.double() - want).norm() <= 3 * M.BF16 * want.norm()


def test_layer_in_a_graph_and_on_two_streams():
    g = gen(11)
    up, down, router = block(g, 16, 256, 128)
    xs = [bf16(g, 24, 256) for _ in range(4)]
    want = [layer(x, up, down, router, 4) for x in xs]
    buf = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(buf, up, down, router, 4)
    for x, y in zip(xs, want):
        buf.copy_(x)
        graph.replay()
        assert torch.equal(out, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, x in enumerate(xs * 5):
        with torch.cuda.stream(streams[i % 2]):
            got.append(layer(x, up, down, router, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i % 4]) for i, a in enumerate(got))
    assert K.check_status(DEV) == 0


def test_two_graphs_of_one_layer():
    """Captured calls share nothing: two graphs over the same weights replay in turn and on two streams."""
    g = gen(12)
    up, down, router = block(g, 16, 256, 128)
    xs = [bf16(g, 40, 256), bf16(g, 3, 256)]
    want = [layer(x, up, down, router, 4) for x in xs]
    graphs = []
    for x in xs:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, up, down, router, 4)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for (graph, out), st in zip(graphs, streams):
            out.zero_()
        torch.cuda.synchronize()
        for (graph, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, y) for (_, out), y in zip(graphs, want))


def test_bias_that_masks_and_same_expert_twice():
    g = gen(13)
    logits = randn(g, 30, 64)
    bias = torch.zeros(64, device=DEV)
    bias[::2] = -torch.inf                                  # half of the experts are never chosen
    ids, w = K.moe_route(logits, 8, score="sigmoid", bias=bias)
    want = torch.sort(logits[:, 1::2], dim=1, descending=True, stable=True).indices[:, :8] * 2 + 1
    assert torch.equal(ids, want)
    # a token that names one expert in several slots has a row for each
    ids = torch.tensor([[3, 3, 1], [1, 3, 3]], device=DEV)
    p = K.moe_plan(ids, 4)
    assert p.order.tolist() == [2, 3, 0, 1, 4, 5] and p.pos.tolist() == [[2, 3, 0], [1, 4, 5]]
    rows = bf16(g, 6, 16)
    wt = torch.rand(2, 3, device=DEV, generator=g)
    M.near(K.moe_combine(rows, p, wt), *M.combine(rows, p.pos, wt))


@pytest.mark.parametrize("rows", [3, 40, 600])
def test_linear_takes_any_magnitude(rows):
    """Gates far to either side, zeros, the largest numbers: as the formula in 64 bits, rounded once."""
    g = gen(rows)
    x = bf16(g, rows, 64)
    x[0] = 0
    x[1] *= 2.0 ** 60
    w = bf16(g, 96, 64)
    i, z = torch.arange(rows, device=DEV), torch.zeros(rows, dtype=torch.long, device=DEV)
    got = K.linear_fused(x, LinearBank(w, act="swiglu"))
    want, bound = M.linear(x, w[None], None, "swiglu", i, z)
    big = want.abs() > torch.finfo(torch.bfloat16).max      # beyond bf16: infinity of the same sign
    assert torch.equal(got[big].double(), torch.sign(want[big]) * torch.inf)
    M.near(got[~big], want[~big], bound[~big])
