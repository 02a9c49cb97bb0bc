"""The multi-adapter projection against its formula in 64 bits.

Tolerance: bf16 rounding of the result (unit roundoff 2^-8: 8 significant bits), and for what comes before it the bound of a sum in 32 bits
in any order, (K + R + 8) 2^-24, plus 2^-16 for the low-rank row held as two bf16 numbers, both times the sum of
the absolute terms."""
import numpy as np
import pytest
import torch

from vllm_sly_radiance_b200.models.lora import AdapterBank, AdapterPlan
from vllm_sly_radiance_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(T, Kd, sizes, R, L, fp8, seed=0, ranks=None, pad=0):
    g = torch.Generator().manual_seed(seed)
    sl = np.concatenate([[0], np.cumsum(sizes)]).tolist()
    S, N = len(sizes), sl[-1]
    rk = torch.full((L,), R, dtype=torch.int32) if ranks is None else torch.tensor(ranks, dtype=torch.int32)
    keep = torch.arange(R)[None] < rk[:, None]
    a = (torch.randn(L, S, R, Kd, generator=g) * Kd ** -0.5 * keep[:, None, :, None]).to(torch.bfloat16)
    b = (torch.randn(L, N, R, generator=g) * 0.1 * keep[:, None]).to(torch.bfloat16)
    sc = torch.rand(L, generator=g) * 2 + 0.25
    y = torch.randn(T, N + pad, generator=g).to(torch.bfloat16)[:, :N]
    x = torch.randn(T, Kd + pad, generator=g)
    if fp8:
        s = x.abs().amax(1).clamp(min=1e-6) / 448
        x = ((x / s[:, None]).to(torch.float8_e4m3fn)[:, :Kd], s)
    else:
        x = x.to(torch.bfloat16)[:, :Kd]
    return y, x, a, b, sc, rk, sl


def dev(x):
    # keeps the row stride of a view (Tensor.cuda() would compact it)
    if isinstance(x, tuple):
        return tuple(dev(t) for t in x)
    if x.dim() == 2 and x.stride(0) != x.shape[1]:
        full = torch.empty(x.shape[0], x.stride(0), dtype=x.dtype, device=DEV)
        v = full[:, :x.shape[1]]
        v.copy_(x)
        return v
    return x.to(DEV)


def formula(y, x, a, b, sc, rk, sl, slots):
    """(out, bound) in 64 bits."""
    xd = x[0].double() * x[1].double()[:, None] if isinstance(x, tuple) else x.double()
    out = y.double().clone()
    mag = torch.zeros_like(out)
    for t, l in enumerate(slots):
        if l < 0:
            continue
        r = int(rk[l])
        for s in range(len(sl) - 1):
            A, B = a[l, s, :r].double(), b[l, sl[s]:sl[s + 1], :r].double()
            out[t, sl[s]:sl[s + 1]] += float(sc[l]) * (B @ (A @ xd[t]))
            mag[t, sl[s]:sl[s + 1]] = float(sc[l]) * (B.abs() @ (A.abs() @ xd[t].abs()))
    c = (a.shape[3] + a.shape[2] + 8) * 2.0 ** -24 + 2.0 ** -16
    return out, 2.0 ** -8 * (out.abs() + c * mag) + c * mag


def run(y, x, a, b, sc, rk, sl, slots, inplace=False, tile_rows=None):
    bank = AdapterBank(a.to(DEV), b.to(DEV), sc.to(DEV), rk.to(DEV), sl)
    if tile_rows is None:
        plan = AdapterPlan.build(np.asarray(slots), a.shape[0], DEV)
    else:
        w, t16, t128 = AdapterPlan.pack(np.asarray(slots), a.shape[0], tall_from=1 if tile_rows == 128 else None,
                                        tiles128=0 if tile_rows == 16 else None)
        plan = AdapterPlan(torch.from_numpy(w).to(DEV), len(slots), t16, t128, a.shape[0])
    yd = dev(y)
    got = K.lora_add(yd, dev(x), bank, plan, out=yd if inplace else None)
    torch.cuda.synchronize()
    K.check_status(got.device)
    assert (got.data_ptr() == yd.data_ptr()) == inplace
    if not inplace:
        assert torch.equal(yd.cpu().view(torch.int16), y.contiguous().view(torch.int16))
    return got.cpu().double()


def check(*case, slots, **kw):
    want, tol = formula(*case, slots)
    got = run(*case, slots, **kw)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()))


CASES = [
    # T, K, slice sizes, R, adapters, fp8
    (1, 256, [512], 16, 1, True), (1, 5120, [384, 128, 128], 16, 3, True), (3, 264, [40], 8, 2, False),
    (8, 512, [256, 256], 16, 8, True), (17, 768, [640], 32, 4, False), (64, 1024, [512, 96], 32, 24, True),
    (37, 1250, [77, 13, 35], 8, 5, False), (5, 33, [9, 1], 8, 2, True), (130, 1088, [136], 64, 1, False),
    (300, 640, [264, 48], 16, 3, True), (515, 512, [520], 64, 2, False), (260, 392, [256, 8], 128, 2, True),
    (9, 136, [64], 256, 2, False), (200, 136, [64], 256, 1, False), (150, 96, [7, 9, 33], 40, 3, True),
]


@pytest.mark.parametrize("T,Kd,sizes,R,L,fp8", CASES)
@pytest.mark.parametrize("inplace", [False, True])
def test_lora_add(T, Kd, sizes, R, L, fp8, inplace):
    rng = np.random.default_rng(T + Kd)
    slots = rng.integers(-1, L, T)
    slots[0] = L - 1
    check(*make(T, Kd, sizes, R, L, fp8, seed=T), slots=slots, inplace=inplace)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_lora_tiles(tile_rows, fp8):
    """Both tile heights at row counts around the tile's end, mixed ranks (0 among them), row strides of views."""
    for T in (1, 15, 16, 17, 127, 128, 129, 257):
        case = make(T, 320, [96, 24, 8], 32, 5, fp8, seed=T, ranks=[32, 1, 0, 9, 16], pad=16)
        slots = np.random.default_rng(T).integers(-1, 5, T)
        check(*case, slots=slots, tile_rows=tile_rows)
        check(*case, slots=np.full(T, 3), tile_rows=tile_rows)


@pytest.mark.parametrize("tile_rows", [16, 128])
def test_lora_rows_without_adapter(tile_rows):
    """Rows without an adapter come back bit for bit, whatever their x and y hold; NaN and infinities stay in their
    own rows, and what a slot holds beyond its rank or in an unused slot is never read."""
    for T in (6, 140):
        y, x, a, b, sc, rk, sl = make(T, 192, [72, 16], 16, 3, False, seed=5, ranks=[16, 5, 16])
        a[1, :, 5:], b[1, :, 5:] = float("nan"), float("inf")
        a[2], b[2], sc[2] = float("nan"), float("nan"), float("nan")
        slots = np.arange(T) % 3 - 1                       # none, 0, 1
        x[slots == -1] = float("nan")
        x[1], y[2, 3] = float("inf"), float("nan")         # rows of adapters 0 and 1
        got = run(y, x, a, b, sc, rk, sl, slots, tile_rows=tile_rows)
        none = torch.tensor(slots == -1)
        assert torch.equal(got[none], y.double()[none])
        want, tol = formula(y, x, a, b, sc, rk, sl, slots)
        keep = torch.ones(T, dtype=torch.bool)
        keep[1] = False                                    # an infinite x row has no finite result
        keep[2] = False
        assert not (~((got - want).abs() <= tol))[keep].any()
        assert torch.isnan(got[2, 3]) and not torch.isnan(got[2, :3]).any()
        assert not torch.isfinite(got[1]).all()


def test_lora_infinite_low_rank_row():
    """A low-rank row that overflows to infinity gives infinities of the products' signs, not NaN."""
    a = torch.full((1, 1, 1, 8), 3e38).to(torch.bfloat16).expand(1, 1, 8, 8).contiguous()
    b = torch.zeros(1, 16, 8, dtype=torch.bfloat16)
    b[0, :, 0] = torch.tensor([1.0, -2.0] * 8).to(torch.bfloat16)
    rk = torch.tensor([1], dtype=torch.int32)
    x = torch.full((2, 8), 4.0).to(torch.bfloat16)
    y = torch.zeros(2, 16, dtype=torch.bfloat16)
    for tr in (16, 128):
        got = run(y, x, a, b, torch.ones(1), rk, [0, 16], [0, 0], tile_rows=tr)
        assert torch.equal(got, torch.tensor([[float("inf"), -float("inf")] * 8] * 2).double())


def test_lora_repeatable_and_streams():
    """The same call twice gives the same bits; calls on two streams at once do not disturb each other."""
    case = make(300, 2048, [1024], 64, 4, False, seed=9)
    y, x, a, b, sc, rk, sl = case
    slots = np.random.default_rng(1).integers(-1, 4, 300)
    bank = AdapterBank(a.to(DEV), b.to(DEV), sc.to(DEV), rk.to(DEV), sl)
    plan = AdapterPlan.build(slots, 4, DEV)
    yd, xd = y.to(DEV), x.to(DEV)
    first = K.lora_add(yd, xd, bank, plan)
    x2 = -xd
    other = K.lora_add(yd, x2, bank, plan)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(8):
        with torch.cuda.stream(s1):
            got.append((K.lora_add(yd, xd, bank, plan), first))
        with torch.cuda.stream(s2):
            got.append((K.lora_add(yd, x2, bank, plan), other))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in got)


def test_lora_graph_replay_with_new_plan():
    """A captured call follows the plan buffer: other rows and adapters at replay, fewer tiles than captured."""
    T, L = 24, 6
    y, x, a, b, sc, rk, sl = make(T, 512, [192], 16, L, True, seed=3)
    bank = AdapterBank(a.to(DEV), b.to(DEV), sc.to(DEV), rk.to(DEV), sl)
    words, t16, t128 = AdapterPlan.pack(np.arange(T) % L, L, tiles16=T, tiles128=0)
    buf = torch.from_numpy(words).to(DEV)
    plan = AdapterPlan(buf, T, t16, t128, L)
    yd, xd = y.to(DEV), dev(x)
    for _ in range(2):
        K.lora_add(yd, xd, bank, plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = K.lora_add(yd, xd, bank, plan)
    for slots in (np.full(T, -1), np.full(T, 2), np.random.default_rng(0).integers(-1, L, T)):
        w, _, _ = AdapterPlan.pack(slots, L, tiles16=T, tiles128=0)
        buf.copy_(torch.from_numpy(w))
        g.replay()
        torch.cuda.synchronize()
        want, tol = formula(y, x, a, b, sc, rk, sl, slots)
        assert not (~((out.cpu().double() - want).abs() <= tol)).any()
    K.check_status(out.device)


def test_lora_bad_plan_is_reported():
    """A plan buffer that names rows or slots that do not exist is refused on the device, with the status word set."""
    y, x, a, b, sc, rk, sl = make(4, 128, [64], 8, 2, False)
    bank = AdapterBank(a.to(DEV), b.to(DEV), sc.to(DEV), rk.to(DEV), sl)
    for tall in (0, 1):
        for at, val in ((0, 3), (4, 2), (5, 129), (5, -1), (12, 4), (12, -1)):
            w, t16, t128 = AdapterPlan.pack(np.array([0, 0, 1, 1]), 2, tall_from=1, tiles128=2 * tall)
            w[at + 4 * tall] = val                      # an empty 16-row list is 4 words
            plan = AdapterPlan(torch.from_numpy(w).to(DEV), 4, t16, t128, 2)
            K.lora_add(y.to(DEV), x.to(DEV), bank, plan)
            with pytest.raises(K.KernelFaultError):
                K.check_status(torch.device(DEV, 0))
    K.check_status(torch.device(DEV, 0))


def test_lora_refusals():
    y, x, a, b, sc, rk, sl = make(4, 32, [16, 8], 8, 3, False)
    bank = AdapterBank(a.to(DEV), b.to(DEV), sc.to(DEV), rk.to(DEV), sl)
    y, x = y.to(DEV), x.to(DEV)
    plan = AdapterPlan.build([0, 1, 2, -1], 3, DEV)
    q = torch.zeros(4, 32, device=DEV).to(torch.float8_e4m3fn)
    buf = torch.zeros(8 * 24, dtype=torch.bfloat16, device=DEV)
    yv = buf[:96].view(4, 24)
    for args in ((y[:, :23], x, plan), (y.float(), x, plan), (y, x[:, :31], plan), (y, x[:3], plan), (y, x.half(), plan),
                 (y, torch.zeros(32, 4, dtype=torch.bfloat16, device=DEV).t(), plan), (y, (q, torch.ones(4, 1, device=DEV)), plan),
                 (y, (q, torch.ones(4)), plan), (y, (x, torch.ones(4, device=DEV)), plan), (y, q, plan),
                 (y, x, AdapterPlan.build([0, 1, 2], 3, DEV)), (y, x, AdapterPlan.build([0, 1, 2, 0], 4, DEV)),
                 (y, x, AdapterPlan.build([0, 1, 2, 0], 3, "cpu")), (y, x, plan, y.float()), (y, x, plan, y[:3]),
                 (yv, x, plan, buf[24:120].view(4, 24)),                      # overlaps y but is not y
                 (y, x, plan, x[:, :24]),                                     # overlaps x
                 (y, x, plan, y[:1].expand(4, 24))):                          # rows on top of one another
        with pytest.raises(ValueError):
            K.lora_add(args[0], args[1], bank, args[2], out=args[3] if len(args) > 3 else None)
    assert K.lora_add(y[:0], x[:0], bank, AdapterPlan.build([], 3, DEV)).shape == (0, 24)
    K.check_status(y.device)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("T", [1, 40])
def test_lora_broadcast_and_unaligned_views(tile_rows, T):
    """A broadcast x and y (row stride 0), and operands that start off any vector boundary."""
    case = make(T, 128, [48, 16], 16, 2, False, seed=T)
    y, x, a, b, sc, rk, sl = case
    slots = np.arange(T) % 2
    bank = AdapterBank(a.to(DEV), b.to(DEV), sc.to(DEV), rk.to(DEV), sl)
    w, t16, t128 = AdapterPlan.pack(slots, 2, tall_from=1 if tile_rows == 128 else None, tiles128=0 if tile_rows == 16 else None)
    plan = AdapterPlan(torch.from_numpy(w).to(DEV), T, t16, t128, 2)

    def same(yd, xd, out=None):
        want, tol = formula(yd.cpu(), xd.cpu(), a, b, sc, rk, sl, slots)
        got = K.lora_add(yd, xd, bank, plan, out=out)
        torch.cuda.synchronize()
        K.check_status(got.device)
        assert not (~((got.cpu().double() - want).abs() <= tol)).any()
    same(y[:1].to(DEV).expand(T, 64), x.to(DEV))
    same(y.to(DEV), x[:1].to(DEV).expand(T, 128))
    same(y[:1].to(DEV).expand(T, 64), x[:1].to(DEV).expand(T, 128))

    def shifted(t, off):
        v = torch.empty(t.numel() + off, dtype=t.dtype, device=DEV)[off:].view(t.shape)
        return v.copy_(t)
    for off in (1, 4):
        same(shifted(y, off), shifted(x, off), out=shifted(torch.zeros_like(y), 3 * off))
