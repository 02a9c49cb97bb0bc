"""Adapter plans, refusals, and the CPU form of the multi-adapter projection."""
import numpy as np
import pytest
import torch

from vllm_sly_radiance_b200.models.lora import AdapterBank, AdapterPlan
from vllm_sly_radiance_b200.ops import kernels as K


def bank(L=3, S=2, R=8, Kd=32, N=24, sl=(0, 16, 24)):
    g = torch.Generator().manual_seed(0)
    return AdapterBank(torch.randn(L, S, R, Kd, generator=g).to(torch.bfloat16),
                       torch.randn(L, N, R, generator=g).to(torch.bfloat16), torch.rand(L, generator=g),
                       torch.full((L,), R, dtype=torch.int32), sl)


@pytest.mark.parametrize("T", [0, 1, 15, 16, 17, 100, 1000])
@pytest.mark.parametrize("tall_from", [None, 1, 128])
@pytest.mark.parametrize("room", [None, 80])
def test_plan_covers_every_row_once(T, tall_from, room):
    slots = np.random.default_rng(T).integers(-1, 7, T)
    if T == 1000:
        slots[300:700] = 2
    w, t16, t128 = AdapterPlan.pack(slots, 7, tiles16=room, tiles128=room, tall_from=tall_from)
    assert w.size == AdapterPlan.words(t16, t128)
    seen, at = [], 0
    for height, room_ in ((16, t16), (128, t128)):
        n, none = w[at], w[at + 1]
        tiles = w[at + 4:at + 4 + 4 * n].reshape(n, 4)
        assert n <= room_ and (tiles[:none, 0] == -1).all() and (tiles[none:, 0] >= 0).all()
        for i, (s, rows, seq, _) in enumerate(tiles):
            assert 0 < rows <= height
            r = w[at + 4 + 4 * room_ + i * height:][:rows]
            assert (slots[r] == s).all() and seq == (np.diff(r) == 1).all()
            seen += r.tolist()
        at += 4 + (4 + height) * room_
    assert sorted(seen) == list(range(T))


def test_plan_heights():
    """Few rows of an adapter go into short tiles, unless there are tall tiles anyway and few such remainders."""
    few = np.repeat(np.arange(3), 20)
    assert AdapterPlan.pack(few, 3)[1:] == (6, 0)
    assert AdapterPlan.pack(np.r_[few, np.full(60, 3)], 4)[1:] == (0, 4)
    many = np.r_[np.zeros(200, int), np.arange(1, 41)]
    assert AdapterPlan.pack(many, 41)[1:] == (40, 2)
    assert AdapterPlan.pack(np.zeros(140, int), 1, tall_from=128)[1:] == (1, 1)


def test_plan_of_short_tiles_only():
    w, t16, t128 = AdapterPlan.pack(np.zeros(300, int), 1, tiles16=300, tiles128=0)
    assert (t16, t128, w[0]) == (300, 0, 19)


def test_plan_refusals():
    with pytest.raises(ValueError):
        AdapterPlan.pack(np.array([0, 3]), 3)
    with pytest.raises(ValueError):
        AdapterPlan.pack(np.array([-2]), 3)
    with pytest.raises(ValueError):
        AdapterPlan.pack(np.arange(5), 5, tiles16=4)
    with pytest.raises(ValueError):
        AdapterPlan.pack(np.zeros(300, int), 5, tiles128=1)


def test_cpu_form():
    bk = bank()
    y, x = torch.randn(4, 24).to(torch.bfloat16), torch.randn(4, 32).to(torch.bfloat16)
    plan = AdapterPlan.build([2, -1, 0, 2], 3, "cpu")
    got = K.lora_add(y, x, bk, plan)
    assert torch.equal(got[1], y[1])
    for t, l in ((0, 2), (2, 0), (3, 2)):
        w = torch.cat([bk.b[l, :16].double() @ bk.a[l, 0].double(), bk.b[l, 16:].double() @ bk.a[l, 1].double()])
        want = y[t].double() + float(bk.scale[l]) * (w @ x[t].double())
        # bf16 rounding (unit roundoff 2^-8) and a 32-bit sum of 32 x 8 terms
        mag = float(bk.scale[l]) * (w.abs() @ x[t].double().abs()) + want.abs()
        assert ((got[t].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * mag).all()
    out = y.clone()
    assert K.lora_add(out, x, bk, plan, out=out) is out and torch.equal(out, got)
    assert K.lora_add(y[:0], x[:0], bk, AdapterPlan.build([], 3, "cpu")).shape == (0, 24)


@pytest.mark.parametrize("change", [
    dict(y=torch.zeros(4, 23, dtype=torch.bfloat16)), dict(y=torch.zeros(4, 24)),
    dict(x=torch.zeros(4, 31, dtype=torch.bfloat16)), dict(x=torch.zeros(3, 32, dtype=torch.bfloat16)),
    dict(x=torch.zeros(4, 32, dtype=torch.float16)), dict(x=torch.zeros(32, 4, dtype=torch.bfloat16).t()),
    dict(x=(torch.zeros(4, 32).to(torch.float8_e4m3fn), torch.ones(4, 1))),
    dict(x=(torch.zeros(4, 32, dtype=torch.bfloat16), torch.ones(4))),
    dict(slots=[0, 1, 2]), dict(out=torch.zeros(4, 24)), dict(out=torch.zeros(5, 24, dtype=torch.bfloat16)),
    dict(plan_slots=5)])
def test_refusals(change):
    a = dict(y=torch.zeros(4, 24, dtype=torch.bfloat16), x=torch.zeros(4, 32, dtype=torch.bfloat16),
             slots=[0, 1, 2, -1], out=None, plan_slots=3)
    a.update(change)
    plan = AdapterPlan.build(a["slots"], a["plan_slots"], "cpu")
    with pytest.raises(ValueError):
        K.lora_add(a["y"], a["x"], bank(), plan, out=a["out"])


@pytest.mark.parametrize("change", [
    dict(sl=(0, 24)), dict(sl=(0, 16, 20)), dict(sl=(0, 0, 24)), dict(sl=(1, 16, 24)), dict(S=9, sl=tuple(range(9)) + (24,)),
    dict(R=257)])
def test_bank_refusals(change):
    with pytest.raises(ValueError):
        bank(**change)


def test_bank_types():
    bk = bank()
    for kw in (dict(a=bk.a.float()), dict(scale=bk.scale.double()), dict(ranks=bk.ranks.long()),
               dict(b=bk.b[:, :, :4]), dict(a=bk.a[:2]), dict(scale=bk.scale[:2])):
        args = dict(a=bk.a, b=bk.b, scale=bk.scale, ranks=bk.ranks, slices=bk.slices)
        args.update(kw)
        with pytest.raises(ValueError):
            AdapterBank(**args)
