"""Pages and state slots moved inside the caches: bit for bit, on the CPU and with the kernel."""
import numpy as np
import pytest
import torch

from vllm_sly_radiance_b200.engine.cache_moves import CacheMover, plan_compaction
from vllm_sly_radiance_b200.models.hybrid import ModelCaches

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def caches(device, dtype=torch.uint8, layers=3, blocks=12, heads=2, page=16, row=48, slots=6, conv=(40, 3), ssm=(2, 8, 8),
           seed=0):
    g = torch.Generator().manual_seed(seed)

    def bits(*shape, dt):
        n = int(np.prod(shape)) * torch.empty(0, dtype=dt).element_size()
        return torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8).view(dt).view(*shape).to(device)

    k = [bits(blocks, heads, page, row, dt=dtype) for _ in range(layers)]
    v = [bits(blocks, heads, page, row, dt=dtype) for _ in range(layers)]
    c = [bits(slots, *conv, dt=torch.bfloat16) for _ in range(layers)]
    s = [bits(slots, *ssm, dt=torch.float32) for _ in range(layers)]
    return ModelCaches(k, v, c, s, page)


def raw(c):
    return [t.cpu().clone().view(torch.uint8) for t in c.k + c.v], \
           [t.cpu().reshape(t.shape[0], -1).clone().view(torch.uint8) for t in c.conv + c.ssm]


def expect(kv, st, blocks, slots):
    for t in kv:
        old = t.clone()
        for s, d, n in blocks:
            t[d, :, :n] = old[s, :, :n]
    for t in st:
        old = t.clone()
        for s, d in slots:
            t[d] = old[s]
    return kv, st


def same(c, want):
    if c.k and c.k[0].is_cuda:
        torch.cuda.synchronize()
        from vllm_sly_radiance_b200.ops import kernels as K
        K.check_status(c.k[0].device)
    got = raw(c)
    return all(torch.equal(a, b) for u, v in zip(got, want) for a, b in zip(u, v))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("geometry", [
    dict(), dict(dtype=torch.float8_e4m3fn, page=64, row=64), dict(dtype=torch.bfloat16, row=32, heads=1),
    dict(row=12, conv=(5, 3), ssm=(1, 3, 3)),                 # rows and states that 16 bytes do not divide
    dict(page=64, row=256, heads=4, layers=1),                # several pieces a page
    dict(row=256, heads=5, page=64, conv=(4096, 3), ssm=(4, 64, 64))])
def test_copy(device, geometry):
    c = caches(device, **geometry)
    page = c.block_size
    blocks = [(1, 2, 1), (1, 3, 1), (5, 4, page), (6, 7, page - 1), (8, 9, 0), (8, 10, 5), (1, 11, page)]
    slots = [(1, 2), (1, 3), (4, 5)]
    want = expect(*raw(c), blocks, slots)
    CacheMover(c).copy(blocks, slots)
    assert same(c, want)


@pytest.mark.parametrize("device", DEVICES)
def test_copy_views_of_larger_tensors(device):
    """Caches that are views (every other block of a tensor) with a stride of their own."""
    c = caches(device, blocks=24)
    c.k = [t[::2] for t in c.k]
    c.v = [t[1::2] for t in c.v]
    want = expect(*raw(c), [(0, 5, 7), (3, 11, 16)], [])
    CacheMover(c).copy([(0, 5, 7), (3, 11, 16)])
    assert same(c, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 64, 65, 200, 1700, 3200])
def test_many_moves(device, n):
    """Lists of every size class of the launch, one destination and several a source."""
    c = caches(device, layers=1, blocks=2 * n + 3, heads=1, page=2, row=16, slots=2)
    ids = 1 + np.random.default_rng(n).permutation(2 * n + 2)
    one = [(int(s), int(d)) for s, d in zip(ids[:n], ids[n:2 * n])]
    want = expect(*raw(c), [(s, d, 2) for s, d in one], [])
    CacheMover(c).copy(one)
    assert same(c, want)
    fan = [(int(ids[i // 100]), int(ids[n + i]), 1) for i in range(n)]
    want = expect(*raw(c), fan, [])
    CacheMover(c).copy(fan)
    assert same(c, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("live", [[], [1], [11], [1, 2, 3], [11, 5, 2, 9], list(range(1, 12))])
def test_compact(device, live):
    c = caches(device)
    t = np.full((2, 7), -1, np.int32)
    t[0, :min(6, len(live))] = live[:6]
    t[1, :len(live[6:])] = live[6:]
    if live:
        t[1, 6] = live[0]                                     # a page that two sequences share
    old = raw(c)
    new, n = CacheMover(c).compact(t)
    assert n == len(live) and sorted(set(new[new > 0].tolist())) == list(range(1, n + 1))
    assert ((new > 0) == (t > 0)).all() and new.dtype == t.dtype
    got = raw(c)
    for (i, j) in np.argwhere(t > 0):
        for a, b in zip(got[0], old[0]):
            assert torch.equal(a[new[i, j]], b[t[i, j]])
    for a, b in zip(got[0], old[0]):
        assert torch.equal(a[0], b[0])
    assert all(torch.equal(a, b) for a, b in zip(got[1], old[1]))


def test_plan_moves_only_what_it_must():
    used = np.zeros(10, bool)
    used[[0, 2, 3, 8, 9]] = True
    src, dst, n = plan_compaction(used)
    assert (src.tolist(), dst.tolist(), n) == ([8, 9], [1, 4], 4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("blocks,slots", [
    ([(1, 12)], []), ([(-1, 2)], []), ([(1, 2), (2, 3)], []), ([(1, 2), (3, 2)], []), ([(1, 2, 17)], []),
    ([(1, 2, -1)], []), ([(1, 1)], []), ([], [(0, 6)]), ([], [(1, 2), (2, 1)]), ([], [(1, 2, 3)]), ([(1, 2, 3, 4)], []),
    ([(1, 2)], [(0, 9)])])
def test_refusals(device, blocks, slots):
    c = caches(device)
    want = raw(c)
    with pytest.raises(ValueError):
        CacheMover(c).copy(blocks, slots)
    if not (blocks and slots):
        assert same(c, want)


def test_compact_refuses_unknown_blocks():
    with pytest.raises(ValueError):
        CacheMover(caches("cpu")).compact(np.array([[3, 12]]))
