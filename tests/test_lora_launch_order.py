"""The adapters' prompt kernels hold their tensor memory before a dependent launch may start.

A kernel that lets the next one start before its own blocks have allocated tensor memory can be shut out by the
next one's blocks, which keep theirs until the first has finished.  The order is checked in the source; the shapes where
both kernels' blocks fit on one SM and ask for more columns than it has run on the GPU."""
import re
from pathlib import Path

import numpy as np
import pytest

SOURCE = Path(__file__).resolve().parent.parent / "vllm_sly_radiance_b200" / "csrc" / "lora.cu"


def kernels():
    """name -> body, without comments."""
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    out = {}
    for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^)]*\) )?(\w+)\(", text):
        at = m.end()
        depth, i = 0, text.index("{", at)
        start = i
        while True:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
            if depth == 0:
                break
        out[m.group(1)] = text[start:i]
    return out


def test_tensor_memory_before_the_trigger():
    found = {n: b for n, b in kernels().items() if "tmem_alloc(" in b}
    assert set(found) == {"shrink128_kernel", "expand128_kernel", "shrink128_any_kernel", "expand128_any_kernel"}
    for name, body in found.items():
        assert body.count("tmem_alloc(") == body.count("pdl_trigger()") == 1, name
        alloc, trigger = body.index("tmem_alloc("), body.index("pdl_trigger()")
        assert "__syncthreads()" in body[alloc:trigger], name


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Kd,sizes,R", [
    (131, [41, 17, 9], 48),        # 144 rank rows: 256 columns a block beside the plain expand's 128
    (131, [264, 64], 16),          # 32 columns beside the expand with TMA, 256 a block
    (131, [264], 8)])
def test_prompts_whose_rows_tma_cannot_take(Kd, sizes, R, fp8):
    import torch
    from test_lora_gpu import make, run
    T = 128 * 150
    case = make(T, Kd, sizes, R, 3, fp8, seed=R)
    y, x, a, b, sc, rk, sl = case
    slots = np.random.default_rng(T).integers(-1, 3, T)
    got = run(*case, slots, tile_rows=128)
    xd = x[0].double() * x[1].double()[:, None] if fp8 else x.double()
    want, mag = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    for l in range(3):
        rows = torch.tensor(np.flatnonzero(slots == l))
        for s, (n0, n1) in enumerate(zip(sl, sl[1:])):
            A, B = a[l, s].double().t(), b[l, n0:n1].double().t()
            want[rows, n0:n1] += float(sc[l]) * (xd[rows] @ A @ B)
            mag[rows, n0:n1] = float(sc[l]) * (xd[rows].abs() @ A.abs() @ B.abs())
    # bf16 rounding of the result, 32-bit sums of Kd and R terms, the low-rank row as two bf16 numbers
    c = (Kd + R + 8) * 2.0 ** -24 + 2.0 ** -16
    assert not (~((got - want).abs() <= 2.0 ** -8 * (want.abs() + c * mag) + c * mag)).any()
