"""MoE blocks of sizes beyond the kernels' on the GPU, without a shared expert, and routed rows without a stop for the host."""
import pytest
import torch

from test_moe_block_gpu import near
from test_moe_sizes_cpu import MANY_A_TOKEN, MANY_EXPERTS, block, x_of
from vllm_sly_radiance_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("sizes", [MANY_A_TOKEN, MANY_EXPERTS], ids=["40 a token", "1100 experts"])
@pytest.mark.parametrize("T", [1, 50])
def test_bf16_block_of_any_size(sizes, T):
    c, g = block(**sizes), block(device=DEV, **sizes)
    near(g.forward(x_of(T).to(DEV)), c.forward(x_of(T)))


@pytest.mark.parametrize("sizes", [dict(MANY_A_TOKEN, moe_intermediate_size=128), dict(MANY_EXPERTS, moe_intermediate_size=128)],
                         ids=["40 a token", "1100 experts"])
@pytest.mark.parametrize("T", [1, 50])
def test_block_scaled_block_of_any_size(sizes, T):
    g = block("mxfp4", DEV, **sizes)
    x = x_of(T).to(DEV)
    q, s = K.quant_fp8(x)
    ids, w = g.route(x)
    got = g.local_experts(x, (q, s), ids, w)
    want = torch.zeros(T, 256, device=DEV)
    for j in range(ids.shape[1]):
        want += w[:, j:j + 1] * g.expert_rows(q, s, None, ids[:, j]).float()
    near(got, want.cpu())
    assert g.forward(x).isfinite().all() and K.check_status(DEV) == 0


@pytest.mark.parametrize("sizes", [MANY_A_TOKEN, MANY_EXPERTS], ids=["40 a token", "1100 experts"])
def test_block_scaled_block_of_any_size_in_a_graph(sizes):
    g = block("mxfp4", DEV, **dict(sizes, moe_intermediate_size=128))
    x = x_of(3).to(DEV)
    want = g.forward(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = g.forward(x)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_block_without_shared_expert():
    c, g = (block(device=d, shared_expert_intermediate_size=0) for d in ("cpu", DEV))
    near(g.forward(x_of(20).to(DEV)), c.forward(x_of(20)))
    assert K.check_status(DEV) == 0


def test_rows_by_expert_do_not_stop_for_the_host():
    g = block(device=DEV)
    x, le = x_of(50).to(DEV), torch.randint(0, 16, (50,), generator=torch.Generator().manual_seed(0)).to(DEV)
    want = g.expert_rows(None, None, x, le)
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = g.expert_rows(None, None, x, le)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(got, want)
