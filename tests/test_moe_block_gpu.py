"""The MoE block on the GPU against the same block on the CPU, and the MoE hybrid through the engine with decode graphs."""
import dataclasses

import pytest
import torch

import moe_oracle as M
from test_moe_block_cpu import ROUTERS, config
from vllm_sly_radiance_b200.config import EngineConfig
from vllm_sly_radiance_b200.engine.llm_engine import LLMEngine
from vllm_sly_radiance_b200.engine.request import SamplingParams
from vllm_sly_radiance_b200.models.hybrid import HybridModel, TPInfo
from vllm_sly_radiance_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pair(quant, router=None, tp=None):
    cfg = config(router or {})
    c = HybridModel(cfg, quant=quant, device="cpu", seed=0, tp=tp)
    g = HybridModel(cfg, quant=quant, device=DEV, seed=0, tp=tp, init_device="cpu")
    return c.layers[1].mlp, g.layers[1].mlp


def near(got, want):
    """Roundings to bf16: activations (on the CPU of both factors, the product, the shared rows too), expert rows and the sum on
    one side or the other, eight in all, each at most half a step; in the 2-norm their sum bounds the difference."""
    d = (got.cpu().double() - want.double()).norm()
    assert d <= 8 * M.BF16 * want.double().norm(), float(d / want.double().norm())


@pytest.mark.parametrize("router", ROUTERS)
@pytest.mark.parametrize("T", [1, 7, 64, 200])
def test_bf16_block(router, T):
    c, g = pair("bf16", router)
    x = torch.randn(T, 256, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    ids, _ = c.route(x)
    gi, _, _ = g._route_and_gate(x.to(DEV))
    assert torch.equal(gi.cpu(), ids)
    near(g.forward(x.to(DEV)), c.forward(x))
    assert K.check_status(DEV) == 0


@pytest.mark.parametrize("T", [1, 33, 300])
def test_block_scaled_block(T):
    """W4A8 experts: rows sorted and gathered by the plan, products as before, summed by token."""
    _, g = pair("mxfp4")
    x = torch.randn(T, 256, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
    q, s = K.quant_fp8(x)
    ids, w = g.route(x)
    got = g.local_experts(x, (q, s), ids, w)
    # the same rows, one token slot after another, by the path that expert parallelism takes
    want = torch.zeros(T, 256, device=DEV)
    for j in range(ids.shape[1]):
        want += w[:, j:j + 1] * g.expert_rows(q, s, None, ids[:, j]).float()
    near(got, want.cpu())


@pytest.mark.parametrize("quant", ["bf16", "mxfp4"])
def test_expert_slices_add_up(quant):
    """Expert parallelism over a tensor-parallel group: each rank's experts alone, the ranks' sums together."""
    x = torch.randn(40, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    _, whole = pair(quant)
    ids, w = whole.route(x)
    qs = K.quant_fp8(x) if quant == "mxfp4" else (None, None)
    want = whole.local_experts(x, qs, ids, w).float()
    parts = [pair(quant, tp=TPInfo(r, 2))[1] for r in range(2)]
    got = sum(p.local_experts(x, qs, ids, w).float() for p in parts)
    near(got, want.cpu())


def test_rows_of_one_expert_each():
    _, g = pair("bf16")
    x = torch.randn(50, 256, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    le = torch.randint(0, 16, (50,), device=DEV, generator=torch.Generator(DEV).manual_seed(0))
    y = g.expert_rows(None, None, x, le)
    p = K.moe_plan(le[:, None], 16)
    w = torch.ones(50, 1, device=DEV)
    _, _, up, down = g._banks
    assert torch.equal(y, K.moe_combine(K.linear_fused(K.linear_fused(x, up, plan=p, by_token=True), down, plan=p), p, w))


@pytest.mark.parametrize("quant", ["bf16", "mxfp4", "int4"])
def test_engine_with_decode_graphs(quant):
    """bf16 experts read counts on the host before: no decode graph could hold them."""
    prompts = [list(range(10, 60)), list(range(100, 131)), list(range(7, 27))]
    sp = SamplingParams(temperature=0, max_tokens=6, ignore_eos=True)

    def run(graphs):
        cfg = EngineConfig(model="tiny_moe", quantization=quant, kv_cache_dtype="bf16", device=DEV, max_model_len=512,
                           max_num_seqs=4, max_num_batched_tokens=256, num_kv_blocks=32, enable_cuda_graphs=graphs)
        e = LLMEngine(cfg)
        return [o.outputs[0].token_ids for o in e.generate(prompts, sp)]
    assert run(True) == run(False)
    assert K.check_status(DEV) == 0


def test_engine_with_another_router():
    cfg = EngineConfig(model="tiny_moe", quantization="bf16", device=DEV, max_model_len=512, max_num_seqs=4,
                       max_num_batched_tokens=256, num_kv_blocks=32)
    m = HybridModel(dataclasses.replace(config(ROUTERS[1])), quant="bf16", device=DEV, seed=0)
    out = LLMEngine(cfg, model=m).generate([list(range(10, 50))], SamplingParams(temperature=0, max_tokens=4, ignore_eos=True))
    assert len(out[0].outputs[0].token_ids) == 4
