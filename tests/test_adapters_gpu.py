"""Adapters, parallel samples and cache compaction through the engine's CUDA kernels and graphs."""
import pytest
import torch

from test_adapters_cpu import GREEDY, engine, tensors, tokens
from vllm_sly_radiance_b200.config import tiny_hybrid
from vllm_sly_radiance_b200.engine.request import SamplingParams
from vllm_sly_radiance_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
PROMPTS = [list(range(9, 70)), list(range(9, 70)), list(range(300, 340)), list(range(9, 170))]
NAMES = ["x", None, "y", "y"]


def make(quant="bf16", kv="bf16", graphs=False, std=0.05, **kw):
    cfg = tiny_hybrid()
    e = engine("cuda", quant, kv, enable_cuda_graphs=graphs, max_loras=3, max_lora_rank=16, **kw)
    e.adapters.add_tensors("x", tensors(cfg, 4, 2, std), 4, 2.0)
    e.adapters.add_tensors("y", tensors(cfg, 16, 3, std), 16, 1.0)
    return e


def test_bf16_logits_match_the_cpu():
    """One prefill step of three prompts with different adapters: GPU kernels against the CPU form."""
    outs = []
    for dev in ("cpu", "cuda"):
        cfg = tiny_hybrid()
        from vllm_sly_radiance_b200.config import EngineConfig
        from vllm_sly_radiance_b200.engine.llm_engine import LLMEngine
        from vllm_sly_radiance_b200.models.hybrid import HybridModel
        model = HybridModel(cfg, quant="bf16", device=dev, seed=0, init_device="cpu")
        e = LLMEngine(EngineConfig(model="tiny_hybrid", device=dev, max_model_len=512, max_num_batched_tokens=512, num_kv_blocks=48,
                                   quantization="bf16", kv_cache_dtype="bf16", block_size=16, enable_cuda_graphs=False,
                                   max_loras=3, max_lora_rank=16), model=model)
        e.adapters.add_tensors("x", tensors(cfg, 4, 2), 4, 2.0)
        e.adapters.add_tensors("y", tensors(cfg, 16, 3), 16, 1.0)
        for p, n in zip(PROMPTS, NAMES):
            e.add_request(p, SamplingParams(max_tokens=1, **GREEDY), adapter=n)
        outs.append(e.runner.execute(e.scheduler.schedule(), want_logits=True).logits.float().cpu())
    assert float((outs[1] - outs[0]).norm() / outs[0].norm()) < 2e-2


@pytest.mark.parametrize("quant,kv", [("bf16", "bf16"), ("mxfp4", "fp8"), ("mxfp4", "int4")])
def test_graphs_equal_eager(quant, kv):
    """Decode graphs that follow the plan buffer, batches with and without adapters in turn."""
    sp = SamplingParams(max_tokens=10, **GREEDY)
    res = []
    for graphs in (False, True):
        e = make(quant, kv, graphs)
        res.append((tokens(e.generate(PROMPTS, sp, NAMES)), tokens(e.generate(PROMPTS, sp)),
                    tokens(e.generate(PROMPTS[:2], sp, ["y", "x"]))))
        K.check_status(e.device)
    assert res[0] == res[1]
    assert res[0][0] != res[0][1]


@pytest.mark.parametrize("quant", ["bf16", "mxfp4", "int4"])
def test_zero_adapter_changes_nothing(quant):
    sp = SamplingParams(max_tokens=8, **GREEDY)
    e = make(quant, "fp8", graphs=True, std=0.0)
    assert tokens(e.generate(PROMPTS, sp, NAMES)) == tokens(e.generate(PROMPTS, sp))


@pytest.mark.parametrize("kv", ["bf16", "fp8", "int4"])
def test_samples_and_compaction(kv):
    """Greedy samples under an adapter are the single run's answer, with the pool compacted on the way."""
    sp = SamplingParams(max_tokens=9, **GREEDY)
    want = tokens(make(kv=kv).generate([PROMPTS[0]], sp, "y"))[0]
    e = make(kv=kv)
    other = e.add_request(PROMPTS[2], SamplingParams(max_tokens=3, **GREEDY))
    e.add_request(PROMPTS[0], SamplingParams(max_tokens=9, n=3, **GREEDY), "g", adapter="y")
    got, k = {}, 0
    while e.has_unfinished_requests():
        for o in e.step():
            if o.finished:
                got[o.request_id] = [c.token_ids for c in o.outputs]
        k += 1
        if k % 3 == 0:
            e.compact_cache()
    assert got["g"] == [want] * 3 and len(got[other][0]) == 3
    K.check_status(e.device)
