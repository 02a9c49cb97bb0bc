"""Decode graphs of steps with adapters are captured at start, as those of steps without."""
import pytest
import torch

from test_adapters_cpu import GREEDY, engine, tensors, tokens
from vllm_sly_radiance_b200.config import tiny_hybrid
from vllm_sly_radiance_b200.engine.request import SamplingParams

PLAIN = {(b, m) for b in (1, 2, 4) for m in ("greedy", "window")}


@pytest.mark.parametrize("slots", [0, 2])
def test_keys_captured_at_start(monkeypatch, slots):
    e = engine(**(dict(max_loras=slots, max_lora_rank=8) if slots else {}))
    e.runner.enable_graphs = True
    plans = []
    monkeypatch.setattr(e.runner, "_capture", lambda bucket, mode, meta, ids: plans.append(meta.adapter_plan) or {})
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    e.runner.capture_all()
    assert set(e.runner.graphs) == PLAIN | ({k + ("adapters",) for k in PLAIN} if slots else set())
    assert sum(p is not None for p in plans) == (len(PLAIN) if slots else 0)


@pytest.mark.gpu
def test_no_capture_inside_a_step_with_adapters():
    e = engine("cuda", "mxfp4", "fp8", enable_cuda_graphs=True, max_loras=2, max_lora_rank=8)
    e.adapters.add_tensors("x", tensors(tiny_hybrid(), 8, 2), 8, 2.0)
    before = set(e.runner.graphs)
    assert before == PLAIN | {k + ("adapters",) for k in PLAIN}
    prompts = [list(range(9 + i, 60 + i)) for i in range(4)]
    greedy = SamplingParams(max_tokens=6, **GREEDY)
    drawn = SamplingParams(temperature=0.8, top_k=20, seed=1, max_tokens=6, ignore_eos=True)
    for n in (1, 2, 3, 4):
        for p in (greedy, drawn):
            e.generate(prompts[:n], p, ["x"] + [None] * (n - 1))
    assert set(e.runner.graphs) == before
    plain = engine("cuda", "mxfp4", "fp8", enable_cuda_graphs=False, max_loras=2, max_lora_rank=8)
    plain.adapters.add_tensors("x", tensors(tiny_hybrid(), 8, 2), 8, 2.0)
    assert tokens(e.generate(prompts, greedy, "x")) == tokens(plain.generate(prompts, greedy, "x"))
