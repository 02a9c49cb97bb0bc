"""Two adapters and four samples of one prompt in one batch, on the tiny random-weight model.

    python examples/adapters_and_samples.py [cuda|cpu]
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from vllm_sly_radiance_b200 import LLM, SamplingParams          # noqa: E402


def random_adapter(adapters, rank, seed):
    """Low-rank matrices for the MLP of every layer, under the names of a PEFT checkpoint."""
    g = torch.Generator().manual_seed(seed)
    t = {}
    for i, banks in enumerate(adapters.banks):
        for module, lin, n in (("gate_proj", "gate_up", 2), ("up_proj", "gate_up", 2), ("down_proj", "down", 1)):
            b = banks[lin]
            t[f"model.layers.{i}.mlp.{module}.lora_A.weight"] = torch.randn(rank, b.K, generator=g) * b.K ** -0.5
            t[f"model.layers.{i}.mlp.{module}.lora_B.weight"] = torch.randn(b.N // n, rank, generator=g) * 0.1
    return t


def main(device):
    llm = LLM("tiny_hybrid", device=device, max_loras=2, max_lora_rank=16, max_model_len=512, num_kv_blocks=64)
    for k, name in enumerate(("first", "second")):
        llm.engine.adapters.add_tensors(name, random_adapter(llm.engine.adapters, 8, k), rank=8, scale=2.0)
    prompt = list(range(10, 80))
    greedy = SamplingParams(temperature=0, max_tokens=8, ignore_eos=True)
    samples = SamplingParams(temperature=0.8, top_k=50, n=4, seed=0, max_tokens=8, ignore_eos=True)
    names = [None, "first", "second", "first"]
    for name, out in zip(names, llm.generate([prompt] * 4, [greedy, greedy, greedy, samples], adapters=names)):
        for o in out.outputs:
            print(f"{name or 'no adapter':>10}  sample {o.index}: {o.token_ids}")
    print("blocks in use after compaction:", llm.engine.compact_cache())


if __name__ == "__main__":
    main(sys.argv[1] if len(sys.argv) > 1 else ("cuda" if torch.cuda.is_available() else "cpu"))
