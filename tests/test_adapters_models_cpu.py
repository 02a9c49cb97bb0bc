"""Adapters on the MoE hybrid (its mixers' projections) and with speculative decoding (CPU)."""
import pytest
import torch

from test_adapters_cpu import GREEDY, engine, modules, tensors, tokens
from vllm_sly_radiance_b200.config import tiny_hybrid, tiny_moe
from vllm_sly_radiance_b200.engine.request import SamplingParams


def moe_tensors(rank, seed, std=0.05):
    g = torch.Generator().manual_seed(seed)
    cfg, t = tiny_moe(), {}
    for i in range(cfg.num_layers):
        for name, k, n in modules(cfg, i):
            if not name.startswith("mlp."):
                p = f"base_model.model.model.layers.{i}.{name}."
                t[p + "lora_A.weight"] = torch.randn(rank, k, generator=g) * k ** -0.5
                t[p + "lora_B.weight"] = torch.randn(n, rank, generator=g) * std
    return t


def logits(e, adapter=None):
    e.add_request(list(range(5, 60)), SamplingParams(max_tokens=1, **GREEDY), "r", adapter=adapter)
    return e.runner.execute(e.scheduler.schedule(), want_logits=True).logits.float()


def test_moe_hybrid_matches_merged_weights():
    """Adapters on the mixers of the MoE hybrid: as with W + scale B A in the weights (bf16 rounds W again, and a router
    near a tie may pick another expert: compared in norm)."""
    from vllm_sly_radiance_b200.quant.loaders import gdn_in_proj_permutation
    cfg = tiny_moe()
    eng, ref = engine(model="tiny_moe", max_loras=2, max_lora_rank=8), engine(model="tiny_moe")
    t, perm = moe_tensors(8, 1), gdn_in_proj_permutation(cfg)
    eng.adapters.add_tensors("other", moe_tensors(4, 5), 4, 1.0)
    eng.adapters.add_tensors("a", t, 8, 2.0)
    for i, layer in enumerate(ref.model.layers):
        d = {}
        for name, k, n in modules(cfg, i):
            p = f"base_model.model.model.layers.{i}.{name}."
            if p + "lora_A.weight" in t:
                d[name] = 2.0 * t[p + "lora_B.weight"].to(torch.bfloat16).float() @ t[p + "lora_A.weight"].to(torch.bfloat16).float()
        m = layer.mixer
        if layer.is_attn:
            m.qkv.w = (m.qkv.w.float() + torch.cat([d[f"self_attn.{n}_proj"] for n in "qkv"])).to(torch.bfloat16)
            m.o_proj.w = (m.o_proj.w.float() + d["self_attn.o_proj"]).to(torch.bfloat16)
        else:
            w = torch.cat([d["linear_attn.in_proj_qkvz"][perm[0]], d["linear_attn.in_proj_ba"][perm[1]]])
            m.in_proj.w[:len(w)] = (m.in_proj.w[:len(w)].float() + w).to(torch.bfloat16)
            m.out_proj.w = (m.out_proj.w.float() + d["linear_attn.out_proj"]).to(torch.bfloat16)
    plain, merged = logits(engine(model="tiny_moe")), logits(ref)
    assert float((logits(eng, "a") - merged).norm() / merged.norm()) < 0.1
    assert float((plain - merged).norm() / merged.norm()) > 0.3


def test_moe_hybrid_batch_equals_single_runs():
    def make():
        e = engine(model="tiny_moe", max_loras=2, max_lora_rank=8)
        e.adapters.add_tensors("x", moe_tensors(8, 2), 8, 2.0)
        return e
    sp = SamplingParams(max_tokens=5, **GREEDY)
    prompts, names = [list(range(9, 60)), list(range(9, 60)), list(range(300, 330))], ["x", None, "x"]
    together = tokens(make().generate(prompts, sp, names))
    assert together == [tokens(make().generate([p], sp, n))[0] for p, n in zip(prompts, names)]
    assert together[0] != together[1] and together[1] == tokens(engine(model="tiny_moe").generate([prompts[1]], sp))[0]
    with pytest.raises(ValueError):                        # experts have no adapters
        make().adapters.add_tensors("y", tensors(tiny_hybrid(), 8, 0), 8, 1.0)


@pytest.mark.parametrize("method", ["lookup", "dflash2", "mtp"])
def test_speculative_decoding_keeps_the_answers(method):
    """Greedy answers under adapters with drafts to verify are those without, requests with and without adapters mixed."""
    def make(**kw):
        e = engine(max_loras=2, max_lora_rank=16, **kw)
        e.adapters.add_tensors("x", tensors(tiny_hybrid(), 4, 2), 4, 2.0)
        e.adapters.add_tensors("y", tensors(tiny_hybrid(), 16, 3), 16, 1.0)
        return e
    sp = SamplingParams(max_tokens=14, **GREEDY)
    prompts = [[5, 6, 7, 8] * 12, list(range(9, 70)), [5, 6, 7, 8] * 12]
    names = ["x", None, "y"]
    want = tokens(make().generate(prompts, sp, names))
    e = make(speculative_method=method, num_speculative_tokens=4)
    if method == "lookup":
        def propose(sched, sampled):             # partly right drafts: the answer with every third token wrong
            for q in sched.seqs:
                t = sampled.get(q.req.request_id)
                n = len(q.req.output_token_ids) + len(t or [])
                d = want[names.index(q.req.adapter)][n:n + 4] if t else []
                q.req.draft_token_ids = [(v + 1) % 4096 if (n + i) % 3 == 2 else v for i, v in enumerate(d)]
        e.spec._propose = propose
    assert tokens(e.generate(prompts, sp, names)) == want
    assert e.spec.stats["draft_tokens"] > 0
