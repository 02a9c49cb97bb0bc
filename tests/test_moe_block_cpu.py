"""The MoE block's router by configuration, and its parts, on the CPU."""
import dataclasses

import pytest
import torch

import moe_oracle as M
from vllm_sly_radiance_b200.config import EngineConfig, ModelConfig, config_from_hf, tiny_moe
from vllm_sly_radiance_b200.engine.llm_engine import LLMEngine
from vllm_sly_radiance_b200.engine.request import SamplingParams
from vllm_sly_radiance_b200.models.hybrid import HybridModel

ROUTERS = [dict(), dict(moe_score="sigmoid", moe_router_bias=True, moe_num_groups=4, moe_top_groups=2, moe_routed_scale=2.5),
           dict(moe_renormalize=False)]


def config(router):
    return dataclasses.replace(tiny_moe(), **router)


@pytest.mark.parametrize("router", ROUTERS)
def test_router_by_configuration(router):
    blk = HybridModel(config(router), quant="bf16", device="cpu", seed=3).layers[1].mlp
    x = torch.randn(9, 256, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    ids, w = blk.route(x)
    c = blk.cfg
    want_ids, want = M.route(x.float() @ blk.router.float().t(), 4, c.moe_score, blk.router_bias, c.moe_num_groups,
                             c.moe_top_groups, c.moe_renormalize, c.moe_routed_scale)
    assert (blk.router_bias is not None) == c.moe_router_bias
    assert torch.equal(ids, want_ids) and torch.allclose(w.double(), want, rtol=1e-6)


@pytest.mark.parametrize("router", ROUTERS[1:])
def test_model_with_such_a_router_generates(router):
    cfg = EngineConfig(model="tiny_moe", device="cpu", max_model_len=512, max_num_seqs=2, max_num_batched_tokens=128,
                       num_kv_blocks=32)
    eng = LLMEngine(cfg, model=HybridModel(config(router), quant="bf16", device="cpu", seed=0))
    out = eng.generate([list(range(10, 50))], SamplingParams(temperature=0, max_tokens=4, ignore_eos=True))
    assert len(out[0].outputs[0].token_ids) == 4


def test_router_keys_of_a_checkpoint():
    base = dict(vocab_size=64, hidden_size=64, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
                num_experts=16, num_experts_per_tok=4, model_type="x")
    c = config_from_hf(base)
    assert (c.moe_score, c.moe_router_bias, c.moe_num_groups, c.moe_renormalize, c.moe_routed_scale) == \
        ("softmax", False, 1, True, 1.0)
    c = config_from_hf({**base, "scoring_func": "sigmoid", "topk_method": "noaux_tc", "n_group": 8, "topk_group": 4,
                        "norm_topk_prob": False, "routed_scaling_factor": 2.5})
    assert (c.moe_score, c.moe_router_bias, c.moe_num_groups, c.moe_top_groups, c.moe_renormalize, c.moe_routed_scale) == \
        ("sigmoid", True, 8, 4, False, 2.5)
    assert ModelConfig.from_dict({"moe_score": "sigmoid"}).moe_score == "sigmoid"
