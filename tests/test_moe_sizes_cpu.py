"""MoE blocks of sizes beyond the kernels', routers that no block can have, and the router's keys of a checkpoint."""
import dataclasses

import pytest
import torch

import moe_oracle as M
from vllm_sly_radiance_b200.config import config_from_hf, tiny_moe
from vllm_sly_radiance_b200.models.hybrid import TPInfo
from vllm_sly_radiance_b200.models.moe import MoEBlock
from vllm_sly_radiance_b200.models.weights import RandomWeights


def block(quant="bf16", device="cpu", **sizes):
    cfg = dataclasses.replace(tiny_moe(), **sizes)
    blk = MoEBlock(cfg, TPInfo(), quant, RandomWeights(cfg, 0, "cpu"), "layers.1.")
    return blk.to(device) if device != "cpu" else blk


def x_of(T):
    return torch.randn(T, 256, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)


MANY_A_TOKEN = dict(num_experts=64, num_experts_per_tok=40, moe_intermediate_size=32)
MANY_EXPERTS = dict(num_experts=1100, num_experts_per_tok=4, moe_intermediate_size=32)


@pytest.mark.parametrize("sizes", [MANY_A_TOKEN, MANY_EXPERTS])
def test_block_of_any_size(sizes):
    blk, x = block(**sizes), x_of(6)
    ids, w = blk.route(x)
    want_ids, want = M.route(x.float() @ blk.router.float().t(), sizes["num_experts_per_tok"])
    assert torch.equal(ids, want_ids) and torch.allclose(w.double(), want, rtol=1e-6)
    assert blk.forward(x).isfinite().all()


@pytest.mark.parametrize("router", [dict(moe_score="tanh"), dict(moe_num_groups=3), dict(moe_num_groups=4, moe_top_groups=5),
                                    dict(moe_num_groups=8, moe_top_groups=1), dict(moe_num_groups=0),
                                    dict(moe_num_groups=16, moe_top_groups=8, moe_router_bias=True),
                                    dict(num_experts_per_tok=17), dict(num_experts_per_tok=0)])
def test_router_that_cannot_be_is_refused_at_load(router):
    """Not by the first forward pass."""
    with pytest.raises(ValueError, match="MoE"):
        block(**router)


def test_greedy_choice_knows_no_groups():
    base = dict(vocab_size=64, hidden_size=64, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
                num_experts=16, num_experts_per_tok=4, model_type="x", n_group=8, topk_group=3)
    assert config_from_hf({**base, "topk_method": "greedy"}).moe_num_groups == 1
    assert config_from_hf({**base, "topk_method": "group_limited_greedy"}).moe_num_groups == 8
    assert config_from_hf(base).moe_num_groups == 8


def test_router_bias_of_a_checkpoint(tmp_path):
    """``mlp.gate.e_score_correction_bias`` stays in 32 bits."""
    from safetensors.torch import save_file
    from vllm_sly_radiance_b200.quant.loaders import CheckpointWeights
    bias = torch.randn(16, generator=torch.Generator().manual_seed(0))
    save_file({"model.layers.1.mlp.gate.e_score_correction_bias": bias, "model.norm.weight": torch.ones(4)},
              str(tmp_path / "model.safetensors"))
    W = CheckpointWeights(str(tmp_path), dataclasses.replace(tiny_moe(), moe_router_bias=True))
    got = W.tensor("layers.1.router_bias", (16,), "router_bias")
    assert got.dtype == torch.float32 and torch.equal(got, bias)
