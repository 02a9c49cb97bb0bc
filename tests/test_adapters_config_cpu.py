"""Adapter directories whose configuration means something else than one alpha / r for every matrix are refused."""
import json

import pytest

from test_adapters_cpu import engine, save
from vllm_sly_radiance_b200.config import tiny_hybrid


@pytest.mark.parametrize("extra", [
    {"alpha_pattern": {"q_proj": 32}}, {"rank_pattern": {"q_proj": 4}}, {"use_dora": True}, {"bias": "lora_only"},
    {"lora_bias": True}, {"modules_to_save": ["lm_head"]}, {"layer_replication": [[0, 2], [1, 3]]},
    {"trainable_token_indices": [1]}, {"alora_invocation_tokens": [5, 6]}, {"peft_type": "IA3"}])
def test_refused_configurations(tmp_path, extra):
    path = save(tmp_path / "a", tiny_hybrid(), 8, 16, 1)
    cfg = {"r": 8, "lora_alpha": 16}
    (tmp_path / "a" / "adapter_config.json").write_text(json.dumps({**cfg, **extra}))
    e = engine(max_loras=1, max_lora_rank=8)
    with pytest.raises(ValueError, match=next(iter(extra))):
        e.add_adapter("a", path)
    assert not e.adapters.slots and all(int(b.ranks.sum()) == 0 for bs in e.adapters.banks for b in bs.values())


def test_configurations_that_change_nothing(tmp_path):
    """What PEFT writes when none of these is used."""
    path = save(tmp_path / "a", tiny_hybrid(), 8, 16, 1)
    (tmp_path / "a" / "adapter_config.json").write_text(json.dumps({
        "peft_type": "LORA", "r": 8, "lora_alpha": 16, "alpha_pattern": {}, "rank_pattern": {}, "use_dora": False, "bias": "none",
        "lora_bias": False, "modules_to_save": None, "layer_replication": None, "trainable_token_indices": None}))
    e = engine(max_loras=1, max_lora_rank=8)
    e.add_adapter("a", path)
    assert float(next(iter(e.adapters.banks[0].values())).scale[0]) == 2.0
