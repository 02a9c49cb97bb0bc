"""Engine calls around adapters and samples that must not lose a request."""
import pytest

from test_adapters_cpu import GREEDY, engine, tensors
from vllm_sly_radiance_b200.config import tiny_hybrid
from vllm_sly_radiance_b200.engine.request import SamplingParams


def test_generate_refuses_adapters_of_another_length():
    """A shorter list left the last prompts without an answer."""
    e = engine(max_loras=1, max_lora_rank=8)
    e.adapters.add_tensors("x", tensors(tiny_hybrid(), 8, 2), 8, 2.0)
    sp = SamplingParams(max_tokens=2, **GREEDY)
    for names in (["x"], ["x"] * 3, []):
        with pytest.raises(ValueError):
            e.generate([[1, 2, 3], [4, 5, 6]], sp, names)
    assert not e.requests and len(e.generate([[1, 2, 3], [4, 5, 6]], sp, ["x", None])) == 2
