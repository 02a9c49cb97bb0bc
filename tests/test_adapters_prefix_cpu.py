"""Cached prefixes of different adapters are told apart whatever the adapters' names, loads and the prompts' tokens."""
import itertools

from test_adapters_cpu import GREEDY, engine, tensors, tokens
from vllm_sly_radiance_b200.config import tiny_hybrid
from vllm_sly_radiance_b200.engine.kv_cache import KVCacheManager
from vllm_sly_radiance_b200.engine.request import SamplingParams


def test_hashes_of_salts_that_run_into_the_tokens():
    kv = KVCacheManager(8, 4, 2)
    rest = [20, 21, 22, 23, 24, 25, 26]
    salts, firsts = ["", "x#1", "x#11", "x#1,1", "x#", "x#12", "1", "12"], [2, 12, 112, 1, 11]
    seen = {}
    for salt, first in itertools.product(salts, firsts):
        for i, h in enumerate(kv._hashes([first] + rest, salt)):
            assert seen.setdefault(h, (salt, first, i)) == (salt, first, i)


def test_eleventh_load_under_the_same_name():
    """Load 1 with a prompt that starts with token 12, load 11 with one that starts with token 2 and goes on alike."""
    cfg = tiny_hybrid()
    sp = SamplingParams(max_tokens=4, **GREEDY)
    e = engine(max_loras=1, max_lora_rank=8, enable_prefix_caching=True)
    e.adapters.add_tensors("x", tensors(cfg, 8, 2), 8, 2.0)
    e.generate([[12] + list(range(20, 90))], sp, "x")
    for _ in range(10):
        e.remove_adapter("x")
        e.adapters.add_tensors("x", tensors(cfg, 8, 7), 8, 2.0)
    hits = e.kv.hits
    got = tokens(e.generate([[2] + list(range(20, 90))], sp, "x"))
    fresh = engine(max_loras=1, max_lora_rank=8)
    fresh.adapters.add_tensors("x", tensors(cfg, 8, 7), 8, 2.0)
    assert e.kv.hits == hits and got == tokens(fresh.generate([[2] + list(range(20, 90))], sp, "x"))
