"""Adapters behind the data-parallel front end and its server: every replica has them, requests can name them."""
import pytest
from fastapi.testclient import TestClient

from test_adapters_cpu import GREEDY, engine, save, tokens
from vllm_sly_radiance_b200.config import EngineConfig, tiny_hybrid
from vllm_sly_radiance_b200.engine.request import SamplingParams
from vllm_sly_radiance_b200.entrypoints.dp import DataParallelEngine
from vllm_sly_radiance_b200.entrypoints.openai_server import build_app


@pytest.mark.timeout(600)
def test_adapters_behind_two_replicas(tmp_path):
    path = save(tmp_path / "a", tiny_hybrid(), 8, 16, 1)
    kw = dict(max_loras=1, max_lora_rank=8, lora_modules=f"a={path}")
    prompts, names = [list(range(5 + i, 40 + i)) for i in range(4)], ["a", None, None, "a"]
    sp = SamplingParams(max_tokens=4, **GREEDY)
    one = engine(**kw)                           # one request at a time: rows of a batch may differ by a rounding
    want = [tokens(one.generate([p], sp, [n]))[0] for p, n in zip(prompts, names)]
    assert want[0] != tokens(engine().generate(prompts[:1], sp))[0]
    dp = DataParallelEngine(EngineConfig(model="tiny_hybrid", device="cpu", max_model_len=512, max_num_seqs=4, max_num_batched_tokens=96,
                                         num_kv_blocks=48, quantization="bf16", kv_cache_dtype="bf16", enable_cuda_graphs=False,
                                         block_size=16, **kw), 2)
    try:
        assert dp.adapter_names == ["a"]
        for i in (0, 2):                         # two requests at once, one on each replica
            assert tokens(dp.generate(prompts[i:i + 2], sp, names[i:i + 2])) == want[i:i + 2]
        with pytest.raises(ValueError):
            dp.add_request(prompts[0], sp, adapter="b")
        with pytest.raises(ValueError):
            dp.generate(prompts, sp, ["a"])
        assert not dp.has_unfinished_requests()
        with pytest.raises(ValueError):
            build_app(dp, "a")
        with TestClient(build_app(dp, "base")) as c:
            assert [m["id"] for m in c.get("/v1/models").json()["data"]] == ["base", "a"]
            for model in ("base", "a"):
                r = c.post("/v1/completions", json={"model": model, "prompt": prompts[0], "max_tokens": 4, "temperature": 0,
                                                    "ignore_eos": True}).json()
                assert r["model"] == model and (r["choices"][0]["token_ids"] == want[0]) == (model == "a")
            c.app.state.engine_loop.running = False
    finally:
        dp.shutdown()


def test_modules_without_slots_are_refused_before_any_replica_starts():
    with pytest.raises(ValueError):
        DataParallelEngine(EngineConfig(model="tiny_hybrid", device="cpu", lora_modules="a=b"), 2)
