"""Adapters, parallel samples and cache compaction through the engine (CPU)."""
import json

import pytest
import torch

from vllm_sly_radiance_b200.config import EngineConfig, tiny_hybrid
from vllm_sly_radiance_b200.engine.llm_engine import LLMEngine
from vllm_sly_radiance_b200.engine.request import SamplingParams

GREEDY = dict(temperature=0, ignore_eos=True)


def engine(device="cpu", quant="bf16", kv="bf16", **kw):
    a = dict(model="tiny_hybrid", device=device, max_model_len=512, max_num_seqs=4, max_num_batched_tokens=96,
             num_kv_blocks=48, quantization=quant, kv_cache_dtype=kv, enable_cuda_graphs=False, block_size=16)
    a.update(kw)
    return LLMEngine(EngineConfig(**a))


def modules(cfg, i):
    """(module, in features, out features) of layer i in the checkpoint's names."""
    H, I = cfg.hidden_size, cfg.intermediate_size
    m = [("mlp.gate_proj", H, I), ("mlp.up_proj", H, I), ("mlp.down_proj", I, H)]
    if cfg.is_attention_layer(i):
        q, kv = cfg.num_q_heads * cfg.head_dim, cfg.num_kv_heads * cfg.head_dim
        return m + [("self_attn.q_proj", H, 2 * q), ("self_attn.k_proj", H, kv), ("self_attn.v_proj", H, kv),
                    ("self_attn.o_proj", q, H)]
    return m + [("linear_attn.in_proj_qkvz", H, 2 * cfg.gdn_key_dim + 2 * cfg.gdn_value_dim),
                ("linear_attn.in_proj_ba", H, 2 * cfg.gdn_num_v_heads), ("linear_attn.out_proj", cfg.gdn_value_dim, H)]


def tensors(cfg, rank, seed, std=0.05):
    g = torch.Generator().manual_seed(seed)
    t = {}
    for i in range(cfg.num_layers):
        for name, k, n in modules(cfg, i):
            p = f"base_model.model.model.layers.{i}.{name}."
            t[p + "lora_A.weight"] = torch.randn(rank, k, generator=g) * k ** -0.5
            t[p + "lora_B.weight"] = torch.randn(n, rank, generator=g) * std
    return t


def save(path, cfg, rank, alpha, seed):
    from safetensors.torch import save_file
    path.mkdir()
    save_file(tensors(cfg, rank, seed), str(path / "adapter_model.safetensors"))
    (path / "adapter_config.json").write_text(json.dumps({"r": rank, "lora_alpha": alpha}))
    return str(path)


def tokens(out):
    return [o.outputs[0].token_ids for o in out]


def test_adapter_matches_merged_weights(tmp_path):
    """Logits with an adapter are those of the model with W + scale B A in its weights (bf16 rounds W again and the
    projection once more: compared in norm)."""
    cfg = tiny_hybrid()
    path = save(tmp_path / "a", cfg, 8, 16, 1)
    eng = engine(max_loras=2, max_lora_rank=8, lora_modules=f"a={path}")
    ref = engine()
    from vllm_sly_radiance_b200.quant.loaders import gdn_in_proj_permutation
    t, perm = tensors(cfg, 8, 1), gdn_in_proj_permutation(cfg)
    for i, layer in enumerate(ref.model.layers):
        d = {}
        for name, k, n in modules(cfg, i):
            p = f"base_model.model.model.layers.{i}.{name}."
            d[name] = 2.0 * t[p + "lora_B.weight"].to(torch.bfloat16).float() @ t[p + "lora_A.weight"].to(torch.bfloat16).float()
        m = layer.mixer
        if layer.is_attn:
            m.qkv.w = (m.qkv.w.float() + torch.cat([d[f"self_attn.{n}_proj"] for n in "qkv"])).to(torch.bfloat16)
            m.o_proj.w = (m.o_proj.w.float() + d["self_attn.o_proj"]).to(torch.bfloat16)
        else:
            w = torch.cat([d["linear_attn.in_proj_qkvz"][perm[0]], d["linear_attn.in_proj_ba"][perm[1]]])
            m.in_proj.w[:len(w)] = (m.in_proj.w[:len(w)].float() + w).to(torch.bfloat16)
            m.out_proj.w = (m.out_proj.w.float() + d["linear_attn.out_proj"]).to(torch.bfloat16)
        layer.mlp.gate_up.w = (layer.mlp.gate_up.w.float() + torch.cat([d["mlp.gate_proj"], d["mlp.up_proj"]])).to(torch.bfloat16)
        layer.mlp.down.w = (layer.mlp.down.w.float() + d["mlp.down_proj"]).to(torch.bfloat16)

    def logits(e, adapter=None):
        e.add_request(list(range(5, 60)), SamplingParams(max_tokens=1, **GREEDY), "r", adapter=adapter)
        s = e.scheduler.schedule()
        return e.runner.execute(s, want_logits=True).logits.float()
    with_adapter, merged = logits(eng, "a"), logits(ref)
    plain = logits(engine())
    assert float((with_adapter - merged).norm() / merged.norm()) < 0.05
    assert float((plain - merged).norm() / merged.norm()) > 0.3


def test_batch_of_adapters_equals_single_runs():
    cfg = tiny_hybrid()
    prompts = [list(range(9, 70)), list(range(9, 70)), list(range(300, 340)), list(range(9, 70))]
    names = ["x", None, "y", "y"]
    sp = SamplingParams(max_tokens=6, **GREEDY)

    def make():
        e = engine(max_loras=3, max_lora_rank=16)
        e.adapters.add_tensors("x", tensors(cfg, 4, 2), 4, 2.0)
        e.adapters.add_tensors("y", tensors(cfg, 16, 3), 16, 1.0)
        return e
    together = tokens(make().generate(prompts, sp, names))
    for p, n, t in zip(prompts, names, together):
        assert tokens(make().generate([p], sp, [n]))[0] == t
    assert together[1] == tokens(engine().generate([prompts[1]], sp))[0]     # no adapter: what ran before
    assert together[0] != together[1] and together[3] != together[1]


def test_prefix_cache_keeps_adapters_apart():
    cfg = tiny_hybrid()
    e = engine(max_loras=2, max_lora_rank=8, enable_prefix_caching=True)
    e.adapters.add_tensors("x", tensors(cfg, 8, 2), 8, 2.0)
    sp = SamplingParams(max_tokens=4, **GREEDY)
    p = list(range(20, 90))
    want = {n: tokens(e.generate([p], sp, n))[0] for n in (None, "x")}
    hits = e.kv.hits
    assert {n: tokens(e.generate([p], sp, n))[0] for n in (None, "x")} == want and e.kv.hits == hits + 2
    e.remove_adapter("x")
    e.adapters.add_tensors("x", tensors(cfg, 8, 7), 8, 2.0)                  # other weights, the same name
    assert tokens(e.generate([p], sp, "x"))[0] != want["x"] and e.kv.hits == hits + 2


def test_adapter_refusals(tmp_path):
    cfg = tiny_hybrid()
    with pytest.raises(ValueError):
        engine().add_request([1, 2], adapter="a")
    with pytest.raises(ValueError):
        engine().add_adapter("a", "nowhere")
    with pytest.raises(ValueError):
        engine(lora_modules="a=b")
    e = engine(max_loras=1, max_lora_rank=8)
    good = tensors(cfg, 8, 0)
    for bad, rank in ((good, 9), (tensors(cfg, 4, 0), 8), ({"layers.0.mlp.experts.0.up_proj.lora_A.weight": torch.zeros(8, 256)}, 8),
                      ({k: v for k, v in good.items() if "lora_B" not in k}, 8)):
        with pytest.raises(ValueError):
            e.adapters.add_tensors("a", bad, rank, 1.0)
    assert not e.adapters.slots and all(int(b.ranks.sum()) == 0 for bs in e.adapters.banks for b in bs.values())
    e.adapters.add_tensors("a", good, 8, 1.0)
    for name in ("a", "b"):                                # loaded already; no slot left
        with pytest.raises(ValueError):
            e.adapters.add_tensors(name, good, 8, 1.0)
    e.add_request([1, 2, 3], SamplingParams(max_tokens=2), "r", adapter="a")
    with pytest.raises(ValueError):
        e.remove_adapter("a")
    e.abort_request("r")
    e.remove_adapter("a")
    with pytest.raises(ValueError):
        e.remove_adapter("a")


@pytest.mark.parametrize("length", [1, 2, 16, 17, 33, 120])
@pytest.mark.parametrize("kv", ["bf16", "fp8", "int4"])
def test_greedy_samples_are_the_single_run(length, kv):
    """n greedy samples of one prompt, forked at every place in a page, are n times the single answer."""
    p = list(range(7, 7 + length))
    sp = SamplingParams(max_tokens=5, **GREEDY)
    one = tokens(engine(kv=kv).generate([p], sp))[0]
    e = engine(kv=kv)
    out = e.generate([p, list(range(400, 430))], [SamplingParams(max_tokens=5, n=3, **GREEDY), sp])
    assert [o.index for o in out[0].outputs] == [0, 1, 2] and out[0].finished
    assert [o.token_ids for o in out[0].outputs] == [one] * 3
    assert e.kv.blocks.num_free == e.num_blocks - 1 and not e.groups and not e.member and not e.requests


def test_samples_differ_and_share_the_prompt():
    e = engine()
    out = e.generate([list(range(50))], SamplingParams(temperature=1.0, top_k=50, max_tokens=8, n=4, seed=3, ignore_eos=True))[0]
    assert len({tuple(o.token_ids) for o in out.outputs}) == 4
    e.add_request(list(range(40)), SamplingParams(max_tokens=50, n=3, **GREEDY), "g")
    while not e.scheduler.running or len(e.scheduler.running) < 3:
        e.step()
    a, b, c = (set(r.block_ids) for r in e.scheduler.running)
    assert len(a & b & c) == 2                             # 39 tokens: two full pages shared, the third copied
    assert e.abort_request("g") and not e.requests and e.kv.blocks.num_free == e.num_blocks - 1


def test_more_samples_than_room():
    """Samples that find no slot or block wait, and give the same answer."""
    sp = SamplingParams(max_tokens=4, n=7, **GREEDY)
    p = list(range(60, 100))
    one = tokens(engine().generate([p], SamplingParams(max_tokens=4, **GREEDY)))[0]
    for kw in (dict(max_num_seqs=2), dict(num_kv_blocks=8)):
        out = engine(**kw).generate([p], sp)[0]
        assert [o.token_ids for o in out.outputs] == [one] * 7


def test_samples_with_prefix_cache():
    sp = SamplingParams(max_tokens=4, n=3, **GREEDY)
    p = list(range(60, 109))                               # 49 tokens: the cached prefix ends before the last one
    e = engine(enable_prefix_caching=True)
    first = [o.token_ids for o in e.generate([p], sp)[0].outputs]
    again = [o.token_ids for o in e.generate([p], sp)[0].outputs]
    assert first == again and e.kv.hits >= 1


def test_n_refusals():
    with pytest.raises(ValueError):
        SamplingParams(n=0)
    with pytest.raises(ValueError):
        engine(speculative_method="lookup").add_request([1, 2, 3], SamplingParams(n=2))


@pytest.mark.parametrize("caching", [False, True])
def test_compaction_between_steps(caching):
    """Requests go on unchanged after their blocks moved; shared and cached blocks move once."""
    prompts = [list(range(i, i + 40 + 7 * i)) for i in range(1, 5)]
    params = [SamplingParams(max_tokens=m, **GREEDY) for m in (2, 12, 3, 12)]
    want = tokens(engine(enable_prefix_caching=caching).generate(prompts, params))
    e = engine(enable_prefix_caching=caching)
    ids = [e.add_request(p, s) for p, s in zip(prompts, params)]
    got = {}
    k = 0
    while e.has_unfinished_requests():
        for o in e.step():
            if o.finished:
                got[o.request_id] = o.outputs[0].token_ids
        k += 1
        if k in (3, 6, 9):
            n = e.compact_cache()
            live = {b for r in e.scheduler.running for b in r.block_ids} | set(e.kv.lru)
            assert live == set(range(1, n + 1)) and e.kv.blocks.num_free == e.num_blocks - 1 - n
    assert [got[i] for i in ids] == want
    if caching:
        hits = e.kv.hits
        assert tokens(e.generate([prompts[1]], params[1]))[0] == want[1] and e.kv.hits == hits + 1
