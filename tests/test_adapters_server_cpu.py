"""Adapters and parallel samples through the OpenAI-compatible server (CPU)."""
import json

import pytest
from fastapi.testclient import TestClient

from test_adapters_cpu import engine, tensors
from vllm_sly_radiance_b200.config import tiny_hybrid
from vllm_sly_radiance_b200.entrypoints.openai_server import build_app

BODY = {"prompt": "hello world", "max_tokens": 5, "temperature": 0, "ignore_eos": True}


@pytest.fixture(scope="module")
def served():
    e = engine(max_loras=3, max_lora_rank=8)
    e.adapters.add_tensors("x", tensors(tiny_hybrid(), 8, 2), 8, 2.0)
    with TestClient(build_app(e, "tiny,alias")) as c:
        yield e, c


def post(c, path="/v1/completions", **body):
    return c.post(path, json={**BODY, **body})


def test_adapter_is_a_model_of_its_own(served):
    e, c = served
    assert [m["id"] for m in c.get("/v1/models").json()["data"]] == ["tiny", "alias", "x"]
    base, x = post(c, model="tiny").json(), post(c, model="x").json()
    assert (base["model"], x["model"]) == ("tiny", "x")
    assert base["choices"][0]["token_ids"] != x["choices"][0]["token_ids"]
    assert post(c, model="y").status_code == 404


def test_an_adapter_cannot_take_the_base_models_name(served):
    e, c = served
    with pytest.raises(ValueError):
        e.adapters.add_tensors("alias", tensors(tiny_hybrid(), 8, 2), 8, 2.0)
    assert [m["id"] for m in c.get("/v1/models").json()["data"]] == ["tiny", "alias", "x"]
    other = engine(max_loras=1, max_lora_rank=8)
    other.adapters.add_tensors("tiny", tensors(tiny_hybrid(), 8, 2), 8, 2.0)
    with pytest.raises(ValueError):
        build_app(other, "tiny")


CHAT = dict(path="/v1/chat/completions", prompt=None, messages=[{"role": "user", "content": "hi"}])


@pytest.mark.parametrize("path", [{}, CHAT])
def test_samples(served, path):
    e, c = served
    r = post(c, n=3, temperature=1.0, top_k=50, seed=4, **path).json()
    assert [o["index"] for o in r["choices"]] == [0, 1, 2] and r["usage"]["completion_tokens"] == 15
    assert post(c, n=1, **path).status_code == post(c, n=None, **path).status_code == 200
    assert not e.requests and not e.groups


@pytest.mark.parametrize("path", [{}, CHAT])
@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("n", [-1, 129, 10 ** 9, "many", [2], {"a": 1}, 1.5])
def test_refused_numbers_of_samples(served, path, stream, n):
    """The request is at fault (400), and nothing of it reaches the engine."""
    e, c = served
    assert post(c, n=n, stream=stream, **path).status_code == 400
    assert not e.requests and not e.groups


def test_samples_from_a_server_with_speculative_decoding():
    """A server that drafts answers n > 1 as one without does."""
    e = engine(speculative_method="lookup", num_speculative_tokens=3)
    with TestClient(build_app(e, "tiny")) as c:
        one = post(c).json()["choices"][0]
        r = post(c, n=2)
        assert r.status_code == 200, r.text
        assert [(o["index"], o["token_ids"]) for o in r.json()["choices"]] == [(i, one["token_ids"]) for i in range(2)]
        assert post(c, CHAT["path"], prompt=None, messages=CHAT["messages"], n=3).status_code == 200
    assert not e.requests and not e.groups


def stream(c, **body):
    """-> (chunks, choices by index: text and finish reasons)."""
    path = body.pop("path", "/v1/completions")
    with c.stream("POST", path, json={**BODY, "stream": True, **body}) as r:
        assert r.status_code == 200, r.read()
        lines = [s[6:] for s in r.iter_lines() if s.startswith("data: ")]
    assert lines[-1] == "[DONE]"
    chunks = [json.loads(s) for s in lines[:-1]]
    out = {}
    for k in chunks:
        (o,) = k["choices"]
        text, ends, roles = out.setdefault(o["index"], ([], [], []))
        assert not ends                          # nothing after a sample's end
        text.append(o["text"] if "text" in o else o["delta"].get("content", ""))
        roles += [o["delta"]["role"]] if "role" in o.get("delta", {}) else []
        ends += [o["finish_reason"]] if o["finish_reason"] else []
    return chunks, {i: ("".join(t), e, r) for i, (t, e, r) in out.items()}


@pytest.mark.parametrize("path,content,roles", [({}, lambda o: o["text"], []), (CHAT, lambda o: o["message"]["content"], ["assistant"])])
@pytest.mark.parametrize("n", [1, 3])
def test_streamed_samples(served, path, content, roles, n):
    """Every sample arrives under its index, as the whole answer has it."""
    e, c = served
    kw = dict(n=n, temperature=1.0, top_k=50, seed=4, max_tokens=12, **path)
    want = post(c, **kw).json()["choices"]
    _, got = stream(c, **kw)
    assert got == {o["index"]: (content(o), [o["finish_reason"]], roles) for o in want} and len(got) == n
    assert not e.requests and not e.groups


def test_streamed_samples_with_parsers():
    """Reasoning is split sample by sample."""
    e = engine()
    with TestClient(build_app(e, "tiny", reasoning_parser="qwen3")) as c:
        kw = dict(n=2, temperature=1.0, top_k=50, seed=4, max_tokens=12, **CHAT)
        want = post(c, **kw).json()["choices"]
        chunks, got = stream(c, **kw)
        for o in want:
            r = "".join(k["choices"][0]["delta"].get("reasoning_content", "") for k in chunks
                        if k["choices"][0]["index"] == o["index"])
            assert (r, got[o["index"]][0]) == (o["message"]["reasoning_content"], o["message"]["content"])


@pytest.mark.parametrize("path", [{}, CHAT])
def test_streams_name_the_adapter(served, path):
    e, c = served
    assert {k["model"] for k in stream(c, model="x", **path)[0]} == {"x"}
    assert {k["model"] for k in stream(c, **path)[0]} == {"tiny"}
