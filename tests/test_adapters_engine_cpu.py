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


@pytest.mark.parametrize("method", ["lookup", "dflash2"])
def test_samples_with_speculative_decoding(method):
    """generate answers n > 1 under speculative decoding too: greedy samples are the single answer, drawn ones differ."""
    p = list(range(7, 50))
    one = engine().generate([p], SamplingParams(max_tokens=6, **GREEDY))[0].outputs[0].token_ids
    e = engine(speculative_method=method, num_speculative_tokens=3)
    out = e.generate([p, p], [SamplingParams(max_tokens=6, n=3, **GREEDY),
                              SamplingParams(temperature=1.0, top_k=50, seed=1, n=3, max_tokens=6, ignore_eos=True)])
    assert [o.token_ids for o in out[0].outputs] == [one] * 3 and [o.index for o in out[0].outputs] == [0, 1, 2]
    assert len({tuple(o.token_ids) for o in out[1].outputs}) == 3
    assert all(o.finished for o in out) and not e.requests and not e.groups and not e.member
    assert e.kv.blocks.num_free == e.num_blocks - 1


def test_tensor_parallel_ranks_take_the_same_options():
    """What rank 0's server broadcasts reaches the other ranks' engines with every option."""
    from vllm_sly_radiance_b200.parallel.spmd import follower_loop
    got = []

    class Engine:
        def add_request(self, *a, **kw):
            got.append((a, kw))

        def has_unfinished_requests(self):
            return False

    class Broadcaster:
        steps = [[("add", [1, 2], SamplingParams(n=2), "a", dict(share_prompt=False)), ("add", [3], SamplingParams(), "b", {})],
                 [("shutdown",)]]

        def broadcast(self, cmds):
            return self.steps.pop(0)
    follower_loop(Engine(), Broadcaster())
    assert got == [(([1, 2], SamplingParams(n=2), "a"), dict(share_prompt=False)), (([3], SamplingParams(), "b"), {})]
