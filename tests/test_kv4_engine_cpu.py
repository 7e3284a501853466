"""Serving over a 4-bit KV cache on CPU, and page sharing, forking and compaction of any cache."""
import pytest
import torch

from deltaserve_vllm_b200 import ops
from deltaserve_vllm_b200.config import EngineConfig, FinetuneConfig
from deltaserve_vllm_b200.engine.ft.store import FinetuningStore
from deltaserve_vllm_b200.engine.kv_cache import BlockAllocator, KVCache, PrefixCachingAllocator
from deltaserve_vllm_b200.engine.llm_engine import CoServingEngine
from deltaserve_vllm_b200.engine.request import SamplingParams


def engine(tmp=None, **kw):
    ft = kw.pop("ft", False)
    ecfg = EngineConfig(model="qwen3-test", device="cpu", max_model_len=256, block_size=16, max_loras=2,
                        max_lora_rank=8, **dict(dict(max_num_batched_tokens=96, kv_cache_dtype="int4"), **kw))
    if not ft:
        return CoServingEngine(ecfg, FinetuneConfig(enable_finetuning=False))
    fcfg = FinetuneConfig(enable_finetuning=True, max_saved_finetuning_tokens=96, learning_rate=1e-3)
    store = FinetuningStore.synthetic(4096, 8, 16, 40, seed=0, max_saved_finetuning_tokens=96, total_epochs=1)
    return CoServingEngine(ecfg, fcfg, ft_store=store)


def prompts(n):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 4096, (7 + 19 * i,), generator=g).tolist() for i in range(n)]


def generate(eng, n=3, tokens=6, **params):
    for i, p in enumerate(prompts(n)):
        eng.add_request(f"r{i}", p, SamplingParams(max_tokens=tokens, **params))
    eng.run_until_idle(max_steps=500)
    return {r.request_id: r.output_ids for r in eng.finished}


def test_pages_are_several_times_smaller():
    a = KVCache.bytes_per_block(4, 8, 64, 128)
    assert a / KVCache.bytes_per_block(4, 8, 64, 128, kv_group=64) == 256 / 72
    kv = KVCache(4, 3, 8, 64, 128, "cpu", kv_group=64)
    assert kv.nbytes() == 3 * KVCache.bytes_per_block(4, 8, 64, 128, kv_group=64)


def test_chunking_does_not_change_the_tokens():
    """Every step attends to the same codes, however the prompt was cut."""
    whole, cut = generate(engine(max_num_batched_tokens=256)), generate(engine(max_num_batched_tokens=24))
    assert whole == cut and all(len(v) == 6 for v in whole.values())


def test_logits_stay_near_the_unquantised_cache():
    def first_logits(eng):
        seen = []
        fwd = eng.model.forward
        eng.model.forward = lambda *a, **k: seen.append(fwd(*a, **k)) or seen[-1]
        generate(eng, n=1, tokens=1)
        return seen[0]
    a, b = first_logits(engine()), first_logits(engine(kv_cache_dtype="auto"))
    # a code is off by up to half a step of 1 / 15 of its group's range: well inside a third of the logits' spread
    assert float((a - b).norm() / (b - b.mean()).norm()) < 1 / 3


def test_finetuning_rows_attend_to_their_own_keys():
    """Finetuning samples train the same over a 4-bit and over a plain cache."""
    def losses(**kw):
        eng = engine(ft=True, **kw)
        eng.add_request("r", prompts(1)[0], SamplingParams(max_tokens=4))
        eng.run_until_idle(max_steps=500)
        assert eng.kv.allocator.num_free == eng.kv.allocator.num_blocks
        return eng.trainer.losses
    a, b = losses(), losses(kv_cache_dtype="auto")
    assert len(a) >= 2
    torch.testing.assert_close(torch.tensor(a), torch.tensor(b), rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype", ["int4", "auto"])
@pytest.mark.parametrize("caching", [False, True])
def test_fork_and_compact_keep_the_tokens(dtype, caching):
    plain = generate(engine(kv_cache_dtype=dtype), n=3, tokens=12)
    eng = engine(kv_cache_dtype=dtype, enable_prefix_caching=caching)
    for i, p in enumerate(prompts(3)):
        eng.add_request(f"r{i}", p, SamplingParams(max_tokens=12 if i else 2))
    while len(eng.requests["r2"].output_ids) < 3:
        eng.step()
    child = eng.fork_request("r2", "fork")
    full = eng.requests["r2"].num_computed // 16
    assert child.block_ids[:full] == eng.requests["r2"].block_ids[:full]
    assert child.block_ids[full:] != eng.requests["r2"].block_ids[full:full + 1]
    used = eng.compact_kv()                       # r0 has left holes behind
    assert max(p for r in eng.scheduler.running for p in r.block_ids) < used
    assert used == eng.kv.num_blocks - len(eng.kv.allocator._free)
    eng.run_until_idle(max_steps=500)
    got = {r.request_id: r.output_ids for r in eng.finished}
    assert got["fork"] == got["r2"] == plain["r2"] and got["r1"] == plain["r1"]
    assert eng.kv.allocator.num_free == eng.kv.allocator.num_blocks


def test_fork_refusals():
    eng = engine()
    eng.add_request("a", prompts(1)[0], SamplingParams(max_tokens=3))
    with pytest.raises(KeyError):
        eng.fork_request("a", "b")                # not decoding yet
    eng.step()
    with pytest.raises(ValueError):
        eng.fork_request("a", "a")
    with pytest.raises(KeyError):
        eng.fork_request("zz", "b")
    taken = eng.kv.allocator.allocate(eng.kv.allocator.num_free)
    before = list(eng.requests["a"].block_ids)
    with pytest.raises(MemoryError):
        eng.fork_request("a", "b")
    assert eng.requests["a"].block_ids == before and "b" not in eng.requests
    eng.kv.allocator.free(taken)
    eng.run_until_idle(max_steps=50)
    assert eng.kv.allocator.num_free == eng.kv.allocator.num_blocks


@pytest.mark.parametrize("kind", [BlockAllocator, PrefixCachingAllocator])
def test_shared_pages_return_with_their_last_holder(kind):
    a = kind(6)
    p = a.allocate(3)
    a.share(p[:2])
    a.share(p[:1])
    a.free(p)
    assert a.num_free == 4
    a.free(p[:2])
    assert a.num_free == 5
    a.free(p[:1])
    assert a.num_free == 6 and sorted(a.allocate(6)) == list(range(6))


@pytest.mark.parametrize("kind", [BlockAllocator, PrefixCachingAllocator])
def test_compaction_moves_the_fewest_pages(kind):
    a = kind(10)
    p = a.allocate(8)
    a.share([p[7]])
    a.free([p[1], p[3], p[4]])
    moves = a.compact()
    live = {p[i] for i in (0, 2, 5, 6, 7)}
    to = dict(moves)
    assert {to.get(x, x) for x in live} == set(range(5)) and len(moves) == len([x for x in live if x >= 5])
    assert not set(to) & set(to.values())
    assert a.num_free == 5 and sorted(a.allocate(5)) == list(range(5, 10))
    a.free([to.get(p[7], p[7])])
    assert a.num_free == 0
    a.free([to.get(p[7], p[7])])
    assert a.num_free == 1
    assert kind(4).compact() == []


def test_compaction_keeps_cached_prefixes():
    a = PrefixCachingAllocator(6)
    p = a.allocate(5)
    for i, x in enumerate(p):
        a.register(x, bytes([i]))
    a.free(p[:2] + p[3:])
    a._evict(p[0])
    a._free.append(p[0])
    to = dict(a.compact())
    assert a.lookup([bytes([4])]) == [to.get(p[4], p[4])] and a.lookup([bytes([2])]) == [to.get(p[2], p[2])]
    assert set(a.hash_of) == set(range(4))


def test_configuration_refusals():
    for bad in (dict(kv_cache_dtype="int3"), dict(kv_cache_group=48)):
        with pytest.raises(ValueError):
            EngineConfig(**bad)
    with pytest.raises(ValueError):               # head_dim 64
        CoServingEngine(EngineConfig(model="qwen3-tiny", device="cpu", kv_cache_dtype="int4", block_size=16),
                        FinetuneConfig(enable_finetuning=False))
    with pytest.raises(ValueError):
        KVCache(1, 2, 1, 16, 64, "cpu", kv_group=64)
    with pytest.raises(ValueError):
        ops.kv4_cache_shape(1, 1, 8, 64)


def test_comparison_command_runs():
    from deltaserve_vllm_b200.eval.kv4_compare import main
    res = main(["--model", "llama3-test", "--batch", "2", "--prompt", "40", "--tokens", "8", "--device", "cpu",
                "--blocks", "16"])
    assert res["int4"]["page_bytes"] * 2 * 256 == res["auto"]["page_bytes"] * 72      # fp32 pages on CPU
    assert res["int4"]["fork"]["same_tokens"]


def test_fork_and_compact_copy_on_the_forward_stream(monkeypatch):
    """The pages that move are the forward's: their copies belong to the stream it runs on, whatever the caller's is."""
    eng = engine()
    for i, p in enumerate(prompts(3)):
        eng.add_request(f"r{i}", p, SamplingParams(max_tokens=8))
    while len(eng.requests["r2"].output_ids) < 3:
        eng.step()
    current, copied = ["caller's"], []

    class On:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            current.append(self.stream)

        def __exit__(self, *exc):
            current.pop()
    copy = ops.copy_pages
    monkeypatch.setattr(torch.cuda, "stream", On)
    monkeypatch.setattr(ops, "copy_pages", lambda *a: (copied.append((current[-1], len(a[1]))), copy(*a)))
    monkeypatch.setattr(eng, "fwd_stream", "forward")
    eng.fork_request("r2", "fork")
    eng.scheduler.abort("r1")                     # leaves holes for the compaction
    eng.compact_kv()
    assert [s for s, _ in copied] == ["forward"] * 2 and all(n for _, n in copied)


def test_a_forks_timeline_is_its_tokens():
    """A fork carries its parent's tokens and their times: no time runs backwards, no gap spans several tokens."""
    eng = engine()
    for i, p in enumerate(prompts(2)):
        eng.add_request(f"r{i}", p, SamplingParams(max_tokens=8))
    while len(eng.requests["r1"].output_ids) < 5:
        eng.step()
    r = eng.requests["r1"]
    child = eng.fork_request("r1", "fork")
    assert child.ttft() == r.ttft() > 0
    assert child.num_cached_tokens == child.num_prompt
    eng.run_until_idle(max_steps=50)
    for x in (r, child):
        assert len(x.tbts()) == len(x.output_ids) - 1 == 7
        assert all(t >= 0 for t in x.tbts())
    assert child.tbts()[:4] == r.tbts()[:4] and child.token_times is not r.token_times
    assert child.finish_time - child.arrival_time >= child.ttft() + sum(child.tbts())


def test_a_fork_has_tokens_left_to_produce():
    """A fork's parameters allow at least one more token, within the model's length; a refused fork changes nothing."""
    eng = engine()
    eng.add_request("a", prompts(2)[1], SamplingParams(max_tokens=8))
    while len(eng.requests["a"].output_ids) < 4:
        eng.step()
    free, block_ids = eng.kv.allocator.num_free, list(eng.requests["a"].block_ids)
    for n in (0, 2, 4, 256 - 26 + 1):
        with pytest.raises(ValueError):
            eng.fork_request("a", "b", SamplingParams(max_tokens=n))
    assert eng.kv.allocator.num_free == free and eng.requests["a"].block_ids == block_ids and "b" not in eng.requests
    child = eng.fork_request("a", "b", SamplingParams(max_tokens=5))
    longest = eng.fork_request("a", "c", SamplingParams(max_tokens=256 - 26))
    eng.run_until_idle(max_steps=500)
    assert len(child.output_ids) == 5 and len(longest.output_ids) == 256 - 26
    assert eng.kv.allocator.num_free == eng.kv.allocator.num_blocks


@pytest.mark.parametrize("parent,child,ok", [({}, dict(logprobs=True), False),
                                             (dict(logprobs=True), dict(logprobs=True, top_logprobs=2), False),
                                             (dict(logprobs=True, top_logprobs=2), dict(logprobs=True, top_logprobs=1), True),
                                             (dict(logprobs=True), {}, True)])
def test_a_forks_logprobs_are_its_tokens(parent, child, ok):
    """Log-probabilities are read by the token's position: a fork can only go on with those that its parent recorded."""
    eng = engine()
    eng.add_request("a", prompts(1)[0], SamplingParams(max_tokens=6, **parent))
    while len(eng.requests["a"].output_ids) < 3:
        eng.step()
    if not ok:
        with pytest.raises(ValueError):
            eng.fork_request("a", "b", SamplingParams(max_tokens=6, **child))
        return
    r = eng.fork_request("a", "b", SamplingParams(max_tokens=6, **child))
    eng.run_until_idle(max_steps=50)
    if r.params.logprobs:
        assert len(r.output_logprobs) == 6 and (not r.params.top_logprobs or len(r.output_top_logprobs) == 6)
