"""Serving over a 4-bit KV cache on the GPU: against the CPU path, with CUDA
graphs, co-serving with finetuning, and with forked requests."""
import pytest
import torch

from deltaserve_vllm_b200 import ops
from deltaserve_vllm_b200.config import EngineConfig, FinetuneConfig
from deltaserve_vllm_b200.engine.ft.store import FinetuningStore
from deltaserve_vllm_b200.engine.kv_cache import KVCache
from deltaserve_vllm_b200.engine.llm_engine import CoServingEngine
from deltaserve_vllm_b200.engine.model_runner import ModelRunner
from deltaserve_vllm_b200.engine.request import Request, SamplingParams
from deltaserve_vllm_b200.engine.scheduler import Scheduler
from deltaserve_vllm_b200.models.configs import PRESETS
from deltaserve_vllm_b200.models.decoder import DecoderModel
from deltaserve_vllm_b200.models.weights import init_weights

pytestmark = pytest.mark.gpu


def run(name, dev, dt, forced=None, graphs=False):
    arch = PRESETS[name]
    w = init_weights(arch, seed=11, device="cpu", dtype=torch.float32).to(dev, dt)
    kv = KVCache(arch.num_layers, 32, arch.num_kv_heads, 64, 128, dev, dt, kv_group=64)
    sched = Scheduler(kv.allocator, 64, max_num_batched_tokens=160, max_model_len=1024)
    runner = ModelRunner(DecoderModel(w, kv.k, kv.v, None), 64, dev, max_model_len=1024, decode_graphs=graphs)
    g = torch.Generator().manual_seed(0)
    for i, n in enumerate([200, 37, 1, 130]):
        sched.add(Request(str(i), torch.randint(0, arch.vocab, (n,), generator=g).tolist(), SamplingParams(max_tokens=4)))
    logits_all, toks_all = [], []
    for step in range(20):
        out = sched.schedule()
        if out.is_empty():
            break
        toks, logits = runner.execute(out)
        by_rid = {s.req.request_id: toks[s.req.seq_no] for s in out.seqs if s.req.seq_no in toks}
        if forced is not None:
            by_rid = forced[step]
            toks = {s.req.seq_no: by_rid[s.req.request_id] for s in out.seqs if s.req.request_id in by_rid}
        toks_all.append(by_rid)
        logits_all.append(None if logits is None else logits.float().cpu().clone())
        sched.update(out, toks)
    if dev == "cuda":
        assert ops.check_device_error() == 0
    return logits_all, toks_all, runner


@pytest.mark.parametrize("name", ["qwen3-test", "llama3-test"])
def test_gpu_matches_cpu(name):
    """bf16 activations move some codes by a step: the two runs differ by less
    than quantisation itself does (a third of the logits' spread at most)."""
    cpu, toks, _ = run(name, "cpu", torch.float32)
    gpu, _, _ = run(name, "cuda", torch.bfloat16, forced=toks)
    assert len(cpu) == len(gpu)
    for a, b in zip(gpu, cpu):
        if a is not None and a.numel():
            assert float((a - b).norm() / (b - b.mean()).norm()) < 1 / 3


@pytest.mark.parametrize("name", ["qwen3-test", "llama3-test"])
def test_decode_graphs_match_eager(name):
    _, toks, _ = run(name, "cpu", torch.float32)
    eager, _, _ = run(name, "cuda", torch.bfloat16, forced=toks)
    graph, _, runner = run(name, "cuda", torch.bfloat16, forced=toks, graphs=True)
    assert runner.graphs.replays > 0
    for a, b in zip(eager, graph):
        if a is not None and a.numel():
            torch.testing.assert_close(b, a, rtol=2e-2, atol=5e-2)


def test_coserving_over_a_4_bit_cache():
    ecfg = EngineConfig(model="qwen3-test", max_model_len=1024, block_size=64, max_num_batched_tokens=2048, max_loras=2,
                        max_lora_rank=16, num_gpu_blocks_override=256, kv_cache_dtype="int4",
                        enable_prefix_caching=True)
    fcfg = FinetuneConfig(enable_finetuning=True, backward_cuda_graph=True, max_saved_finetuning_tokens=512,
                          learning_rate=1e-3)
    store = FinetuningStore.synthetic(4096, 40, 64, 128, seed=0, max_saved_finetuning_tokens=512, total_epochs=2)
    eng = CoServingEngine(ecfg, fcfg, ft_store=store)
    eng.load_inference_adapter("inf", rank=16, alpha=32)
    g = torch.Generator().manual_seed(0)
    for i in range(12):
        eng.add_request(f"r{i}", torch.randint(0, 4096, (50 + 30 * i,), generator=g).tolist(),
                        SamplingParams(max_tokens=8), adapter="inf" if i % 2 else None)
    eng.run_until_idle(max_steps=5000)
    eng.synchronize()
    assert ops.check_device_error() == 0
    assert eng.coord.completed_cycles >= 4, eng.finetuning_status()
    assert all(l == l and l > 0 for l in eng.trainer.losses)
    assert len([r for r in eng.finished if r.request_id.startswith("r")]) == 12
    assert eng.kv.allocator.num_free == eng.kv.allocator.num_blocks


@pytest.mark.parametrize("dtype", ["int4", "auto"])
def test_fork_and_compact(dtype):
    """A greedy fork repeats its parent, and compaction between steps changes nothing."""
    ecfg = EngineConfig(model="llama3-test", max_model_len=1024, block_size=64, max_num_batched_tokens=2048, max_loras=2,
                        max_lora_rank=16, num_gpu_blocks_override=64, kv_cache_dtype=dtype)
    eng = CoServingEngine(ecfg, FinetuneConfig(enable_finetuning=False))
    g = torch.Generator().manual_seed(2)
    for i, n in enumerate((100, 300, 70)):
        eng.add_request(f"r{i}", torch.randint(0, 4096, (n,), generator=g).tolist(),
                        SamplingParams(max_tokens=20 if i else 2))
    while len(eng.requests["r2"].output_ids) < 4:
        eng.step()
    eng.fork_request("r2", "fork")
    used = eng.compact_kv()
    assert max(p for r in eng.scheduler.running for p in r.block_ids) < used
    eng.run_until_idle(max_steps=500)
    assert ops.check_device_error() == 0
    got = {r.request_id: r.output_ids for r in eng.finished}
    assert got["fork"] == got["r2"] and len(got["r1"]) == 20
    assert eng.kv.allocator.num_free == eng.kv.allocator.num_blocks


def _busy(stream, n=60):
    """Plain work that keeps ``stream`` busy for some 50 ms."""
    with torch.cuda.stream(stream):
        a = torch.ones(8192, 8192, device="cuda", dtype=torch.bfloat16)
        for _ in range(n):
            a @ a


def _serve(dtype, lengths, budget=2048, **tokens):
    ecfg = EngineConfig(model="llama3-test", max_model_len=1024, block_size=64, max_num_batched_tokens=budget, max_loras=2,
                        max_lora_rank=16, num_gpu_blocks_override=64, kv_cache_dtype=dtype)
    eng = CoServingEngine(ecfg, FinetuneConfig(enable_finetuning=False))
    g = torch.Generator().manual_seed(3)
    for i, n in enumerate(lengths):
        eng.add_request(f"r{i}", torch.randint(0, 4096, (n,), generator=g).tolist(),
                        SamplingParams(max_tokens=tokens.get(f"r{i}", 16)))
    return eng


@pytest.mark.parametrize("dtype", ["int4", "auto"])
def test_fork_and_compact_with_a_busy_caller(dtype):
    """The caller's stream is far behind: the next forward still finds the pages copied, and no copy comes after it."""
    eng = _serve(dtype, (100, 300, 90), r0=2)
    while len(eng.requests["r2"].output_ids) < 4:
        eng.step()
    _busy(torch.cuda.current_stream())
    eng.fork_request("r2", "fork")
    eng.step()
    _busy(torch.cuda.current_stream())
    eng.compact_kv()
    eng.run_until_idle(max_steps=500)
    torch.cuda.synchronize()
    assert ops.check_device_error() == 0
    plain = _serve(dtype, (100, 300, 90), r0=2)
    plain.run_until_idle(max_steps=500)
    got = {r.request_id: r.output_ids for r in eng.finished}
    exp = {r.request_id: r.output_ids for r in plain.finished}
    assert got["fork"] == got["r2"] and got["r2"][:4] == exp["r2"][:4]


@pytest.mark.parametrize("dtype", ["int4", "auto"])
def test_compact_behind_a_running_chunk(dtype):
    """A prefill chunk that samples nothing is still running when its pages are moved."""
    def run(compact):
        eng = _serve(dtype, (300, 900), budget=128, r0=2)
        while any(r.request_id == "r0" for r in eng.scheduler.running + list(eng.scheduler.waiting)):
            eng.step()
        r1 = eng.requests["r1"]
        before, at = list(r1.block_ids), r1.num_computed
        _busy(eng.fwd_stream)
        eng.step()
        assert r1.in_prefill and r1.num_computed > at
        if compact:
            eng.compact_kv()
            assert r1.block_ids[:len(before)] != before
        eng.run_until_idle(max_steps=500)
        return r1.output_ids
    assert run(True) == run(False)


@pytest.mark.parametrize("tc", [True, False])
def test_a_mixed_batch_attends_as_on_the_cpu(tc, monkeypatch):
    """Decode, prefill and finetuning rows of one batch over the same codes: the model's attention on both devices.

    bf16 results (2^-8), and as many as the kernels' roundings move an average of values: 2^-7 of the largest."""
    from deltaserve_vllm_b200.models.decoder import ForwardBatch
    monkeypatch.setattr(ops, "ATTN_TC", tc)
    arch = PRESETS["qwen3-test"]
    g = torch.Generator().manual_seed(5)
    hq, hkv, page = arch.num_heads, arch.num_kv_heads, 64
    dec, new, old, ft = [1, 70, 300], [5, 130], [200, 0], [40, 17]
    contexts = dec + [a + b for a, b in zip(new, old)]
    need = [-(-c // page) for c in contexts]
    perm = torch.randperm(sum(need) + 3, generator=g).tolist()
    tables = torch.zeros(5, max(need), dtype=torch.int32)
    cache = torch.zeros(ops.kv4_cache_shape(len(perm), hkv, page, 64), dtype=torch.uint8)
    for i, c in enumerate(contexts):
        mine = [perm.pop() for _ in range(need[i])]
        tables[i, :need[i]] = torch.tensor(mine, dtype=torch.int32)
        slots = torch.tensor([mine[p // page] * page + p % page for p in range(c)])
        ops.kv4_write(torch.randn(c, hkv * 128, generator=g), torch.randn(c, hkv * 128, generator=g), cache, slots)
    lo = len(dec) + sum(new)
    qkv = torch.randn(lo + sum(ft), (hq + 2 * hkv) * 128, generator=g).to(torch.bfloat16)
    starts = torch.tensor([0] + ft).cumsum(0)[:-1].tolist()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)

    def run(dev, dt):
        model = DecoderModel(init_weights(arch, seed=1, device="cpu", dtype=torch.float32).to(dev, dt),
                             [cache.to(dev)], [], None)
        b = ForwardBatch(input_ids=None, positions=None, slot_mapping=None, num_decode=len(dec),
                         dec_block_tables=tables[:3].to(dev), dec_ctx_lens=i32(dec).to(dev), num_prefill_seqs=2,
                         pf_cu_q=i32([0, new[0], sum(new)]).to(dev), pf_ctx_lens=i32(contexts[3:]).to(dev),
                         pf_block_tables=tables[3:].contiguous().to(dev),
                         ft_attn_tiles=ops.dense_attn_tiles(starts, ft, dev, bm=128 if tc else 64), ft_lo=lo, ft_hi=lo + sum(ft))
        out = torch.full((lo + sum(ft), hq * 128), float("nan"), device=dev, dtype=dt)
        model.attention(0, qkv.to(dev, dt), out, b)
        return out.float().cpu()
    a, b = run("cuda", torch.bfloat16), run("cpu", torch.float32)
    assert ops.check_device_error() == 0
    assert bool(((a - b).abs() <= b.abs() * 2 ** -8 + float(qkv.abs().max()) * 2 ** -7).all()), float((a - b).abs().max())
    rel = (a - b).norm(dim=1) / b.norm(dim=1)
    assert bool((rel <= 2 ** -7).all()), rel.max()


def test_finetuning_rows_without_the_tcgen05_kernels(monkeypatch):
    """DSV_ATTN_TC=0: finetuning samples over a 4-bit cache train on the warp-level kernels as well."""
    monkeypatch.setattr(ops, "ATTN_TC", False)
    ecfg = EngineConfig(model="qwen3-test", max_model_len=512, block_size=64, max_num_batched_tokens=512, max_loras=2,
                        max_lora_rank=16, num_gpu_blocks_override=64, kv_cache_dtype="int4")
    fcfg = FinetuneConfig(enable_finetuning=True, max_saved_finetuning_tokens=256, learning_rate=1e-3)
    store = FinetuningStore.synthetic(4096, 8, 64, 100, seed=0, max_saved_finetuning_tokens=256, total_epochs=1)
    eng = CoServingEngine(ecfg, fcfg, ft_store=store)
    eng.add_request("r", list(range(40)), SamplingParams(max_tokens=4))
    eng.run_until_idle(max_steps=2000)
    eng.synchronize()
    assert ops.check_device_error() == 0
    assert eng.coord.completed_cycles >= 1 and all(l == l and l > 0 for l in eng.trainer.losses)
