"""Serving with the KV cache in bf16 and in 4 bits, side by side.

    python -m deltaserve_vllm_b200.eval.kv4_compare --model llama3-8b --batch 64 --prompt 1024 --tokens 64

The same prompts are generated greedily by an engine with each cache: page
bytes, pages that fit, prefill and decode times, and how long the generated
tokens agree. The 4-bit engine also forks a request half way (its last page is
copied, the others shared) and compacts its pool. Weights are random unless
``--model`` is a directory: token agreement then says little about a trained
model's.
"""

from __future__ import annotations

import argparse
import json
import time


def run(model: str, batch: int, prompt: int, tokens: int, dtype: str, group: int, device: str | None = None,
        blocks: int | None = None, seed: int = 0) -> dict:
    import torch

    from ..config import EngineConfig, FinetuneConfig
    from ..engine.llm_engine import CoServingEngine
    from ..engine.request import SamplingParams

    ecfg = EngineConfig(model=model, device=device, max_model_len=prompt + tokens + 64, block_size=64,
                        max_num_seqs=max(batch + 1, 8), max_num_batched_tokens=8192, max_loras=1, max_lora_rank=8,
                        seed=seed, kv_cache_dtype=dtype, kv_cache_group=group, num_gpu_blocks_override=blocks)
    eng = CoServingEngine(ecfg, FinetuneConfig(enable_finetuning=False))
    g = torch.Generator().manual_seed(seed)
    for i in range(batch):                       # first use of every kernel and CUDA graph
        eng.add_request(f"w{i}", [1] * 8, SamplingParams(max_tokens=3))
    eng.run_until_idle(max_steps=1000)
    reqs = [eng.add_request(f"r{i}", torch.randint(0, eng.arch.vocab, (prompt,), generator=g).tolist(),
                            SamplingParams(max_tokens=tokens)) for i in range(batch)]

    def until(done) -> float:
        t0 = time.perf_counter()
        while eng.has_unfinished() and not done():
            eng.step()
        if eng.cuda:
            torch.cuda.synchronize(eng.device)
        return time.perf_counter() - t0

    prefill_s = until(lambda: all(r.output_ids for r in reqs))
    start = sum(len(r.output_ids) for r in reqs)
    decode_s = until(lambda: len(reqs[0].output_ids) >= tokens // 2)
    made = sum(len(r.output_ids) for r in reqs) - start
    forked = None
    if dtype == "int4" and reqs[0] in eng.scheduler.running:
        child = eng.fork_request("r0", "fork")
        in_use = eng.compact_kv()
        forked = {"shared_pages": len(child.block_ids) - 1, "pages_in_use": in_use}
    until(lambda: False)
    if forked is not None:
        forked["same_tokens"] = child.output_ids == reqs[0].output_ids
    return {"kv_cache_dtype": dtype, "page_bytes": eng.kv.nbytes() // eng.kv.num_blocks, "pages": eng.kv.num_blocks,
            "prefill_s": round(prefill_s, 4), "decode_tokens_per_s": round(made / max(decode_s, 1e-9), 1),
            "fork": forked, "tokens": [r.output_ids for r in reqs]}


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--model", default="llama3-8b-2l")
    p.add_argument("--batch", type=int, default=16)
    p.add_argument("--prompt", type=int, default=512)
    p.add_argument("--tokens", type=int, default=32)
    p.add_argument("--group", type=int, default=64, help="channels per scale: 32, 64 or 128")
    p.add_argument("--device", default=None)
    p.add_argument("--blocks", type=int, default=None, help="KV pages (default: what fits)")
    a = p.parse_args(argv)
    res = {}
    for dtype in ("auto", "int4"):
        r = run(a.model, a.batch, a.prompt, a.tokens, dtype, a.group, a.device, a.blocks)
        res[dtype] = r
    same = [next((i for i, (x, y) in enumerate(zip(u, v)) if x != y), len(u))
            for u, v in zip(res["auto"].pop("tokens"), res["int4"].pop("tokens"))]
    res["tokens_before_the_first_difference"] = sum(same) / max(1, len(same))
    print(json.dumps(res, indent=1))
    return res


if __name__ == "__main__":
    main()
