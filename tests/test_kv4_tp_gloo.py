"""A 4-bit KV cache under tensor parallelism, on CPU ranks (gloo): each rank
quantises its own heads, finetuning samples attend to their own rows on every
rank, and both ranks together produce what one produces."""
import os
import socket
import tempfile
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _serve(comm=None, world=1):
    from deltaserve_vllm_b200.config import EngineConfig, FinetuneConfig
    from deltaserve_vllm_b200.engine.ft.store import FinetuningStore
    from deltaserve_vllm_b200.engine.llm_engine import CoServingEngine
    from deltaserve_vllm_b200.engine.request import SamplingParams
    ecfg = EngineConfig(model="qwen3-test", device="cpu", tensor_parallel_size=world, max_model_len=256, block_size=16,
                        max_num_batched_tokens=96, max_loras=2, max_lora_rank=8, kv_cache_dtype="int4")
    fcfg = FinetuneConfig(enable_finetuning=True, max_saved_finetuning_tokens=96, learning_rate=1e-3)
    store = FinetuningStore.synthetic(4096, 8, 16, 40, seed=0, max_saved_finetuning_tokens=96, total_epochs=1)
    eng = CoServingEngine(ecfg, fcfg, comm=comm, ft_store=store)
    if comm is not None and comm.rank != 0:
        eng.follow()
        return None
    g = torch.Generator().manual_seed(0)
    reqs = [eng.add_request(f"r{i}", torch.randint(0, 4096, (20 + 30 * i,), generator=g).tolist(),
                            SamplingParams(max_tokens=6)) for i in range(4)]
    eng.run_until_idle(max_steps=1000)
    out = {"tokens": [r.output_ids for r in reqs], "losses": eng.trainer.losses, "shape": tuple(eng.kv.k[0].shape[1:])}
    with pytest.raises(ValueError) if world > 1 else pytest.raises(KeyError):
        eng.fork_request("r0", "fork")
    if comm is not None:
        eng.shutdown()
    return out


def _worker(rank, world, port, outdir):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world,
                            timeout=timedelta(seconds=60))
    from deltaserve_vllm_b200.parallel.comm import TPComm
    try:
        out = _serve(TPComm(), world)
        if rank == 0:
            torch.save(out, os.path.join(outdir, "res.pt"))
    finally:
        dist.destroy_process_group()


def test_two_ranks_serve_and_train_as_one():
    """The ranks' sums differ from one rank's in fp32 rounding; a code may move by a step where a value lies between two,
    which the first tokens of random weights' logits and the losses' first digits withstand."""
    with tempfile.TemporaryDirectory() as d:
        mp.start_processes(_worker, args=(2, _port(), d), nprocs=2, join=True, start_method="spawn")
        two = torch.load(os.path.join(d, "res.pt"))
    one = _serve()
    assert one["shape"][0] == 2 and two["shape"] == (1, *one["shape"][1:])
    assert two["tokens"] == one["tokens"]
    n = min(len(one["losses"]), len(two["losses"]))
    assert n >= 2
    torch.testing.assert_close(torch.tensor(two["losses"][:n]), torch.tensor(one["losses"][:n]), rtol=1e-2, atol=1e-2)
