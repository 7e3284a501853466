"""The 4-bit KV cache on CPU tensors: the format, attention over it, page copies, refusals."""
import pytest
import torch

from deltaserve_vllm_b200 import ops
from deltaserve_vllm_b200.ops import reference as ref


def rows(seed, *shape):
    return torch.randn(*shape, 128, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def test_every_code_has_its_own_nibble():
    byte, shift = ref.kv4_places("cpu")
    for w in (0, 1):
        nibbles = (2 * byte[w] + shift[w] // 4).flatten()
        assert sorted(nibbles.tolist()) == list(range(2048))
        # a byte belongs to one token: single tokens are written without a read
        tok = torch.arange(16)[:, None].expand(16, 128).flatten()
        owner = torch.full((1024,), -1)
        owner[byte[w].flatten()] = tok
        assert torch.equal(owner[byte[w].flatten()], tok)


@pytest.mark.parametrize("group", ops.KV4_GROUPS)
def test_written_rows_read_back_within_half_a_step(group):
    n, hkv, page = 40, 2, 16
    k, v = rows(1, n, hkv), rows(2, n, hkv)
    cache = torch.zeros(ops.kv4_cache_shape(4, hkv, page, group), dtype=torch.uint8)
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(3))[:n]
    slots[5] = -1
    ops.kv4_write(k.flatten(1), v, cache, slots)
    for x, y in zip((k, v), ops.kv4_read(cache, slots)):
        y = y.view(n, hkv, 128).double()
        assert bool((y[5] == 0).all())
        x, y = x.double()[slots >= 0], y[slots >= 0]
        xs = x.unflatten(-1, (-1, group))
        step = (xs.amax(-1).clamp(min=0) - xs.amin(-1).clamp(max=0)) / 15
        # half a step; the bf16 scale is up to 2^-9 short of 15 steps (0.03) and the fp16 zero point moves both
        # ends by up to 2^-8 of a step; the value is then rounded to bf16
        bound = (0.5 + 0.03 + 0.01) * step.repeat_interleave(group, -1) + x.abs() * 2 ** -8
        assert bool(((x - y).abs() <= bound + step.repeat_interleave(group, -1) * 2 ** -7).all())


def test_limits_of_the_format():
    """Zeros, values past the range, infinities, NaN and vanishing groups."""
    x = torch.zeros(6, 128)
    x[1] = 1e9
    x[2, :64], x[2, 64:] = float("inf"), float("-inf")
    x[3, 3] = float("nan")
    x[4] = 2.0 ** -125
    x[5] = -7.0
    cache = torch.zeros(ops.kv4_cache_shape(1, 1, 16, 64), dtype=torch.uint8)
    ops.kv4_write(x.to(torch.bfloat16), x.to(torch.bfloat16), cache, torch.arange(6))
    for y in ops.kv4_read(cache, torch.arange(6)):
        y = y.float()
        assert bool((y[[0, 3, 4]] == 0).all())
        # 15 steps of a bf16 scale: within 2^-8 of the end of the range
        torch.testing.assert_close(y[1], torch.full((128,), 8192.0), rtol=2 ** -7, atol=0)
        torch.testing.assert_close(y[2], torch.tensor([8192.0, -8192.0]).repeat_interleave(64), rtol=2 ** -7, atol=0)
        torch.testing.assert_close(y[5], torch.full((128,), -7.0), rtol=2 ** -7, atol=0)


@pytest.mark.parametrize("heads,hkv", [(4, 4), (6, 2), (8, 1)])
def test_attention_equals_the_bf16_cache_paths_on_the_same_values(heads, hkv):
    """Attention over the codes is attention over the values they stand for."""
    page, group, contexts, new = 16, 64, [37, 1, 0, 64], [5, 1, 0, 64]
    need = [-(-c // page) for c in contexts]
    cache = torch.zeros(ops.kv4_cache_shape(sum(need) + 1, hkv, page, group), dtype=torch.uint8)
    tables = torch.zeros(4, max(need), dtype=torch.int32)
    perm = torch.randperm(sum(need) + 1, generator=torch.Generator().manual_seed(1)).tolist()
    for i, c in enumerate(contexts):
        mine = [perm.pop() for _ in range(need[i])]
        tables[i, :need[i]] = torch.tensor(mine, dtype=torch.int32)
        slots = torch.tensor([mine[p // page] * page + p % page for p in range(c)], dtype=torch.int64)
        ops.kv4_write(rows(i, c, hkv), rows(9 + i, c, hkv), cache, slots)
    values = ref.kv4_values(cache)
    k, v = (values[:, :, :, w].flatten(2, 3).contiguous() for w in (0, 1))
    ctx = torch.tensor(contexts, dtype=torch.int32)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    q = rows(5, sum(new), heads).flatten(1).float()
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    ops.paged_prefill4(q, cache, tables, cu, ctx, a, heads, 0.1, None)
    ref.paged_prefill(q, k, v, tables, cu, ctx, b, heads, 0.1)
    torch.testing.assert_close(a, b)
    live = [0, 1, 3]
    q = rows(6, 4, heads).flatten(1).float()
    a, b = torch.full_like(q, 9.0), torch.zeros_like(q)
    ops.paged_decode4(q, cache, tables, ctx, a, heads, 0.1, ops.kv4_workspace("cpu"))
    ref.paged_decode(q[live], k, v, tables[live], ctx[live], b[live], heads, 0.1)
    c = torch.zeros(3, heads * 128)
    ref.paged_decode(q[live], k, v, tables[live], ctx[live], c, heads, 0.1)
    torch.testing.assert_close(a[live], c)
    assert bool((a[2] == 0).all())


def test_copy_pages_and_refusals():
    caches = [torch.randn(6, 2, 3) for _ in range(2)]
    before = [c.clone() for c in caches]
    ops.copy_pages(caches, [0, 0, 5], [1, 2, 3])
    for c, b in zip(caches, before):
        assert torch.equal(c[[1, 2, 3]], b[[0, 0, 5]]) and torch.equal(c[[0, 4, 5]], b[[0, 4, 5]])
    for src, dst in (([0], [1, 2]), ([0], [6]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(ValueError):
            ops.copy_pages(caches, src, dst)


def test_refusals():
    cache = torch.zeros(ops.kv4_cache_shape(2, 1, 16, 64), dtype=torch.uint8)
    x, slots = rows(1, 3, 1), torch.arange(3)
    for bad in (dict(cache=cache[..., :1000]), dict(cache=cache.to(torch.int16)), dict(slots=slots[:2]),
                dict(slots=slots.float()), dict(k=x[:, :, :64])):
        a = dict(dict(cache=cache, k=x, slots=slots), **bad)
        with pytest.raises(ValueError):
            ops.kv4_write(a["k"], x, a["cache"], a["slots"])
    for bad in (lambda: ops.kv4_record_bytes(16), lambda: ops.kv4_cache_shape(1, 1, 24, 64),
                lambda: ops.kv4_read(cache, slots.int()),
                lambda: ops.paged_decode4(rows(1, 1, 3).flatten(1), cache.view(2, 1, 1, 2, -1).expand(2, 2, 1, 2, 1152),
                                          torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                                          torch.zeros(1, 384), 3, 1.0, None)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("shape", [(0, 1, 1), (2, 0, 1), (2, 1, 0)])
def test_an_empty_cache_is_refused(shape):
    cache = torch.zeros(*shape, 2, 1152, dtype=torch.uint8)
    q, one, cu = torch.zeros(1, 128), torch.ones(1, dtype=torch.int32), torch.arange(2, dtype=torch.int32)
    tables, slots = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    k = torch.zeros(1, shape[1] * 128, dtype=torch.bfloat16)
    for call in (lambda: ops.kv4_write(k, k, cache, slots), lambda: ops.kv4_read(cache, slots),
                 lambda: ops.paged_decode4(q, cache, tables, one, q.clone(), 1, 1.0, None),
                 lambda: ops.paged_prefill4(q, cache, tables, cu, one, q.clone(), 1, 1.0, None)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("heads", [0, 17, 32])
def test_query_heads_are_1_to_16_times_the_kv_heads(heads):
    cache = torch.zeros(ops.kv4_cache_shape(1, 1, 16, 64), dtype=torch.uint8)
    q, one, cu = torch.zeros(1, heads * 128), torch.ones(1, dtype=torch.int32), torch.arange(2, dtype=torch.int32)
    tables = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_decode4(q, cache, tables, one, q.clone(), heads, 1.0, None)
    with pytest.raises(ValueError):
        ops.paged_prefill4(q, cache, tables, cu, one, q.clone(), heads, 1.0, None)


def test_copy_pages_refuses_caches_that_differ():
    """As on the GPU: nothing is copied when the caches have not one shape."""
    caches = [torch.zeros(6, 2, 3), torch.ones(4, 2, 3)]
    before = [c.clone() for c in caches]
    with pytest.raises(ValueError):
        ops.copy_pages(caches, [0], [5])
    assert all(torch.equal(a, b) for a, b in zip(caches, before))
