"""The 4-bit KV cache's kernels: write / read bit for bit, decode attention
against 64-bit arithmetic on the values the codes stand for, page copies."""
import pytest
import torch

from deltaserve_vllm_b200 import ops
from deltaserve_vllm_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert ops.check_device_error() == 0


@pytest.fixture(scope="module")
def ws():
    return ops.kv4_workspace(DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(g, *shape, wide=6.0):
    x = torch.randn(*shape, 128, generator=g, device=DEV)
    return (x * torch.where(torch.rand(128, generator=g, device=DEV) < 0.05, wide, 1.0)).to(torch.bfloat16)


def empty_cache(pages, hkv, page, group):
    """A cache of 0xff bytes: an unwritten scale or zero point is a NaN."""
    return torch.full(ops.kv4_cache_shape(pages, hkv, page, group), 255, dtype=torch.uint8, device=DEV)


def special_rows(g, n, hkv):
    """Rows with everything a group can hold: zeros, one sign, one value, tiny, huge, infinities, NaN."""
    x = rows(g, n, hkv)
    x[0::8] = 0
    x[1::8] = x[1::8].abs() + 3
    x[2::8] = -2.5
    x[3::8] *= 2.0 ** -130
    x[4::8] *= 3e4
    x[5::8, :, ::17] = float("inf")
    x[6::8, :, 1::29] = float("nan")
    x[7::8, :, 5] = float("-inf")
    return x


@pytest.mark.parametrize("group", ops.KV4_GROUPS)
@pytest.mark.parametrize("n,hkv,page", [(1, 1, 16), (16, 2, 16), (37, 3, 48), (300, 8, 64), (129, 1, 128)])
@pytest.mark.parametrize("start", [0, 5])
def test_write_and_read_match_the_format(n, hkv, page, group, start):
    g = gen(n + page + group)
    k, v = special_rows(g, n, hkv), special_rows(g, n, hkv)
    pages = -(-(start + n) // page) + 2
    perm = torch.randperm(pages, generator=g, device=DEV)
    pos = start + torch.arange(n, device=DEV)
    slots = perm[pos // page] * page + pos % page
    if n > 20:
        slots[3::7] = -1
    got = empty_cache(pages, hkv, page, group)
    exp = got.clone().cpu()
    ops.kv4_write(k.flatten(1), v.flatten(1), got, slots)
    ref.kv4_write(k.flatten(1).cpu(), v.flatten(1).cpu(), exp, slots.cpu())
    assert torch.equal(got.cpu(), exp)
    gk, gv = ops.kv4_read(got, slots)
    ek, ev = ref.kv4_read(exp, slots.cpu())
    assert torch.equal(gk.cpu(), ek) and torch.equal(gv.cpu(), ev)


@pytest.mark.parametrize("group", ops.KV4_GROUPS)
@pytest.mark.parametrize("start", [0, 3, 15])
@pytest.mark.parametrize("kind", ["sequences", "holes", "shuffled", "repeats_a_page"])
def test_many_rows_fill_whole_records_or_not(kind, start, group):
    """Enough rows that 16 of them go together where they fill a record: sequences that begin anywhere,
    -1 slots inside, unordered slots, records that are full in the cache but not by rows that follow one another."""
    g = gen(4 + start)
    n, hkv, page = 4200, 8, 48
    k, v = rows(g, n, hkv).flatten(1), rows(g, n, hkv).flatten(1)
    slots = torch.cat([torch.arange(m, device=DEV) + 48 * 13 * i + (start if i % 2 else 0) for i, m in
                       enumerate([600, 37, 16, 15, 3532])])
    pages = 128
    if kind == "holes":
        slots[5::61] = -1
    elif kind == "shuffled":
        slots = slots[torch.randperm(n, generator=g, device=DEV)]
    elif kind == "repeats_a_page":
        slots = slots.view(-1, 2).flip(1).flatten().clone()
    got = empty_cache(pages, hkv, page, group)
    ops.kv4_write(k, v, got, slots)
    exp = empty_cache(pages, hkv, page, group)
    for i in range(0, n, 100):               # few rows at a time: one by one
        ops.kv4_write(k[i:i + 100], v[i:i + 100], exp, slots[i:i + 100])
    assert torch.equal(got, exp)
    assert torch.equal(ops.kv4_read(got, slots)[0], torch.cat([ops.kv4_read(got, s)[0] for s in slots.split(100)]))


@pytest.mark.parametrize("order", ["shuffled", "reversed", "two_runs"])
def test_write_takes_slots_in_any_order(order):
    """Slots that do not follow one another, or do so only for a part of a 16-token record."""
    g = gen(3)
    n, hkv, page, group = 96, 2, 64, 64
    k, v = rows(g, n, hkv), rows(g, n, hkv)
    slots = {"shuffled": torch.randperm(256, generator=g, device=DEV)[:n],
             "reversed": torch.arange(n - 1, -1, -1, device=DEV) + 64,
             "two_runs": torch.cat([torch.arange(8, device=DEV) + 64, torch.arange(n - 8, device=DEV) + 136])}[order]
    got = empty_cache(4, hkv, page, group)
    exp = got.clone().cpu()
    ops.kv4_write(k.flatten(1), v.flatten(1), got, slots)
    ref.kv4_write(k.flatten(1).cpu(), v.flatten(1).cpu(), exp, slots.cpu())
    assert torch.equal(got.cpu(), exp)


@pytest.mark.parametrize("layout", ["qkv", "heads", "odd"])
def test_write_takes_strided_rows(layout):
    g = gen(5)
    n, hkv, page, group = 50, 2, 16, 32
    slots = torch.arange(n, device=DEV)
    base = rows(g, n, 9).flatten(1)
    if layout == "qkv":           # column blocks of a fused projection
        k, v = base[:, 128:384], base[:, 640:896]
    elif layout == "heads":       # [rows, heads, 128] with its own head stride
        k, v = base.view(n, 9, 128)[:, 1:8:4], base.view(n, 9, 128)[:, 2:9:4]
    else:                         # rows that start at an odd element
        k, v = base[:, 1:257], base[:, 259:515]
    got = empty_cache(4, hkv, page, group)
    exp = got.clone().cpu()
    ops.kv4_write(k, v, got, slots)
    ref.kv4_write(k.cpu(), v.cpu(), exp, slots.cpu())
    assert torch.equal(got.cpu(), exp)


def test_write_outside_the_cache_is_an_error_not_a_write():
    g = gen(6)
    k = rows(g, 2, 1)
    cache = empty_cache(2, 1, 16, 64)
    before = cache.clone()
    ops.kv4_write(k.flatten(1), k.flatten(1), cache, torch.tensor([32, 1 << 40], device=DEV))
    assert torch.equal(cache, before)
    assert ops.check_device_error() != 0


def filled(g, contexts, hkv, page, group, extra_cols=2):
    """A cache of quantised rows for every context, its block tables (unused
    entries out of range) and the values: float64 [n][2][hkv, ctx, 128]."""
    need = [-(-c // page) for c in contexts]
    pages = sum(need) + 1
    perm = torch.randperm(pages, generator=g, device=DEV).tolist()
    tables = torch.full((len(contexts), max(need) + extra_cols), 1 << 30, dtype=torch.int32)
    cache = empty_cache(pages, hkv, page, group)
    values = []
    for i, c in enumerate(contexts):
        mine = [perm.pop() for _ in range(need[i])]
        tables[i, :need[i]] = torch.tensor(mine, dtype=torch.int32)
        slots = torch.tensor([mine[p // page] * page + p % page for p in range(c)], dtype=torch.int64, device=DEV)
        if c:
            ops.kv4_write(rows(g, c, hkv).flatten(1), (rows(g, c, hkv) * 0.5).flatten(1), cache, slots)
        rec = ref.kv4_values(cache[torch.tensor(mine, device=DEV, dtype=torch.long)]).double()
        values.append([rec[:, :, :, w].permute(1, 0, 2, 3, 4).reshape(hkv, -1, 128)[:, :c] for w in (0, 1)])
    return cache, tables.to(DEV), values


def attention64(q, k, v, seen):
    """float64 softmax attention: q [m, heads, 128], k / v [hkv, ctx, 128], seen [m, ctx]."""
    q = q.double().unflatten(1, (k.shape[0], -1))
    s = torch.einsum("mhgd,hkd->mhgk", q, k) * SCALE
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    return torch.einsum("mhgk,hkd->mhgd", torch.softmax(s, -1), v).flatten(1)


def check(got, exp, v):
    """bf16 rounding of the result (2^-9, taken twice for values next to a
    rounding step) and, absolute: weights in 11 bits against codes of up to twice
    the largest value (2^-10), and scores summed in fp32 (below 2^-11 of a weight
    for these inputs, moving an average of values by at most twice that)."""
    assert got.shape == exp.shape
    top = float(v.abs().max()) if v.numel() else 0.0
    err = (got.double() - exp).abs()
    assert bool((err <= exp.abs() * 2 ** -8 + top * 2 ** -9).all()), float((err - exp.abs() * 2 ** -8).max() / top)


def check_decode(contexts, heads, hkv, page, group, ws, seed=0, q=None):
    g = gen(seed + page + group + heads)
    cache, tables, values = filled(g, contexts, hkv, page, group)
    ctx = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    if q is None:
        q = torch.randn(len(contexts), (heads + 2) * 128, generator=g, device=DEV).to(torch.bfloat16)[:, 128:-128]
    out = torch.full((len(contexts), heads * 128 + 8), float("nan"), dtype=torch.bfloat16, device=DEV)[:, :heads * 128]
    ops.paged_decode4(q, cache, tables, ctx, out, heads, SCALE, ws)
    again = torch.empty_like(out)
    ops.paged_decode4(q, cache, tables, ctx, again, heads, SCALE, ws)
    assert torch.equal(out, again)
    for i, c in enumerate(contexts):
        if c == 0:
            assert bool((out[i] == 0).all())
            continue
        exp = attention64(q[i].view(1, heads, 128), *values[i], torch.ones(1, c, dtype=torch.bool, device=DEV))
        check(out[i:i + 1], exp, values[i][1])
    return out


@pytest.mark.parametrize("group", ops.KV4_GROUPS)
@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_decode_ragged(page, group, ws):
    check_decode([0, 1, 15, 16, 17, 63, 64, 65, 127, 300, 0, 1000], 8, 2, page, group, ws)


@pytest.mark.parametrize("per", list(range(1, 17)))
def test_decode_query_heads_per_kv_head(per, ws):
    check_decode([77, 1, 512, 33], 2 * per, 2, 64, 64 if per % 2 else 32, ws)


@pytest.mark.parametrize("batch,ctx", [(1, 1), (1, 5000), (3, 2049), (130, 65), (700, 20)])
def test_decode_batches(batch, ctx, ws):
    check_decode([max(1, ctx - i % 19) for i in range(batch)], 4, 1, 16, 128, ws)


def test_decode_sharp_and_flat_scores(ws):
    """Scores far apart (one key takes everything, later keys raise the maximum) and all equal."""
    g = gen(9)
    q = torch.randn(2, 4 * 128, generator=g, device=DEV)
    q[0] *= 40
    q[1] = 0
    check_decode([700, 700], 4, 2, 64, 64, ws, q=q.to(torch.bfloat16))


def test_decode_query_magnitudes(ws):
    """The query is scaled by a power of two on its way to 16 bits: none overflows or vanishes."""
    g = gen(10)
    q = torch.randn(4, 4 * 128, generator=g, device=DEV) * torch.tensor([1e-30, 1e-4, 1.0, 100.0], device=DEV)[:, None]
    q[2, ::7] *= 1e-4
    check_decode([100, 100, 100, 100], 4, 1, 16, 64, ws, q=q.to(torch.bfloat16))


def test_decode_nan_query_stays_in_its_head(ws):
    g = gen(11)
    cache, tables, values = filled(g, [50], 2, 16, 64)
    q = torch.randn(1, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    q[0, 130] = float("nan")
    out = torch.empty_like(q)
    ops.paged_decode4(q, cache, tables, torch.tensor([50], dtype=torch.int32, device=DEV), out, 4, SCALE, ws)
    assert bool(out[0, 128:256].isnan().all())
    assert bool(out[0, :128].isfinite().all()) and bool(out[0, 256:].isfinite().all())


def test_decode_on_another_stream_and_in_a_graph(ws):
    """The call goes to the current stream, and a captured call follows new lengths and tables."""
    g = gen(12)
    cache, tables, values = filled(g, [400, 90], 2, 64, 64)
    ctx = torch.tensor([400, 90], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 8 * 128, generator=g, device=DEV).to(torch.bfloat16)
    exp = ops.paged_decode4(q, cache, tables, ctx, torch.empty_like(q), 8, SCALE, ws)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.paged_decode4(q, cache, tables, ctx, out, 8, SCALE, ws)
    side.synchronize()
    assert torch.equal(out, exp)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_decode4(q, cache, tables, ctx, out, 8, SCALE, ws)
    ctx.copy_(torch.tensor([13, 65], dtype=torch.int32))
    graph.replay()
    exp = ops.paged_decode4(q, cache, tables, ctx, torch.empty_like(q), 8, SCALE, ws)
    torch.cuda.synchronize()
    assert torch.equal(out, exp)
    check(out[:1], attention64(q[0].view(1, 8, 128), values[0][0][:, :13], values[0][1][:, :13],
                               torch.ones(1, 13, dtype=torch.bool, device=DEV)), values[0][1])


def test_offsets_past_32_bits(ws):
    """A cache of over 4 GiB: pages at its end are written, read, attended and copied."""
    g = gen(13)
    hkv, page, group = 8, 128, 64
    pages = (1 << 32) // (hkv * page * 144) + 40
    cache = torch.zeros(ops.kv4_cache_shape(pages, hkv, page, group), dtype=torch.uint8, device=DEV)
    assert cache.numel() > 1 << 32
    n, last = 200, [pages - 1, pages - 7]
    k, v = rows(g, n, hkv).flatten(1), rows(g, n, hkv).flatten(1)
    pos = torch.arange(n, device=DEV)
    slots = torch.tensor(last, device=DEV)[pos // page] * page + pos % page
    ops.kv4_write(k, v, cache, slots)
    small = torch.zeros(ops.kv4_cache_shape(2, hkv, page, group), dtype=torch.uint8, device=DEV)
    ops.kv4_write(k, v, small, pos)
    assert torch.equal(cache[last], small)
    assert torch.equal(ops.kv4_read(cache, slots)[1], ops.kv4_read(small, pos)[1])
    q = torch.randn(1, 16 * 128, generator=g, device=DEV).to(torch.bfloat16)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    a = ops.paged_decode4(q, cache, torch.tensor([last], dtype=torch.int32, device=DEV), ctx, torch.empty_like(q), 16,
                          SCALE, ws)
    b = ops.paged_decode4(q, small, torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), ctx, torch.empty_like(q), 16,
                          SCALE, ws)
    assert torch.equal(a, b)
    q = q.expand(n, -1).contiguous()
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    a = ops.paged_prefill4(q, cache, torch.tensor([last], dtype=torch.int32, device=DEV), cu, ctx, torch.empty_like(q),
                           16, SCALE, ws)
    b = ops.paged_prefill4(q, small, torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), cu, ctx,
                           torch.empty_like(q), 16, SCALE, ws)
    assert torch.equal(a, b)
    ops.copy_pages([cache], last, [pages - 2, 3])
    assert torch.equal(cache[[pages - 2, 3]], small)


def test_decode_page_outside_the_cache_is_an_error(ws):
    g = gen(14)
    cache, tables, _ = filled(g, [40], 1, 16, 64)
    tables[0, 1] = 1 << 20
    q = torch.randn(1, 128, generator=g, device=DEV).to(torch.bfloat16)
    ops.paged_decode4(q, cache, tables, torch.tensor([40], dtype=torch.int32, device=DEV), torch.empty_like(q), 1,
                      SCALE, ws)
    assert ops.check_device_error() != 0


def test_an_error_leaves_no_state_behind(ws):
    """Clearing an error returns a workspace's arrival counters to zero, whatever the failed call left in them."""
    g = gen(15)
    cache, tables, _ = filled(g, [3000, 90], 2, 64, 64)
    ctx = torch.tensor([3000, 90], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 8 * 128, generator=g, device=DEV).to(torch.bfloat16)
    exp = ops.paged_decode4(q, cache, tables, ctx, torch.empty_like(q), 8, SCALE, ws)
    used = ops.kv4_workspace(DEV)
    used.fill_(1)
    ops.kv4_write(rows(g, 1, 2), rows(g, 1, 2), cache, torch.tensor([1 << 40], device=DEV))
    assert ops.check_device_error() != 0
    assert torch.equal(ops.paged_decode4(q, cache, tables, ctx, torch.empty_like(q), 8, SCALE, used), exp)


def check_prefill(new, old, heads, hkv, page, group, ws, seed=0, q=None):
    """Packed sequences of ``new`` tokens after ``old`` cached ones.

    Besides :func:`check`'s terms the operands are rounded to 11 bits: were a
    group's scale x zero point rounded once (up to twice the largest value), a
    score would move by about 0.005 for these inputs, three times that at worst
    over half of the value range: 2^-7 of it. Over a whole result the differences
    average out to below half a bf16 step (2^-8)."""
    g = gen(seed + page + group + heads)
    contexts = [a + b for a, b in zip(new, old)]
    cache, tables, values = filled(g, contexts, hkv, page, group)
    ctx = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    total = sum(new)
    if q is None:
        q = torch.randn(total, (heads + 2) * 128, generator=g, device=DEV).to(torch.bfloat16)[:, 128:-128]
    out = torch.full((total, heads * 128 + 8), float("nan"), dtype=torch.bfloat16, device=DEV)[:, :heads * 128]
    ops.paged_prefill4(q, cache, tables, cu, ctx, out, heads, SCALE, ws)
    again = torch.empty_like(out)
    ops.paged_prefill4(q, cache, tables, cu, ctx, again, heads, SCALE, ws)
    assert torch.equal(out, again)
    at = 0
    for i, n in enumerate(new):
        key = torch.arange(contexts[i], device=DEV)
        seen = key[None] <= old[i] + torch.arange(n, device=DEV)[:, None]
        if n == 0:
            continue
        exp = attention64(q[at:at + n].reshape(n, heads, 128), *values[i], seen)
        got = out[at:at + n].double()
        top = float(values[i][1].abs().max())
        err = (got - exp).abs()
        assert bool((err <= exp.abs() * 2 ** -8 + top * 2 ** -7).all()), float(err.max() / top)
        assert float(err.norm() / exp.norm()) <= 2 ** -8
        at += n
    return out


@pytest.mark.parametrize("group", ops.KV4_GROUPS)
@pytest.mark.parametrize("page", [16, 48, 64, 128, 256])
def test_prefill_ragged(page, group, ws):
    check_prefill([1, 2, 0, 31, 32, 33, 64, 65, 100, 0, 7], [0, 5, 9, 0, 127, 128, 300, 0, 17, 0, 250], 8, 2, page,
                  group, ws)


@pytest.mark.parametrize("n", [1, 127, 128, 129, 255, 256, 257, 511, 700])
@pytest.mark.parametrize("old", [0, 1, 128])
def test_prefill_lengths(n, old, ws):
    check_prefill([n], [old], 2, 2, 64, 64, ws)


@pytest.mark.parametrize("per", list(range(1, 17)))
def test_prefill_query_heads_per_kv_head(per, ws):
    check_prefill([75, 1, 140], [11, 40, 0], 2 * per, 2, 64, 64 if per % 2 else 32, ws)


def test_prefill_both_tile_widths(ws):
    """Enough rows for two tiles per CTA, and the same rows in calls that take one."""
    g = gen(20)
    new, old = [1200, 300, 900], [100, 0, 33]
    q = torch.randn(sum(new), 16 * 128, generator=g, device=DEV).to(torch.bfloat16)
    check_prefill(new, old, 16, 8, 64, 64, ws, q=q)


@pytest.mark.parametrize("new,old", [([5], [3000]), ([33, 1], [1500, 130]), ([64], [1]), ([128], [2000])])
def test_prefill_few_rows_split_their_keys(new, old, ws):
    """Too few tiles for the SMs: several CTAs share a long context, some of them past its end."""
    check_prefill(new, old, 4, 1, 64, 64, ws)


def test_prefill_many_short_sequences(ws):
    check_prefill([1 + i % 5 for i in range(90)], [i % 41 for i in range(90)], 4, 2, 16, 64, ws)


def test_prefill_sharp_and_flat_scores(ws):
    g = gen(21)
    q = torch.randn(300, 4 * 128, generator=g, device=DEV)
    q[::2] *= 40
    q[1::4] = 0
    q[5] *= 1e-30
    q[7] *= 1e4
    # a score of a query 40 (10^4) times as long moves 40 times as much: only the flat rows are checked as tightly
    cache, tables, values = filled(g, [300], 2, 64, 64)
    ctx = torch.tensor([300], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    q = q.to(torch.bfloat16)
    out = ops.paged_prefill4(q, cache, tables, cu, ctx, torch.empty_like(q), 4, SCALE, ws)
    seen = torch.ones(300, 300, dtype=torch.bool, device=DEV).tril()
    exp = attention64(q.view(300, 4, 128), *values[0], seen)
    top = float(values[0][1].abs().max())
    err = (out.double() - exp).abs()
    assert bool((err[1::2] <= exp[1::2].abs() * 2 ** -8 + top * 2 ** -7)[[i for i in range(150) if i != 3]].all())
    assert bool((err <= exp.abs() * 2 ** -8 + top * 0.5).all()) and bool(out.isfinite().all())


def test_prefill_nothing_to_see(ws):
    """More new tokens than context: rows before the first cached token give zeros."""
    g = gen(22)
    cache, tables, values = filled(g, [20], 2, 16, 64)
    q = torch.randn(200, 2 * 128, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    ops.paged_prefill4(q, cache, tables, torch.tensor([0, 200], dtype=torch.int32, device=DEV),
                       torch.tensor([20], dtype=torch.int32, device=DEV), out, 2, SCALE, ws)
    assert bool((out[:180] == 0).all())
    exp = attention64(q[180:].view(20, 2, 128), *values[0], torch.ones(20, 20, dtype=torch.bool, device=DEV).tril())
    assert bool(((out[180:].double() - exp).abs() <= exp.abs() * 2 ** -8 + float(values[0][1].abs().max()) * 2 ** -7).all())


def test_prefill_agrees_with_decode(ws):
    """The last token of a prefill is a decode over the same cache."""
    g = gen(23)
    cache, tables, values = filled(g, [333, 70], 2, 64, 32)
    ctx = torch.tensor([333, 70], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 8 * 128, generator=g, device=DEV).to(torch.bfloat16)
    a = ops.paged_decode4(q, cache, tables, ctx, torch.empty_like(q), 8, SCALE, ws)
    b = ops.paged_prefill4(q, cache, tables, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), ctx,
                           torch.empty_like(q), 8, SCALE, ws)
    top = float(values[0][1].abs().max())
    assert bool(((a.float() - b.float()).abs() <= a.float().abs() * 2 ** -7 + top * 2 ** -7).all())


def test_prefill_page_outside_the_cache_is_an_error(ws):
    g = gen(24)
    cache, tables, _ = filled(g, [40], 1, 16, 64)
    tables[0, 1] = -5
    q = torch.randn(40, 128, generator=g, device=DEV).to(torch.bfloat16)
    ops.paged_prefill4(q, cache, tables, torch.tensor([0, 40], dtype=torch.int32, device=DEV),
                       torch.tensor([40], dtype=torch.int32, device=DEV), torch.empty_like(q), 1, SCALE, ws)
    assert ops.check_device_error() != 0


@pytest.mark.parametrize("offsets", [[0, 40, 300], [-7, 40, 100], [0, 90, 60], [200, 240, 300], [0, 40, 1 << 30]])
def test_prefill_offsets_outside_the_rows_are_an_error(offsets, ws):
    """No row outside q is read or written; the sequences that are inside are answered."""
    g = gen(25)
    cache, tables, values = filled(g, [50, 60], 2, 16, 64)
    ctx = torch.tensor([50, 60], dtype=torch.int32, device=DEV)
    base = torch.randn(400, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    q, outs = base[100:200], torch.full((400, 4 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_prefill4(q, cache, tables, torch.tensor(offsets, dtype=torch.int32, device=DEV), ctx, outs[100:200], 4, SCALE, ws)
    assert ops.check_device_error() != 0
    assert bool((outs[:100] == 7).all()) and bool((outs[200:] == 7).all())
    for i, n in enumerate((50, 60)):
        lo, hi = offsets[i], offsets[i + 1]
        if 0 <= lo <= hi <= 100:
            seen = torch.arange(n, device=DEV)[None] <= n - (hi - lo) + torch.arange(hi - lo, device=DEV)[:, None]
            live = seen.any(1)
            exp = attention64(q[lo:hi][live].reshape(-1, 4, 128), *values[i], seen[live])
            assert bool(((outs[100 + lo:100 + hi][live].double() - exp).abs() <= exp.abs() * 2 ** -8 +
                         float(values[i][1].abs().max()) * 2 ** -7).all())
            assert bool((outs[100 + lo:100 + hi][~live] == 0).all())


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_a_context_longer_than_its_table_is_an_error(op, ws):
    g = gen(26)
    cache, tables, values = filled(g, [40, 50], 2, 16, 64, extra_cols=0)       # 4 pages a row
    q = torch.randn(2, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    def call(ctx):
        ctx = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        if op == "decode":
            return ops.paged_decode4(q, cache, tables, ctx, out, 4, SCALE, ws).clone()
        cu = torch.arange(3, dtype=torch.int32, device=DEV)
        return ops.paged_prefill4(q, cache, tables, cu, ctx, out, 4, SCALE, ws).clone()
    exp = call([40, 50])
    assert ops.check_device_error() == 0
    got = call([40, 65])
    assert ops.check_device_error() != 0
    assert torch.equal(got[0], exp[0])


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_one_bad_page_spoils_its_own_sequence_only(op, ws):
    """An index that was not followed stays in the error word until it is read; calls meanwhile wait as long as they need."""
    g = gen(27)
    contexts = [40] + [3000] * 40
    cache, tables, _ = filled(g, contexts, 2, 64, 64, extra_cols=0)
    ctx = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    cu = torch.arange(42, dtype=torch.int32, device=DEV)
    q = torch.randn(41, 8 * 128, generator=g, device=DEV).to(torch.bfloat16)
    def call(tables):
        if op == "decode":
            return ops.paged_decode4(q, cache, tables, ctx, torch.empty_like(q), 8, SCALE, ws)
        return ops.paged_prefill4(q, cache, tables, cu, ctx, torch.empty_like(q), 8, SCALE, ws)
    exp, bad = call(tables), tables.clone()
    bad[0, 0] = 1 << 20
    assert torch.equal(call(bad)[1:], exp[1:])
    for _ in range(20):                      # the error has not been read
        assert torch.equal(call(tables), exp)
    assert ops.check_device_error() == 6     # an index out of range, no wait that gave up


# ----------------------------------------------------------------- magnitudes

def held(g, k, v, page, group):
    """One sequence's cache of the rows k / v [n, hkv, 128], its table and the values it stands for: float64 [hkv, n, 128] each."""
    n, hkv = k.shape[:2]
    need = -(-n // page)
    perm = torch.randperm(need + 1, generator=g, device=DEV)[:need]
    cache = empty_cache(need + 1, hkv, page, group)
    pos = torch.arange(n, device=DEV)
    ops.kv4_write(k.to(torch.bfloat16), v.to(torch.bfloat16), cache, perm[pos // page] * page + pos % page)
    rec = ref.kv4_values(cache[perm]).double()
    return cache, perm.to(torch.int32)[None], [rec[:, :, :, w].permute(1, 0, 2, 3, 4).reshape(hkv, -1, 128)[:, :n]
                                               for w in (0, 1)]


def attend(op, q, cache, tables, n, ws):
    """The last len(q) queries of n cached tokens, by prefill, or each over all of them, by decode."""
    m, heads = q.shape[0], q.shape[1] // 128
    out = torch.full_like(q, float("nan"))
    if op == "decode":
        ctx = torch.full((m,), n, dtype=torch.int32, device=DEV)
        return ops.paged_decode4(q, cache, tables.expand(m, -1).contiguous(), ctx, out, heads, SCALE, ws)
    cu = torch.tensor([0, m], dtype=torch.int32, device=DEV)
    return ops.paged_prefill4(q, cache, tables, cu, torch.tensor([n], dtype=torch.int32, device=DEV), out, heads, SCALE, ws)


def check_magnitudes(op, q, k, v, page, group, ws, g):
    """Every row's every channel group against its own norm.

    The result is rounded to bf16 (2^-9 of each channel) and its weights have a common error (of the sum, of a dominant
    key's score) of up to 2^-9: together 2^-8 of the norm. Each key's share p |v| is off by its own roundings to 11 bits
    (weight; in prefill K's and V's two each, those of K moving a score of a few units by some 2^-11): independent
    between keys, rms below 2^-10 sqrt(sum (p |v|)^2), of which twice is allowed."""
    n, hkv = k.shape[:2]
    cache, tables, (k64, v64) = held(g, k, v, page, group)
    got = attend(op, q, cache, tables, n, ws).double().view(q.shape[0], hkv, -1, 128 // group, group)
    qq = q.double().view(q.shape[0], hkv, -1, 128)
    s = torch.einsum("mhgd,hkd->mhgk", qq, k64) * SCALE
    if op == "prefill":
        late = torch.arange(n, device=DEV)[None] > n - q.shape[0] + torch.arange(q.shape[0], device=DEV)[:, None]
        s = s.masked_fill(late[:, None, None], float("-inf"))
    p = torch.softmax(s, -1)
    exp = torch.einsum("mhgk,hkd->mhgd", p, v64).unflatten(-1, (-1, group))
    share = torch.einsum("mhgk,hkx->mhgx", p * p, v64.unflatten(-1, (-1, group)).square().sum(-1)).sqrt()
    err, bound = (got - exp).norm(dim=-1), 2 ** -8 * exp.norm(dim=-1) + 2 ** -9 * share
    assert bool((err <= bound).all()), float((err / bound).max())
    return p


OPS = ["decode", "prefill"]


@pytest.mark.parametrize("group", ops.KV4_GROUPS)
@pytest.mark.parametrize("size", [1e3, 1.0, 1e-2, 1e-4, 1e-5, 1e-6, 1e-7, 1e-12, 1e-30])
@pytest.mark.parametrize("op", OPS)
def test_values_of_any_size(op, size, group, ws):
    g = gen(30)
    q = torch.randn(5, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    check_magnitudes(op, q, rows(g, 700, 2).float(), rows(g, 700, 2).float() * size, 64, group, ws, g)


@pytest.mark.parametrize("size", [1e4, 1.0, 1e-3, 1e-5, 1e-6, 1e-9, 1e-20])
@pytest.mark.parametrize("op", OPS)
def test_keys_of_any_size(op, size, ws):
    """Keys that are small where queries are large: the scores are the same."""
    g = gen(31)
    q = (torch.randn(5, 4 * 128, generator=g, device=DEV) / size * 1.5).to(torch.bfloat16)
    k = torch.randn(700, 2, 128, generator=g, device=DEV) * size
    check_magnitudes(op, q, k.clamp(-8000, 8000), rows(g, 700, 2).float(), 64, 64, ws, g)


@pytest.mark.parametrize("op", OPS)
def test_tokens_of_different_sizes(op, ws):
    """Values from 1e-6 to 1e2 side by side, small ones first and last."""
    g = gen(32)
    n = 1500
    size = 10 ** (torch.rand(n, generator=g, device=DEV) * 8 - 6)
    size[:200] = 1e-6
    size[-300:] = 1e-4
    q = torch.randn(5, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    check_magnitudes(op, q, rows(g, n, 2, wide=1.0).float(), rows(g, n, 2).float() * size[:, None, None], 48, 32, ws, g)


@pytest.mark.parametrize("op", OPS)
def test_zero_values_before_others(op, ws):
    """Pieces whose groups are all zero, and then values of an ordinary size."""
    g = gen(33)
    v = rows(g, 900, 2).float()
    v[:400] = 0
    v[-130:] = 0
    q = torch.randn(5, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    check_magnitudes(op, q, rows(g, 900, 2, wide=1.0).float(), v, 64, 64, ws, g)


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("op", OPS)
def test_channel_groups_of_different_sizes(op, group, ws):
    """A group of channels 1e6 times smaller than its neighbours is as precise as they are."""
    g = gen(34)
    v = rows(g, 3000, 1).float()
    v[..., group:2 * group] *= 1e-6
    q = torch.randn(3, 4 * 128, generator=g, device=DEV).to(torch.bfloat16)
    check_magnitudes(op, q, rows(g, 3000, 1, wide=1.0).float(), v, 64, group, ws, g)


@pytest.mark.parametrize("at", [0, 17000, -40])
@pytest.mark.parametrize("nats,size", [(10.0, 1.0), (13.0, 1.0), (13.0, 1e-2), (14.0, 1e-5), (15.5, 1e-2)])
@pytest.mark.parametrize("op", OPS)
def test_a_dominant_key_with_a_small_value_row(op, nats, size, at, ws):
    """One key of 32768 takes most of the weight and has next to no value: the others' small weights make the result."""
    g = gen(35)
    n = 32768
    u = torch.randn(128, generator=g, device=DEV).sign()
    q = (u + 0.2 * torch.randn(3, 4, 128, generator=g, device=DEV)).flatten(1).to(torch.bfloat16)
    k = torch.randn(n, 1, 128, generator=g, device=DEV) * 0.5
    k[at] = u * nats / (128 * SCALE)
    v = torch.randn(n, 1, 128, generator=g, device=DEV) * size
    v[at] *= 1e-5
    p = check_magnitudes(op, q, k, v, 64, 64, ws, g)
    assert float(p.amax(-1).min()) > 0.3


@pytest.mark.parametrize("kind", ["int4", "bf16", "bytes16"])
@pytest.mark.parametrize("layers,pages,moves", [(1, 2, 1), (3, 40, 20), (200, 9, 3), (2, 1300, 600)])
def test_copy_pages(kind, layers, pages, moves):
    g = gen(layers + pages)
    shape = {"int4": ops.kv4_cache_shape(pages, 2, 16, 64), "bf16": (pages, 2, 16, 128), "bytes16": (pages, 16)}[kind]
    caches = [torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8) for _ in range(layers)]
    if kind == "bf16":
        caches = [c.to(torch.bfloat16) for c in caches]
    exp = [c.clone() for c in caches]
    perm = torch.randperm(pages, generator=g, device=DEV).tolist()
    src, dst = perm[:moves], perm[moves:2 * moves]
    src[-1] = src[0]                       # one page may be copied to several
    ops.copy_pages(caches, src, dst)
    ref.copy_pages(exp, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(caches, exp))


# ----------------------------------------------------------------- refusals

def test_refusals(ws):
    cache = empty_cache(4, 2, 16, 64)
    k = torch.zeros(3, 256, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(3, device=DEV)
    for bad in (dict(cache=cache[..., :1100].contiguous()), dict(cache=cache.view(torch.int8)), dict(cache=cache[:, :1]),
                dict(k=k.float()), dict(k=k[:, :128]), dict(k=k[:2]), dict(k=k.cpu()), dict(slots=slots.int()),
                dict(slots=slots[:2]), dict(slots=slots.cpu()), dict(k=torch.zeros(256, 3, dtype=torch.bfloat16, device=DEV).t())):
        a = dict(dict(cache=cache, k=k, slots=slots), **bad)
        with pytest.raises(ValueError):
            ops.kv4_write(a["k"], k, a["cache"], a["slots"])
    with pytest.raises(ValueError):
        ops.kv4_read(cache, slots.int())
    q = torch.zeros(2, 4 * 128, dtype=torch.bfloat16, device=DEV)
    tables = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    ctx = torch.ones(2, dtype=torch.int32, device=DEV)
    good = dict(q=q, cache=cache, tables=tables, ctx=ctx, out=torch.empty_like(q), heads=4, ws=ws)
    ops.paged_decode4(q, cache, tables, ctx, good["out"], 4, SCALE, ws)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(heads=3), dict(heads=0), dict(heads=8), dict(tables=tables.long()),
                dict(tables=tables[:1]), dict(ctx=ctx.long()), dict(ctx=ctx[:1]), dict(ws=ws[:100]), dict(out=q.float()),
                dict(out=q.cpu()), dict(ctx=ctx.cpu()), dict(q=torch.zeros(2, 4 * 128 + 4, dtype=torch.bfloat16, device=DEV)[:, 4:])):
        a = dict(good, **bad)
        with pytest.raises(ValueError):
            ops.paged_decode4(a["q"], a["cache"], a["tables"], a["ctx"], a["out"], a["heads"], SCALE, a["ws"])
    with pytest.raises(ValueError):
        ops.paged_decode4(q, cache, tables, ctx, good["out"], 4, 0.0, ws)
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    good["cu"] = cu
    ops.paged_prefill4(q, cache, tables, cu, ctx, good["out"], 4, SCALE, ws)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(heads=3), dict(heads=8), dict(tables=tables.long()),
                dict(tables=tables[:1]), dict(ctx=ctx.long()), dict(ctx=ctx[:1]), dict(ws=ws[:100]), dict(cu=cu.long()),
                dict(cu=cu[:2]), dict(cu=cu.cpu()), dict(out=q.float()),
                dict(out=torch.zeros(2, 4 * 128 + 4, dtype=torch.bfloat16, device=DEV)[:, 4:])):
        a = dict(good, **bad)
        with pytest.raises(ValueError):
            ops.paged_prefill4(a["q"], a["cache"], a["tables"], a["cu"], a["ctx"], a["out"], a["heads"], SCALE, a["ws"])
    wide = torch.zeros(2, 34 * 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        ops.paged_decode4(wide, cache, tables, ctx, torch.empty_like(wide), 34, SCALE, ws)


@pytest.mark.parametrize("shape", [(0, 1, 1), (2, 0, 1), (2, 1, 0)])
def test_an_empty_cache_is_refused(shape, ws):
    cache = torch.zeros(*shape, 2, 1152, dtype=torch.uint8, device=DEV)
    q = torch.zeros(1, 128, dtype=torch.bfloat16, device=DEV)
    one, cu = torch.ones(1, dtype=torch.int32, device=DEV), torch.arange(2, dtype=torch.int32, device=DEV)
    tables, slots = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    k = torch.zeros(1, shape[1] * 128, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: ops.kv4_write(k, k, cache, slots), lambda: ops.kv4_read(cache, slots),
                 lambda: ops.paged_decode4(q, cache, tables, one, q.clone(), 1, 1.0, ws),
                 lambda: ops.paged_prefill4(q, cache, tables, cu, one, q.clone(), 1, 1.0, ws)):
        with pytest.raises(ValueError):
            call()


def test_tables_of_too_many_tokens_are_refused(ws):
    """The token count of a table row is 32 bits."""
    cache = empty_cache(1, 1, 1 << 16, 64)
    q = torch.zeros(1, 128, dtype=torch.bfloat16, device=DEV)
    one, cu = torch.ones(1, dtype=torch.int32, device=DEV), torch.arange(2, dtype=torch.int32, device=DEV)
    tables = torch.zeros(1, 1 << 15, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        ops.paged_decode4(q, cache, tables, one, q.clone(), 1, SCALE, ws)
    with pytest.raises(ValueError):
        ops.paged_prefill4(q, cache, tables, cu, one, q.clone(), 1, SCALE, ws)


def test_copy_refusals():
    caches = [empty_cache(4, 1, 16, 64) for _ in range(2)]
    for src, dst in (([0], [1, 2]), ([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0])):
        with pytest.raises(ValueError):
            ops.copy_pages(caches, src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages([caches[0], empty_cache(5, 1, 16, 64)], [0], [1])
    with pytest.raises(ValueError):
        ops.copy_pages([torch.zeros(4, 10, dtype=torch.uint8, device=DEV)], [0], [1])
    ops.copy_pages(caches, [], [])
