"""Steps over "int4" pages at the borders of what the plugin's objects and the entry points let through."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import crit_b200 as pk
from crit_b200.attention import DeviceAttention
from crit_b200.batch import StepBatch
from crit_b200.pool import KVPool
from test_int4_gpu import _attend, _queries
from int4_oracle import Cache4, attention4, bounds4

pytestmark = pytest.mark.gpu


def _filled_pool(kind, rows, length, columns, hkv, dim, seed, **kw):
    """A pool of `rows` sequences of `length` positions, and the step that adds `columns` more to each: (pool, batch)."""
    pool = KVPool([0], hkv, dim, rows * (length + columns + 16), "cuda", kind, sequences=rows, **kw)
    g = torch.Generator().manual_seed(seed)
    for first, count in ((0, length), (length, columns)):
        if first == 0:
            for r in range(rows):
                pool.open(r)
        batch = StepBatch.build([(r, first, count) for r in range(rows)], "cuda")
        slots = pool.reserve(batch)
        make = lambda: torch.randn(batch.tokens, hkv, dim, generator=g).bfloat16().cuda()
        pool.write(0, slots, make(), make())
    return pool, batch


def _as_cache(pool):
    cache = Cache4.__new__(Cache4)
    cache.heads, cache.dim, cache.page = pool.kv_heads, pool.head_dim, pool.page
    cache.k, cache.v, cache.ks, cache.vs = pool.layer_pages(0)
    pool._flush()
    cache.tables = torch.stack([pool.block_tables[pool.row_of[r]] for r in pool.tables])
    return cache


def _round(rows, columns, length):
    """The same step as a captured round has it: sequences in round slots, a width for all."""
    return SimpleNamespace(round=True, prompt=False, rows=rows, width=columns - 1, tokens=rows * columns, slots_t=torch.arange(rows, device="cuda"),
                           starts_t=torch.arange(rows, dtype=torch.int32, device="cuda") * columns,
                           frontier_t=torch.full((rows,), length, device="cuda"))


def _lists(rows, columns, length, block, seed):
    """Lists of four blocks a token: its own, two of its context's, and none."""
    g = torch.Generator().manual_seed(seed)
    own = (length + torch.arange(columns)) // block
    picks = torch.randint(0, length // block, (rows * columns, 2), generator=g)
    return torch.cat([own.repeat(rows)[:, None], picks, torch.full((rows * columns, 1), -1)], 1).to(torch.int32).cuda()


@pytest.mark.parametrize("rows,columns", [(64, 6), (43, 6), (257, 1)])
def test_lists_of_whole_pages_over_more_tokens_than_an_even_launch_has_rows(rows, columns):
    length = 70
    pool, batch = _filled_pool("int4", rows, length, columns, 2, 64, 1, round_rows=256)
    q = torch.randn(rows * columns, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    blocks = _lists(rows, columns, length, 32, 3)
    cache = _as_cache(pool)
    found = [DeviceAttention().forward(0, q, pool, batch, blocks=blocks, block_size=32, lse=True)]         # (as a mask)
    if rows <= 256:
        for r in range(rows):
            pool.bind(r, r, length + columns)
        found.append(DeviceAttention().forward(0, q, pool, _round(rows, columns, length), blocks=blocks, block_size=32, lse=True))
    for r in (0, rows // 2, rows - 1):
        for c in range(columns):
            t = r * columns + c
            want, want_lse, room = attention4(cache, q[t], r, length, c, columns, t, blocks=blocks, block_size=32)
            for out, lse in found:
                assert (np.abs(out[t].double().cpu().numpy() - want) <= bounds4(want, room, length + columns, q.dtype)).all()
                assert (np.abs(lse[t].double().cpu().numpy() - want_lse) <= 3e-4).all()
    args = (q, *pool.layer_pages(0)[:2], "int4", pool.block_tables, torch.arange(rows, dtype=torch.int32, device="cuda"),
            torch.arange(rows, dtype=torch.int32, device="cuda") * columns, torch.full((rows,), length, device="cuda"), columns, pool.page)
    kw = dict(key_scales=cache.ks, value_scales=cache.vs, blocks=blocks, block_size=32)
    named = pk.attend(*args, engine="even" if rows <= 256 else "mma.sync", **kw)                # named for the caller's rows
    chosen = pk.attend(*args, **kw)
    assert torch.equal(named, chosen) and pk.status() == 0


def test_lists_over_many_tokens_of_fp8_pages_read_by_whole_rows():
    """The same rule for the other kernels that list their rows."""
    rows, columns, length = 64, 6, 70
    pool, batch = _filled_pool("fp8:page", rows, length, columns, 8, 128, 4, round_rows=rows)
    for r in range(rows):
        pool.bind(r, r, length + columns)
    q = torch.randn(rows * columns, 8, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    assert pk.engine_for("fp8:page", 128, 128, 8, 8, columns, rows, pool.block_tables.shape[1] * pool.page) == "tcgen05p"
    blocks = _lists(rows, columns, length, 32, 6)
    for step in (_round(rows, columns, length), batch):
        out, lse = DeviceAttention().forward(0, q, pool, step, blocks=blocks, block_size=32, lse=True)
        want, want_lse = DeviceAttention(window_engine="mma.sync").forward(0, q, pool, step, blocks=blocks, block_size=32, lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and pk.status() == 0


@pytest.mark.parametrize("engine", [None, "mma.sync", 64])
@pytest.mark.parametrize("columns", [1, 4])
def test_rows_that_end_or_begin_past_their_page_table(engine, columns):
    """A table of 7 pages of 16 (no multiple of a split), the last row of its tensor, with ids behind it that are no pages: a row
    that ends past it reads nothing there, its columns within it are as they should be; a row that begins past it is reported."""
    page, width = 16, 7
    holds = page * width
    cache = Cache4.filled(8, 128, page, [holds, holds], seed=301)
    behind = torch.full((3, width), 1 << 20, dtype=torch.int32, device="cuda")
    behind[:2] = cache.tables
    cache.tables = behind[:2]
    q = _queries(2 * columns, 16, 128, torch.bfloat16, 302)
    first = holds - (1 if columns == 1 else 2)
    kw = {} if engine is None else {"engine": "mma.sync", "chunk": engine if isinstance(engine, int) else None}
    out, lse = _attend(cache, q, [0, 1], [0, columns], [50, first], columns, **kw)               # (reports nothing)
    _as_many = [columns, holds - first]
    for r, (at, n) in enumerate(zip((50, first), _as_many)):
        for c in range(n):
            t = r * columns + c
            want, want_lse, room = attention4(cache, q[t], r, at, c, n, t)
            assert (np.abs(out[t].double().cpu().numpy() - want) <= bounds4(want, room, at + n, q.dtype)).all()
            assert (np.abs(lse[t].double().cpu().numpy() - want_lse) <= 3e-4).all()
    assert out.isfinite().all()
    before = pk._status[str(q.device)].clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    for beyond in (holds, holds + 500, 1 << 40):
        out = torch.full_like(q, float("nan"))
        pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.arange(2, **i32), torch.arange(2, **i32) * columns, torch.tensor([50, beyond], device="cuda"), columns,
                  page, key_scales=cache.ks, value_scales=cache.vs, out=out, **kw)
        assert pk.status() == 2
        pk._status[str(q.device)].copy_(before)
        for c in range(columns):
            want, _, room = attention4(cache, q[c], 0, 50, c, columns, c)
            assert (np.abs(out[c].double().cpu().numpy() - want) <= bounds4(want, room, 50 + columns, q.dtype)).all()
        assert engine is not None or out[columns:].isnan().all()
    # context rows: one that sees the whole table, and one that says more
    out, lse = _attend(cache, q[:columns], [1], [0], [holds], columns, context=True, **kw)
    for c in range(columns):
        want, _, room = attention4(cache, q[c], 1, holds, c, columns, c, context=True)
        assert (np.abs(out[c].double().cpu().numpy() - want) <= bounds4(want, room, holds, q.dtype)).all()
    pk.attend(q[:columns], cache.k, cache.v, "int4", cache.tables, torch.ones(1, **i32), torch.zeros(1, **i32), torch.tensor([holds + 1], device="cuda"), columns, page,
              key_scales=cache.ks, value_scales=cache.vs, context=True, **kw)
    assert pk.status() == 2
    pk._status[str(q.device)].copy_(before)


def test_arguments_that_a_launch_would_read_or_write_past():
    cache = Cache4.filled(2, 128, 16, [40, 50, 60], seed=311)
    q = _queries(3, 8, 128, torch.bfloat16, 312)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows, firsts = torch.arange(3, **i32), torch.tensor([39, 49, 59], device="cuda")
    ok = dict(tables=cache.tables, rows=rows, starts=rows, firsts=firsts, counts=torch.ones(3, **i32), out=torch.empty_like(q))

    def attend(**change):
        a = {**ok, **change}
        return pk.attend(q, cache.k, cache.v, "int4", a.pop("tables"), a.pop("rows"), a.pop("starts"), a.pop("firsts"), 1, 16, key_scales=cache.ks,
                         value_scales=cache.vs, **a)
    attend()
    wide = torch.zeros(3, 2, **i32)
    space = torch.empty(1 << 20)
    for change, match in ((dict(rows=rows[:2]), "an entry each"), (dict(firsts=firsts[:2]), "an entry each"), (dict(counts=torch.ones(2, **i32)), "an entry each"),
                          (dict(rows=wide[:, 0]), "contiguous"), (dict(firsts=firsts.repeat(2).view(3, 2)[:, 0]), "contiguous"),
                          (dict(counts=torch.ones(3, dtype=torch.int64, device="cuda")), "int32"), (dict(out=torch.empty_like(q)[:2]), "as q"),
                          (dict(out=torch.empty(3, 8, 64, dtype=q.dtype, device="cuda")), "as q"), (dict(workspace=space), "workspace"),
                          (dict(workspace=space, engine="even"), "workspace"), (dict(workspace=space, chunk=16), "workspace")):
        with pytest.raises(ValueError, match=match):
            attend(**change)
    chunk = lambda **kw: pk.prefill(q, cache.k, cache.v, "int4", cache.tables[2], 50, 16, key_scales=cache.ks, value_scales=cache.vs, **kw)
    chunk()
    for kw, match in ((dict(out=torch.empty_like(q)[:2]), "out is"), (dict(out=torch.empty(3, 8, 128, device="cuda")), "out is"), (dict(out=torch.empty_like(q).cpu()), "out is"),
                      (dict(lse=torch.empty(2, 8, device="cuda")), "lse is"), (dict(lse=torch.empty(8, 3, device="cuda").T), "lse is"),
                      (dict(lse=torch.empty(3, 8, dtype=torch.float64, device="cuda")), "lse is"), (dict(lse=torch.empty(3, 8)), "lse is")):
        with pytest.raises(ValueError, match=match):
            chunk(**kw)
    assert pk.status() == 0


def test_a_staged_chunk_whose_padding_passes_the_table():
    """A bucket of 256 at the end of a table of 128 positions, captured: the chunk's tokens as they should be, nothing reported."""
    pool = KVPool([0], 2, 64, 128, "cuda", "int4", page=16)
    g = torch.Generator().manual_seed(321)
    make = lambda n, h: torch.randn(n, h, 64, generator=g).bfloat16().cuda()
    pool.open("a")
    step = StepBatch.build([("a", 0, 90)], "cuda")
    pool.write(0, pool.reserve(step), make(90, 2), make(90, 2))
    pool.keep("a", 90)
    chunk = SimpleNamespace(prompt=True, round=False, sequence="a", frontier=90, count=20, bucket=256, tokens_max=256, tokens=256,
                            frontier_t=torch.tensor([90], device="cuda"))
    q, keys, values, attention = make(256, 4), make(256, 2), make(256, 2), DeviceAttention()
    pool.stage_prompt(chunk)
    pool.write(0, pool.reserve(chunk), keys, values)
    out = attention.forward(0, q, pool, chunk)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = attention.forward(0, q, pool, chunk)
    for frontier, count in ((90, 20), (108, 20)):
        if frontier > 90:
            pool.commit_prompt(chunk)
            chunk.frontier, chunk.count = frontier, count
            chunk.frontier_t.fill_(frontier)
            pool.stage_prompt(chunk)
            pool.write(0, pool.reserve(chunk), keys, values)
        graph.replay()
        assert frontier > 90 or torch.equal(again[:count], out[:count])
        cache = _as_cache(pool)
        for c in (0, 7, count - 1):
            want, _, room = attention4(cache, q[c], 0, frontier, c, count, c)
            assert (np.abs(again[c].double().cpu().numpy() - want) <= bounds4(want, room, frontier + count, q.dtype)).all()
        assert pk.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_read_back_into_a_buffer_of_any_alignment(dtype):
    cache = Cache4.filled(2, 64, 16, [50], seed=331)
    want = pk.gather(cache.k, "int4", 16, table=cache.tables[0], count=50, scales=cache.ks, dtype=dtype)
    slots = cache.slots(0, torch.arange(50)).view(5, 10)
    for shift in range(0, 9):
        buffer = torch.full((50 * 128 + 16,), -1, dtype=dtype, device="cuda")
        out = buffer[shift:shift + 50 * 128].view(50, 2, 64)
        got = pk.gather(cache.k, "int4", 16, table=cache.tables[0], count=50, scales=cache.ks, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and (buffer[:shift] == -1).all() and (buffer[shift + 50 * 128:] == -1).all()
        out.zero_()
        got = pk.gather(cache.k, "int4", 16, slots=slots, scales=cache.ks, out=out)
        assert got.shape == (5, 10, 2, 64) and torch.equal(got.view_as(out), want) and torch.equal(out, want)
    assert pk.status() == 0
