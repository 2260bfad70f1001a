"""Prompt chunks over "int4" pages: the memory their 16-bit copies take, and what a launch shares with others."""
import numpy as np
import pytest
import torch

import crit_b200 as pk
from int4_oracle import Cache4, attention4
from test_int4_gpu import _queries

pytestmark = pytest.mark.gpu


def _check(cache, q, out, starts, firsts, rows=None, step=7):
    """As the windows' bounds, with weights rounded to the queries' type (the sum of them is not)."""
    half = torch.finfo(q.dtype).eps / 2
    for s, first in enumerate(firsts):
        count = starts[s + 1] - starts[s]
        for c in range(0, count, step):
            want, _, room = attention4(cache, q[starts[s] + c], s if rows is None else rows[s], first, c, count, starts[s] + c)
            err = np.abs(out[starts[s] + c].double().cpu().numpy() - want)
            assert (err <= half * np.abs(want) + (half + 2.0 ** -10) * room + 1e-6).all(), (s, c, err.max())


def _peak(call):
    """(bytes a call takes beside what it returns, its result)."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    found = call()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= (found.numel() * 2 + 4096)
    return torch.cuda.max_memory_allocated() - before, found


def _prefill(cache, q, position, **kw):
    return pk.prefill(q, cache.k, cache.v, "int4", kw.pop("table", cache.tables), position, cache.page, key_scales=cache.ks, value_scales=cache.vs, **kw)


@pytest.mark.parametrize("hq,hkv,dim", [(4, 2, 128), (2, 2, 64), (2, 1, 256)])
def test_sequences_of_unequal_lengths_take_the_pages_they_have(hq, hkv, dim):
    firsts, counts = [6000, 0, 30, 1, 500, 17, 0, 64], [20, 3, 33, 1, 16, 0, 1, 64]
    cache = Cache4.filled(hkv, dim, 16, [f + n for f, n in zip(firsts, counts)], seed=401, poison=True)
    starts = [sum(counts[:i]) for i in range(9)]
    q = _queries(starts[-1], hq, dim, torch.bfloat16, 402)
    own = sum(-(-(f + n) // 16) for f, n in zip(firsts, counts)) * 16 * hkv * dim * 4
    took, out = _peak(lambda: _prefill(cache, q, firsts, starts=starts))
    assert took <= 2 * (own + 64 * cache.tables.shape[1]) + out.numel() * 2 + (1 << 20)       # (a power of two; and far below 8 of the longest)
    _check(cache, q, out, starts, firsts)
    exact = torch.empty((own + 4 * 8 * cache.tables.shape[1] + 8 * (8 + 9)) // 4, device="cuda")     # (the pages, their table and the lists)
    assert torch.equal(_prefill(cache, q, firsts, starts=starts, workspace=exact), out)
    device = torch.tensor(firsts, device="cuda")
    assert torch.equal(_prefill(cache, q, device, starts=starts), out)
    assert pk.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_positions_on_the_device_take_no_more_than_the_pool(dtype):
    """Wide tables over few pages, which the sequences share: the copy is of the pool's pages."""
    cache = Cache4.filled(2, 128, 16, [200, 90], seed=411)
    pool = cache.tables.numel() + 1
    wide = torch.full((24, 3000), 1 << 28, dtype=torch.int32, device="cuda")                 # (what is not read may hold anything)
    rows = [s % 2 for s in range(24)]
    wide[:, :cache.tables.shape[1]] = cache.tables[torch.tensor(rows, device="cuda")]
    firsts = [190 - s if s % 2 == 0 else 80 - s for s in range(24)]
    starts = [5 * s for s in range(25)]
    q = _queries(starts[-1], 4, 128, dtype, 412)
    position = torch.tensor(firsts, device="cuda")
    took, out = _peak(lambda: _prefill(cache, q, position, table=wide))
    assert took <= pool * 16 * 2 * 128 * 4 + wide.numel() * 4 + out.numel() * 2 + (3 << 20)
    _check(cache, q, out, starts, firsts, rows)
    assert torch.equal(_prefill(cache, q, firsts, table=wide, starts=starts), out) and pk.status() == 0


def test_a_prompt_that_grows_holds_nothing_between_its_chunks():
    cache = Cache4.filled(8, 128, 16, [3000], seed=421)
    q = _queries(3000, 8, 128, torch.bfloat16, 422)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    kept, before = len(pk._retired), torch.cuda.memory_allocated()
    for at in range(0, 3000, 100):
        _prefill(cache, q[at:at + 100], at, table=cache.tables[0], out=out[at:at + 100])
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before and len(pk._retired) == kept
    _check(cache, q, out, [0, 3000], [0], step=271)


def test_positions_on_the_device_outside_the_table_are_reported():
    """They are brought within it, so that nothing past the table is read."""
    for hq, hkv, dim in ((4, 2, 128), (2, 1, 64), (2, 1, 256)):
        cache = Cache4.filled(hkv, dim, 16, [112, 112], seed=431)
        q = _queries(20, hq, dim, torch.bfloat16, 432)
        before = pk._status[str(q.device)].clone()
        for bad, is_read in ((103, 102), (1 << 40, 102), (-1, 0), (-(1 << 40), 0)):
            out = _prefill(cache, q, torch.tensor([50, bad], device="cuda"))
            assert pk.status() == 2
            pk._status[str(q.device)].copy_(before)
            _check(cache, q, out, [0, 10, 20], [50, is_read])
            out = _prefill(cache, q[:10], torch.tensor([bad], device="cuda"), table=cache.tables[1])
            assert pk.status() == 2
            pk._status[str(q.device)].copy_(before)
            _check(cache, q, out, [0, 10], [is_read], [1])
        for bad in (103, -1):
            with pytest.raises(ValueError, match="position"):
                _prefill(cache, q, [50, bad])
            with pytest.raises(ValueError, match="position"):
                _prefill(cache, q[:10], bad, table=cache.tables[1])
        with pytest.raises(ValueError, match="page table"):
            _prefill(cache, _queries(2 * 113, hq, dim, torch.bfloat16, 433), torch.zeros(2, dtype=torch.int64, device="cuda"))
        with pytest.raises(ValueError, match="workspace"):
            _prefill(cache, q, [50, 60], workspace=torch.empty(1 << 20))


def test_a_prompt_chunk_and_a_decode_step_of_one_owner_on_two_streams():
    cache = Cache4.filled(8, 128, 16, [9000, 700], seed=441)
    q, chunk = _queries(2, 32, 128, torch.bfloat16, 442), _queries(600, 32, 128, torch.bfloat16, 443)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows, firsts = torch.arange(2, **i32), torch.tensor([8999, 699], device="cuda")
    step = lambda out: pk.attend(q, cache.k, cache.v, "int4", cache.tables, rows, rows, firsts, 1, 16, key_scales=cache.ks, value_scales=cache.vs, out=out)
    prompt = lambda out: _prefill(cache, chunk, 8400, table=cache.tables[0], out=out)
    want = step(torch.empty_like(q)), prompt(torch.empty_like(chunk))
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    found = [[torch.empty_like(want[0]) for _ in range(30)], [torch.empty_like(want[1]) for _ in range(8)]]
    torch.cuda.synchronize()
    for i in range(30):
        if i < 8:
            with torch.cuda.stream(streams[1]):
                prompt(found[1][i])
        with torch.cuda.stream(streams[0]):
            step(found[0][i])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[0]) for x in found[0]) and all(torch.equal(x, want[1]) for x in found[1]) and pk.status() == 0


def test_a_first_prompt_chunk_may_be_captured():
    cache = Cache4.filled(2, 128, 16, [300], seed=451)
    q, out = _queries(40, 8, 128, torch.bfloat16, 452), torch.empty(40, 8, 128, dtype=torch.bfloat16, device="cuda")
    position = torch.tensor([100], device="cuda")
    want = _prefill(cache, q, 100, table=cache.tables[0])
    with pk.owner("a prompt's owner"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _prefill(cache, q, position, table=cache.tables[0], out=out)
    _prefill(cache, q, 13, table=cache.tables[0])
    for at in (100, 7):
        position.fill_(at)
        graph.replay()
        assert torch.equal(out, want if at == 100 else _prefill(cache, q, at, table=cache.tables[0]))
    assert pk.status() == 0
