"""The 4-bit page kind on a GPU against a plain implementation in 64 bits: rows written and read back, decode and verify
windows with every mask, and the runs of them that a step makes."""
import numpy as np
import pytest
import torch

import crit_b200 as pk
from int4_oracle import SCALES, Cache4, attention4, bounds4, quantise4, values4

pytestmark = pytest.mark.gpu


def _bits(x):
    return x.view(torch.int16 if x.element_size() == 2 else torch.int32).cpu()


# -- write and gather -------------------------------------------------------------------------------------------------------
ROWS = [(1, 1, 64), (3, 2, 32), (5, 3, 96), (64, 8, 128), (129, 4, 256), (1000, 1, 160)]


def _samples(tokens, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g) * torch.exp2(torch.randint(-20, 14, (tokens, heads, 1), generator=g).float())
    x[torch.rand(x.shape, generator=g) < 0.02] *= 30
    x[0, 0, :32] = 0                                                        # a group of zeros
    if tokens > 2:
        x[1, 0, :32] = torch.arange(-16, 16) * 0.5                          # quotients half way between two codes
        x[2, 0, :32] = 1e-9                                                 # below half the smallest scale
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim", ROWS)
def test_rows_are_written_and_read_back_bit_for_bit(tokens, heads, dim, dtype):
    page, pages = 16, tokens // 16 + 3
    cache = Cache4(heads, dim, page, pages)
    keys, values = _samples(tokens, heads, dim, dtype, 1), _samples(tokens, heads, dim, dtype, 2)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens].cuda()
    pk.write(keys.cuda(), values.cuda(), slots, cache.k, cache.v, "int4", cache.ks, cache.vs)
    for x, pages_, scales in ((keys, cache.k, cache.ks), (values, cache.v, cache.vs)):
        codes, byte = quantise4(x.double().numpy())
        got = pages_.flatten(0, 1)[slots].cpu().numpy()
        assert np.array_equal(got & 15, codes[..., 0::2]) and np.array_equal(got >> 4, codes[..., 1::2])
        assert np.array_equal(scales.flatten(0, 1)[slots].cpu().numpy(), byte)
        want = torch.from_numpy(values4(codes, byte))
        for out in (torch.bfloat16, torch.float16, torch.float32):
            back = pk.gather(pages_, "int4", page, slots=slots, scales=scales, dtype=out)
            assert torch.equal(_bits(back), _bits(want.to(out))), out
            assert torch.equal(back.double().cpu(), want) or out == torch.float16 and want.abs().max() > 65504
        # a code's value is at most half a scale away (below the saturation).  A scale below 2^-14 is up to 2^-18 below
        # max |x| / 7, by rounding to steps of 2^-17, so the code of 7 falls short of max |x| by 7 * 2^-18 there
        step = values4(np.full_like(codes, 9), byte)
        below = np.repeat(byte < 247, 32, -1)
        assert (np.abs(want.numpy() - np.where(below, x.double().numpy(), want.numpy())) <= step / 2 + 7 * 2.0 ** -18).all()
    # the slots that were not named are as they were
    left = torch.ones(pages * page, dtype=torch.bool)
    left[slots.cpu()] = False
    assert not cache.k.flatten(0, 1)[left.cuda()].any() and not cache.vs.flatten(0, 1)[left.cuda()].any()
    assert pk.status() == 0


def test_every_scale_with_quotients_on_and_beside_every_border():
    """For each of the 247 scales: elements half way between two codes, one step of their type beside them, and in between."""
    for dtype in (torch.bfloat16, torch.float32):
        rows = []
        for byte in range(1, 248):
            s = float(SCALES[byte])
            x = torch.tensor([(k + 0.5) * s for k in range(-7, 7)] + [(k + 0.3) * s for k in range(-7, 7)], dtype=dtype)
            around = torch.nextafter(x[:14].float(), torch.tensor(1e9)) if dtype == torch.float32 else x[:14]
            rows.append(torch.cat([x, around.to(dtype)[:3], torch.tensor([7 * s], dtype=dtype)]))
            rows.append(torch.cat([-x, -around.to(dtype)[3:6], torch.tensor([7 * s], dtype=dtype)]))
        x = torch.stack(rows).view(247, 2, 32)
        cache = Cache4(2, 32, 16, 17)
        slots = torch.arange(247).cuda()
        pk.write(x.cuda(), None, slots, cache.k, None, "int4", cache.ks, None)
        codes, byte = quantise4(x.double().numpy())
        assert np.array_equal(cache.ks.flatten(0, 1)[slots].cpu().numpy(), byte)
        got = cache.k.flatten(0, 1)[slots].cpu().numpy()
        assert np.array_equal(got & 15, codes[..., 0::2]) and np.array_equal(got >> 4, codes[..., 1::2])


def test_odd_values_in_a_group():
    x = torch.zeros(6, 1, 64)
    x[0, 0, 3] = float("nan")
    x[1, 0, 3], x[1, 0, 4] = float("inf"), -float("inf")
    x[2] = 3e38
    x[3] = -3e38
    x[4, 0, :32] = torch.finfo(torch.float32).tiny
    x[5, 0, 40] = -0.0
    cache = Cache4(1, 64, 16, 2)
    slots = torch.arange(6).cuda()
    pk.write(x.cuda(), x.cuda(), slots, cache.k, cache.v, "int4", cache.ks, cache.vs)
    back = pk.gather(cache.k, "int4", 16, slots=slots, scales=cache.ks, dtype=torch.float32).cpu()
    assert back[0, 0, :32].isnan().all() and (back[0, 0, 32:] == 0).all()
    assert back[1, 0, 3] == 7 * 61440 and back[1, 0, 4] == -7 * 61440 and back[1, 0, 5] == 0
    assert (back[2] == 7 * 61440).all() and (back[3] == -7 * 61440).all()
    assert (back[4:] == 0).all()
    assert pk.status() == 0


def test_writes_take_strides_skips_and_one_side_only():
    tokens, heads, dim, page = 37, 3, 128, 16
    cache = Cache4(heads, dim, page, 8)
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(tokens, 2 * heads + 1, dim + 8, generator=g).bfloat16().cuda()
    keys, values = wide[:, :heads, 3:dim + 3], wide[:, heads:2 * heads, :dim]          # unaligned rows, and rows apart
    slots = torch.randperm(8 * page, generator=g)[:tokens].cuda()
    slots[4] = -1
    pk.write(keys, values, slots, cache.k, cache.v, "int4", cache.ks, cache.vs)
    live = slots >= 0
    for x, pages, scales in ((keys, cache.k, cache.ks), (values, cache.v, cache.vs)):
        codes, byte = quantise4(x[live].double().cpu().numpy())
        back = pk.gather(pages, "int4", page, slots=slots[live], scales=scales, dtype=torch.float32)
        assert np.array_equal(back.cpu().numpy(), values4(codes, byte))
    other = Cache4(heads, dim, page, 8)
    pk.write(keys, None, slots, other.k, None, "int4", other.ks, None)
    pk.write(None, values, slots, None, other.v, "int4", None, other.vs)
    assert torch.equal(other.k, cache.k) and torch.equal(other.v, cache.v) and torch.equal(other.vs, cache.vs)
    # values narrower than keys
    mixed = Cache4(heads, dim, page, 8)
    narrow = Cache4(heads, 64, page, 8)
    pk.write(keys, values[..., :64], slots, mixed.k, narrow.v, "int4", mixed.ks, narrow.vs)
    assert torch.equal(mixed.k, cache.k) and torch.equal(narrow.v, cache.v[..., :32])


def test_gather_through_a_table_and_into_a_buffer():
    heads, dim, page, count = 2, 128, 32, 77
    cache = Cache4.filled(heads, dim, page, [count], seed=7)
    want = torch.from_numpy(cache.rows("k", 0, count))
    table = cache.tables[0]
    got = pk.gather(cache.k, "int4", page, table=table, count=count, scales=cache.ks, dtype=torch.float32)
    assert torch.equal(got.double().cpu(), want)
    buffer = torch.full((count + 2, heads, dim), -1, dtype=torch.bfloat16, device="cuda")
    same = pk.gather(cache.k, "int4", page, table=table, count=count, scales=cache.ks, out=buffer[1:-1])
    assert same.data_ptr() == buffer[1:-1].data_ptr() and torch.equal(same.double().cpu(), want)
    assert (buffer[0] == -1).all() and (buffer[-1] == -1).all()
    slots = cache.slots(0, torch.arange(6)).view(2, 3)
    assert pk.gather(cache.k, "int4", page, slots=slots, scales=cache.ks).shape == (2, 3, heads, dim)
    assert pk.gather(cache.k, "int4", page, slots=slots[:0], scales=cache.ks).shape == (0, 3, heads, dim)


# -- decode and verify windows ----------------------------------------------------------------------------------------------
def _check(cache, q, out, lse, rows, starts, firsts, counts, **masks):
    """Every token the rows name against the 64-bit attention, within the kernel's roundings (bounds4)."""
    for r, (row, start, first, count) in enumerate(zip(rows, starts, firsts, counts)):
        for c in range(count):
            want, want_lse, room = attention4(cache, q[start + c], row, first, c, count, start + c, **masks)
            got, got_lse = out[start + c].double().cpu().numpy(), lse[start + c].double().cpu().numpy()
            tol = bounds4(want, room, first + count, q.dtype)
            assert np.isfinite(got).all(), (r, c)
            worst = np.max(np.abs(got - want) / tol)
            assert worst <= 1, f"row {r} column {c}: {worst:.3f} of the bound"
            seen = np.isfinite(want_lse)
            assert np.array_equal(seen, np.isfinite(got_lse))
            assert (np.abs(got_lse[seen] - want_lse[seen]) <= 3e-4).all(), (r, c)


def _attend(cache, q, rows, starts, firsts, columns, counts=None, **kw):
    i32 = dict(dtype=torch.int32, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.tensor(rows, **i32), torch.tensor(starts, **i32),
              torch.tensor(firsts, device="cuda"), columns, cache.page, counts=None if counts is None else torch.tensor(counts, **i32),
              key_scales=cache.ks, value_scales=cache.vs, lse=lse, out=out, **kw)
    assert pk.status() == 0
    return out, lse


def _queries(tokens, heads, dim, dtype, seed):
    return torch.randn(tokens, heads, dim, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


GEOMETRIES = [  # q_heads, kv_heads, dim, page, lengths before the window, columns, dtype
    (8, 8, 128, 16, [0], 1, torch.bfloat16),
    (64, 8, 128, 16, [1, 15, 16, 17, 300], 1, torch.bfloat16),
    (32, 8, 128, 32, [31, 500, 64], 3, torch.float16),
    (40, 8, 128, 16, [700, 33], 6, torch.bfloat16),
    (4, 4, 128, 16, [129, 1], 2, torch.bfloat16),
    (20, 4, 128, 48, [250, 47], 5, torch.float16),
    (6, 3, 128, 16, [100, 31], 1, torch.bfloat16),
    (2, 1, 128, 16, [1030], 4, torch.bfloat16),
    (32, 16, 128, 16, [65, 200], 1, torch.bfloat16),
    (1, 1, 64, 16, [40, 0], 1, torch.float16),
    (15, 5, 64, 16, [90, 3], 2, torch.bfloat16),
    (64, 8, 64, 64, [333], 4, torch.bfloat16),
    (24, 4, 256, 64, [410, 64], 1, torch.bfloat16),
    (16, 2, 256, 16, [77], 3, torch.float16),
    (3, 1, 256, 16, [50, 15], 1, torch.bfloat16),
    (14, 2, 128, 16, [120], 64, torch.bfloat16),
]


@pytest.mark.parametrize("hq,hkv,dim,page,before,columns,dtype", GEOMETRIES)
def test_windows_of_every_geometry(hq, hkv, dim, page, before, columns, dtype):
    cache = Cache4.filled(hkv, dim, page, [n + columns for n in before], seed=11, poison=True)
    rows = list(range(len(before)))
    q = _queries(len(before) * columns, hq, dim, dtype, 12)
    starts = [r * columns for r in rows]
    for kw in ({"engine": "mma.sync"}, {"chunk": 64}, {"engine": "even"}):
        out, lse = _attend(cache, q, rows, starts, before, columns, **kw)
        _check(cache, q, out, lse, rows, starts, before, [columns] * len(rows))


def test_ragged_windows_leave_other_tokens_alone():
    before, counts = [200, 64, 0, 31], [4, 0, 2, 1]
    cache = Cache4.filled(8, 128, 16, [n + 4 for n in before], seed=21, poison=True)
    q = _queries(14, 32, 128, torch.bfloat16, 22)
    starts = [0, 4, 5, 9]
    for kw in ({"chunk": 32}, {}):
        out, lse = _attend(cache, q, range(4), starts, before, 4, counts, **kw)
        _check(cache, q, out, lse, range(4), starts, before, counts)
        named = {s + c for s, n in zip(starts, counts) for c in range(n)}
        for token in set(range(14)) - named:
            assert out[token].isnan().all() and lse[token].isnan().all()


@pytest.mark.parametrize("chunk", [None, 48])
def test_trees_sliding_windows_sinks_lists_and_context_rows(chunk):
    before, columns = [100, 37], 5
    cache = Cache4.filled(4, 128, 16, [n + columns for n in before], seed=31, poison=True)
    q = _queries(2 * columns, 12, 128, torch.bfloat16, 32)
    starts, counts = [0, columns], [columns, columns]
    parents = torch.tensor([-1, 0, 0, 1, -1] * 2, device="cuda")
    sinks = torch.linspace(-2, 3, 12, device="cuda")
    blocks = torch.tensor([[0, 2, 6, -1], [6, 1, 1, 0], [3, -1, -1, -1], [-1] * 4, [6, 5, 4, 3]] * 2, dtype=torch.int32, device="cuda")
    for masks in ({"parents": parents}, {"sliding": 20}, {"sliding": 1}, {"sinks": sinks}, {"sinks": sinks, "sliding": 33, "parents": parents},
                  {"blocks": blocks, "block_size": 16}, {"blocks": blocks, "block_size": 20}, {"context": True}):
        kw = {k: v for k, v in masks.items()}
        out, lse = _attend(cache, q, [0, 1], starts, before, columns, chunk=chunk, **kw)
        _check(cache, q, out, lse, [0, 1], starts, before, counts, **masks)


@pytest.mark.parametrize("engine", ["even", "mma.sync"])
def test_a_row_that_sees_nothing_gets_zeros(engine):
    cache = Cache4.filled(8, 128, 16, [40, 40], seed=41)
    q = _queries(4, 8, 128, torch.bfloat16, 42)
    out, lse = _attend(cache, q, [0, 1], [0, 2], [0, 30], 2, context=True, engine=engine)          # a context row with nothing before it
    assert (out[:2] == 0).all() and (lse[:2] == -float("inf")).all()
    _check(cache, q, out, lse, [1], [2], [30], [2], context=True)
    blocks = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    out, lse = _attend(cache, q, [0, 1], [0, 2], [10, 30], 2, blocks=blocks, block_size=24, engine=engine)
    assert (out == 0).all() and (lse == -float("inf")).all()


def test_a_column_has_the_same_bits_alone_in_a_window_and_in_a_batch():
    before = [300, 90, 200]
    cache = Cache4.filled(8, 128, 16, [n + 4 for n in before], seed=51)
    q = _queries(12, 64, 128, torch.bfloat16, 52)
    out, lse = _attend(cache, q, range(3), [0, 4, 8], before, 4, engine="mma.sync", chunk=128)
    for r in range(3):
        for c in range(4):
            one, one_lse = _attend(cache, q[4 * r + c:4 * r + c + 1], [r], [0], [before[r] + c], 1, engine="mma.sync", chunk=128)
            assert torch.equal(one[0], out[4 * r + c]) and torch.equal(one_lse[0], lse[4 * r + c])


def test_far_magnitudes_and_flat_long_rows():
    """Queries and rows of any magnitude; a first position far above four thousand others, whose weights are small
    numbers that still add up."""
    for scale_q, scale_kv, seed in ((1e4, 1e-3, 1), (1e-6, 3e4, 2), (30.0, 1.0, 3), (3e-3, 6e4, 4)):
        cache = Cache4.filled(2, 128, 16, [70], seed=60 + seed, scale=scale_kv)
        q = (_queries(1, 8, 128, torch.float32, 61) * scale_q).bfloat16()
        scale = 0.09 / max(scale_q * scale_kv, 1.0)
        out, lse = _attend(cache, q, [0], [0], [69], 1, scale=scale)
        _check(cache, q, out, lse, [0], [0], [69], [1], scale=scale)
    n = 4100
    cache = Cache4(1, 64, 16, n // 16 + 2)
    cache.tables = torch.arange(n // 16 + 1, dtype=torch.int32, device="cuda")[None]
    keys, values = torch.zeros(n, 1, 64), torch.ones(n, 1, 64)
    keys[0], values[0] = 1.0, 0.0
    cache.write(0, 0, keys.bfloat16().cuda(), values.bfloat16().cuda())
    q = torch.full((1, 1, 64), 0.125).bfloat16().cuda()
    for gap in (4.0, 8.0, 10.0):                                                # logits of 0 against `gap`
        out, lse = _attend(cache, q, [0], [0], [n - 1], 1, scale=gap / 8)
        _check(cache, q, out, lse, [0], [0], [n - 1], [1], scale=gap / 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("engine", ["even", "mma.sync"])
def test_rows_with_a_nan_are_not_spread(engine, dtype):
    cache = Cache4.filled(2, 128, 16, [64, 64], seed=71)
    bad = torch.full((1, 2, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    cache.write(0, 60, bad, bad)
    q = _queries(2, 8, 128, dtype, 72)
    out, lse = _attend(cache, q, [0, 1], [0, 1], [59, 63], 1, engine=engine)     # row 0 ends before the NaN
    _check(cache, q, out, lse, [0, 1], [0, 1], [59, 63], [1, 1])
    out, lse = _attend(cache, q, [0, 1], [0, 1], [63, 63], 1, engine=engine)
    assert out[0].isnan().all() and lse[0].isnan().all()
    _check(cache, q, out, lse, [1], [1], [63], [1])
    parents = torch.tensor([-1, -1], device="cuda")                              # a sibling branch holds the NaN
    out, lse = _attend(cache, _queries(2, 8, 128, dtype, 73), [0], [0], [60], 2, parents=parents, engine=engine)
    assert out[0].isnan().all() and out[1].isfinite().all()
    only_v = torch.ones(1, 2, 128, dtype=torch.bfloat16, device="cuda")          # a NaN among the values alone, in a chain's last column
    cache.write(1, 61, only_v, bad)
    q = _queries(6, 32, 128, dtype, 74)                                          # (several columns of query rows a tile)
    out, lse = _attend(cache, q, [1], [0], [56], 6, engine=engine)
    _check(cache, q, out[:5], lse[:5], [1], [0], [56], [5])
    assert out[5].isnan().all()


def test_bad_page_ids_and_plans_are_reported_and_skipped():
    cache = Cache4.filled(8, 128, 16, [100], seed=81)
    q = _queries(1, 8, 128, torch.bfloat16, 82)
    before = pk._status[str(q.device)].clone()
    cache.tables[0, 3] = 1 << 20
    i32 = dict(dtype=torch.int32, device="cuda")
    out = pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.zeros(1, **i32), torch.zeros(1, **i32),
                    torch.tensor([99], device="cuda"), 1, 16, key_scales=cache.ks, value_scales=cache.vs)
    assert out.isfinite().all() and pk.status() == 3
    pk._status[str(q.device)].copy_(before)
    slots = torch.tensor([0, 1 << 30], device="cuda")
    rows = torch.ones(2, 8, 128, dtype=torch.bfloat16, device="cuda")
    pk.write(rows, rows, slots, cache.k, cache.v, "int4", cache.ks, cache.vs)
    assert pk.status() == 3
    pk._status[str(q.device)].copy_(before)
    assert (pk.gather(cache.k, "int4", 16, slots=slots, scales=cache.ks)[1] == 0).all() and pk.status() == 3
    pk._status[str(q.device)].copy_(before)


def test_many_rows_share_the_blocks_evenly():
    """More rows than a list holds fall back to splits; rows of very different lengths, empty ones among them, in one launch."""
    g = torch.Generator().manual_seed(201)
    lengths = [int(x) for x in torch.randint(1, 90, (40,), generator=g)] + [900, 1, 16, 17]
    counts = [1] * 44
    counts[0] = counts[7] = counts[43] = 0
    cache = Cache4.filled(8, 128, 16, lengths, seed=202, poison=True)
    q = _queries(44, 16, 128, torch.bfloat16, 203)
    firsts = [n - 1 for n in lengths]
    out, lse = _attend(cache, q, range(44), range(44), firsts, 1, counts)
    _check(cache, q, out, lse, range(44), range(44), firsts, counts)
    again, _ = _attend(cache, q, range(44), range(44), firsts, 1, counts)
    assert torch.equal(out[1:7], again[1:7])
    many = 300
    q = _queries(many, 8, 128, torch.bfloat16, 204)
    rows = [r % 40 for r in range(many)]
    out, lse = _attend(cache, q, rows, range(many), [firsts[r] for r in rows], 1)
    picked = [0, 1, 150, 299]
    _check(cache, q, out, lse, [rows[r] for r in picked], picked, [firsts[rows[r]] for r in picked], [1] * 4)
    with pytest.raises(ValueError, match="no kernel"):
        _attend(cache, q, rows, range(many), [firsts[r] for r in rows], 1, engine="even")


@pytest.mark.parametrize("hq,hkv,dim,columns", [(8, 4, 256, 1), (40, 8, 128, 6), (16, 2, 128, 1)])
def test_one_long_row_over_every_block(hq, hkv, dim, columns):
    n = 9000
    cache = Cache4.filled(hkv, dim, 64, [n + columns], seed=211)
    q = _queries(columns, hq, dim, torch.bfloat16, 212)
    out, lse = _attend(cache, q, [0], [0], [n], columns)
    _check(cache, q, out, lse, [0], [0], [n], [columns])


@pytest.mark.parametrize("engine", ["even", "mma.sync"])
def test_a_captured_step_replays(engine):
    """write, then attend, captured and replayed over new lengths and new tokens, on a stream of its own."""
    cache = Cache4.filled(8, 128, 16, [50, 120], seed=91, spare=8)
    keys, values = _queries(2, 8, 128, torch.bfloat16, 92), _queries(2, 8, 128, torch.bfloat16, 93)
    q = _queries(2, 32, 128, torch.bfloat16, 94)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows, starts = torch.arange(2, **i32), torch.arange(2, **i32)
    firsts, slots = torch.tensor([50, 120], device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(2, 32, device="cuda")

    def step():
        pk.write(keys, values, slots, cache.k, cache.v, "int4", cache.ks, cache.vs)
        pk.attend(q, cache.k, cache.v, "int4", cache.tables, rows, starts, firsts, 1, 16, key_scales=cache.ks, value_scales=cache.vs,
                  out=out, lse=lse, engine=engine)
    place = lambda p: torch.cat([cache.slots(0, torch.tensor([p[0]])), cache.slots(1, torch.tensor([p[1]]))])
    slots.copy_(place([50, 120]))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i in range(3):
        at = [51 + i, 121 + i]
        keys.copy_(_queries(2, 8, 128, torch.bfloat16, 95 + i))
        slots.copy_(place(at))
        firsts.copy_(torch.tensor(at, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        _check(cache, q, out, lse, [0, 1], [0, 1], at, [1, 1])
    assert pk.status() == 0


# -- prompt chunks ----------------------------------------------------------------------------------------------------------
PROMPTS = [  # q_heads, kv_heads, dim, page, (tokens, position) a sequence, dtype
    (32, 8, 128, 16, [(70, 100)], torch.bfloat16),
    (8, 8, 128, 32, [(130, 0), (130, 33)], torch.bfloat16),
    (5, 1, 128, 16, [(17, 5), (64, 200), (1, 15)], torch.float16),
    (6, 3, 64, 16, [(40, 0), (20, 300)], torch.bfloat16),
    (8, 2, 256, 64, [(33, 65)], torch.float16),
    (4, 4, 256, 16, [(16, 31), (18, 0)], torch.bfloat16),
]


@pytest.mark.parametrize("hq,hkv,dim,page,chunks,dtype", PROMPTS)
def test_prompt_chunks(hq, hkv, dim, page, chunks, dtype):
    cache = Cache4.filled(hkv, dim, page, [c + p for c, p in chunks], seed=111, poison=True)
    tokens = sum(c for c, _ in chunks)
    q = _queries(tokens, hq, dim, dtype, 112)
    starts = [sum(c for c, _ in chunks[:i]) for i in range(len(chunks) + 1)]
    firsts = [p for _, p in chunks]

    def check(out, lse):
        # beside the output's rounding: a weight rounded to the type, and the scores' FP32 sums in weight and total (4.9e-4)
        for s, (count, position) in enumerate(chunks):
            for c in range(0, count, 7):
                at = starts[s] + c
                want, want_lse, room = attention4(cache, q[at], s, position, c, count, at)
                half = torch.finfo(dtype).eps / 2
                err = np.abs(out[at].double().cpu().numpy() - want)
                assert (err <= half * np.abs(want) + (half + 2.0 ** -10) * room + 1e-6).all(), (s, c, err.max())
                assert (np.abs(lse[at].double().cpu().numpy() - want_lse) <= 3e-4).all()
    args = (q, cache.k, cache.v, "int4")
    kw = dict(key_scales=cache.ks, value_scales=cache.vs)
    device = torch.tensor(firsts, device="cuda")
    for position in (firsts, device):
        lse = torch.full((tokens, hq), float("nan"), device="cuda")
        out = pk.prefill(*args, cache.tables, position, page, lse=lse, starts=starts, **kw)
        check(out, lse)
    for s, (count, position) in enumerate(chunks):                     # one sequence a call, the position an int or on the device
        span = slice(starts[s], starts[s + 1])
        for at in (position, device[s:s + 1]):
            lse = torch.full((tokens, hq), float("nan"), device="cuda")
            one = torch.full_like(q, float("nan"))
            pk.prefill(q[span], cache.k, cache.v, "int4", cache.tables[s], at, page, lse=lse[span], out=one[span], **kw)
            assert torch.equal(one[span], out[span]) and torch.equal(lse[span], lse[span])
    space = torch.empty(8 << 20, device="cuda")
    lse = torch.empty((tokens, hq), device="cuda")
    assert torch.equal(pk.prefill(*args, cache.tables, firsts, page, lse=lse, starts=starts, workspace=space, **kw), out)
    with pytest.raises(ValueError, match="workspace"):
        pk.prefill(*args, cache.tables, firsts, page, starts=starts, workspace=space[:100], **kw)
    with pytest.raises(ValueError, match="scales"):
        pk.prefill(*args, cache.tables, firsts, page, starts=starts, key_scales=cache.ks)
    assert pk.status() == 0


def test_a_captured_prompt_chunk_replays_over_new_positions():
    cache = Cache4.filled(8, 128, 16, [400, 300], seed=121)
    q = _queries(64, 16, 128, torch.bfloat16, 122)
    position, lse = torch.tensor([100, 30], device="cuda"), torch.empty(64, 16, device="cuda")
    out = torch.empty_like(q)
    step = lambda: pk.prefill(q, cache.k, cache.v, "int4", cache.tables, position, 16, key_scales=cache.ks, value_scales=cache.vs, out=out, lse=lse)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for at in ([368, 268], [0, 1], [17, 200]):
        position.copy_(torch.tensor(at))
        graph.replay()
        want = pk.prefill(q, cache.k, cache.v, "int4", cache.tables, at, 16, key_scales=cache.ks, value_scales=cache.vs)
        assert torch.equal(out, want), at
    assert pk.status() == 0


# -- a pool of int4 pages, as an engine drives it ---------------------------------------------------------------------------
def test_a_pool_of_int4_pages_serves_a_prompt_decode_steps_a_fork_and_an_accepted_path():
    from crit_b200.attention import DeviceAttention
    from crit_b200.batch import StepBatch
    from crit_b200.pool import KVPool
    hkv, hq, dim, page = 1, 4, 64, 16
    pool = KVPool([0, 1], hkv, dim, 600, "cuda", "int4", page=page, window=16)
    attention = DeviceAttention()
    g = torch.Generator().manual_seed(131)
    make = lambda n, h: torch.randn(n, h, dim, generator=g).bfloat16().cuda()
    told = {"a": [], "b": [], "c": []}

    def step(rows):
        batch = StepBatch.build(rows, "cuda")
        slots = pool.reserve(batch)
        for layer in (0, 1):
            keys, values, q = make(batch.tokens, hkv), make(batch.tokens, hkv), make(batch.tokens, hq)
            pool.write(layer, slots, keys, values)
            out, lse = attention.forward(layer, q, pool, batch, lse=True)
        for sequence, first, count, position in (batch.row(r) for r in range(batch.rows)):
            del told[sequence][position:]
            told[sequence] += [(keys[first + i], values[first + i]) for i in range(count)]
            pool.keep(sequence, position + count)
            # layer 1 against the rows as a plain quantisation stores them
            rows_ = [np.stack([x[j].double().cpu().numpy() for x in told[sequence]]) for j in (0, 1)]
            k, v = (values4(*quantise4(x)) for x in rows_)
            got = pool.gather(1, sequence, position + count)
            assert np.array_equal(got[0].double().cpu().numpy(), k) and np.array_equal(got[1].double().cpu().numpy(), v)
            for i in range(count):
                n = position + i + 1
                for h in range(hq):
                    s = k[:n, 0] @ q[first + i, h].double().cpu().numpy() * dim ** -0.5
                    w = np.exp(s - s.max())
                    want = w @ v[:n, 0] / w.sum()
                    room = w @ np.abs(v[:n, 0]) / w.sum()
                    err = np.abs(out[first + i, h].double().cpu().numpy() - want)
                    assert (err <= 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -9) * room + n * 2.0 ** -20).all()
                    assert abs(float(lse[first + i, h]) - s.max() - np.log(w.sum())) <= 3e-4
    for sequence in ("a", "b"):
        pool.open(sequence)
    step([("a", 0, 45), ("b", 0, 20)])
    step([("a", 45, 1), ("b", 20, 3)])
    pool.fork("a", "c")
    told["c"] = list(told["a"])
    step([("a", 46, 1), ("c", 46, 1), ("b", 23, 1)])
    step([("b", 24, 40), ("a", 47, 2)])
    assert pk.status() == 0
    # an accepted draft path: rows of two bytes of scales a slot move one by one
    source, target = pool.slots_at(torch.zeros(1, 1, dtype=torch.long).cuda(), torch.zeros(1, 1, dtype=torch.long).cuda()), None
    table = pool.table("a")
    source = torch.tensor([[table[0] * page + 5, table[1] * page + 3]], device="cuda")
    target = torch.tensor([[table[0] * page + 2, table[0] * page + 3]], device="cuda")
    before = pool.rows_at(1, source)
    for store in (pool.k, pool.v, pool.k_scales, pool.v_scales):
        pk.move_rows(store.view(2, pool.stored_slots, -1), source, target)
    after = pool.rows_at(1, target)
    assert all(torch.equal(x, y) for x, y in zip(before, after)) and pk.status() == 0


# -- refusals ---------------------------------------------------------------------------------------------------------------
def test_what_the_entry_points_refuse():
    cache = Cache4.filled(8, 128, 16, [40], seed=101)
    rows, slots = _queries(3, 8, 128, torch.bfloat16, 102), torch.arange(3).cuda()
    ok = [rows, rows, slots, cache.k, cache.v, "int4", cache.ks, cache.vs]

    def refuse(changes, error=ValueError, match=None):
        args = list(ok)
        for i, x in changes.items():
            args[i] = x
        with pytest.raises(error, match=match):
            pk.write(*args)
    refuse({6: None}, match="take scales")
    refuse({7: None}, match="scales beside them")
    refuse({3: cache.k.view(torch.int8)}, match="uint8")
    refuse({6: cache.ks.half()}, match="uint8")
    refuse({6: cache.ks[:, :8].contiguous()}, match="scales")
    refuse({0: rows[..., :64]}, match="go to pages")
    refuse({1: rows[:2]}, match="go to pages")
    refuse({2: slots.int()}, match="int64")
    refuse({2: slots.cpu()}, match="device")
    refuse({3: cache.k.cpu(), 6: cache.ks.cpu()}, match="device")
    refuse({0: rows.cpu()}, RuntimeError, match="CUDA devices only")
    with pytest.raises(ValueError, match="uint8"):
        pk.gather(cache.k.view(torch.int8), "int4", 16, slots=slots, scales=cache.ks)
    with pytest.raises(ValueError, match="take scales"):
        pk.gather(cache.k, "int4", 16, slots=slots)
    with pytest.raises(ValueError, match="device"):
        pk.gather(cache.k, "int4", 16, slots=slots.cpu(), scales=cache.ks)
    with pytest.raises(ValueError, match="device"):
        _attend_with(cache, _queries(1, 32, 128, torch.bfloat16, 103), counts=torch.ones(1, dtype=torch.int32))
    for out in (torch.empty(2, 8, 128, device="cuda"), torch.empty(3, 8, 128), torch.empty(3, 128, 8, device="cuda").transpose(1, 2),
                torch.empty(3, 8, 128, dtype=torch.float64, device="cuda")):
        with pytest.raises(ValueError, match="out is a contiguous"):
            pk.gather(cache.k, "int4", 16, slots=slots, scales=cache.ks, out=out)
    q = _queries(1, 32, 128, torch.bfloat16, 103)
    with pytest.raises(ValueError, match="alike"):
        _attend_with(cache, q, value_scales=None)
    with pytest.raises(ValueError, match="q's width"):
        _attend_with(cache, q[..., :64].contiguous())
    with pytest.raises(ValueError, match="uint8"):
        _attend_with(cache, q, key_scales=cache.ks.float())
    with pytest.raises(ValueError):
        _attend_with(cache, q.float())
    with pytest.raises(ValueError, match="workspace"):
        _attend_with(cache, q, engine="even", workspace=torch.empty(100, device="cuda"))
    with pytest.raises(NotImplementedError, match="int4"):
        pages = torch.zeros(4, 16, 8, 128, dtype=torch.bfloat16, device="cuda")
        i32 = torch.zeros(1, dtype=torch.int32, device="cuda")
        pk.attend(q, pages, pages, "bf16", cache.tables, i32, i32, torch.tensor([5], device="cuda"), 1, 16, engine="even")
    for engine in ("tcgen05", "tcgen05p", "tcgen05t"):
        with pytest.raises(ValueError, match="no kernel"):
            _attend_with(cache, q, engine=engine)
    narrow = Cache4(8, 96, 16, 4)
    narrow.tables = cache.tables
    with pytest.raises(ValueError, match="no kernel"):
        _attend_with(narrow, _queries(1, 8, 96, torch.bfloat16, 104))
    assert pk.status() == 0


def _attend_with(cache, q, **kw):
    i32 = dict(dtype=torch.int32, device="cuda")
    kw = {"key_scales": cache.ks, "value_scales": cache.vs, **kw}
    return pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.zeros(1, **i32), torch.zeros(1, **i32),
                     torch.tensor([5], device="cuda"), 1, 16, **kw)


# -- at the borders of what a call says -------------------------------------------------------------------------------------
@pytest.mark.parametrize("engine", [None, "mma.sync"])
def test_a_row_of_more_positions_than_its_table_is_reported_and_left_out(engine):
    """Two rows, one of which says more positions than a table row holds: the other one is as it should be."""
    cache = Cache4.filled(8, 128, 16, [100, 70], seed=221)
    q = _queries(2, 32, 128, torch.bfloat16, 222)
    before = pk._status[str(q.device)].clone()
    out, lse = torch.full_like(q, float("nan")), torch.full((2, 32), float("nan"), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    if engine is None:                   # (launches cut into splits end with their grid)
        firsts = torch.tensor([99, 1 << 40], device="cuda")
        pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.arange(2, **i32), torch.arange(2, **i32), firsts, 1, 16, key_scales=cache.ks,
                  value_scales=cache.vs, out=out, lse=lse)
        assert pk.status() == 2 and out[1].isnan().all() and lse[1].isnan().all()
        pk._status[str(q.device)].copy_(before)
    else:
        out[:1], lse[:1] = _attend(cache, q[:1], [0], [0], [99], 1, engine=engine)
    _check(cache, q, out[:1], lse[:1], [0], [0], [99], [1])
    assert pk.status() == int(before)


@pytest.mark.parametrize("hq,hkv,dim,engine", [(32, 8, 128, None), (32, 8, 128, "mma.sync"), (32, 8, 128, "tcgen05:single"), (32, 8, 128, "tcgen05:pair"),
                                               (8, 2, 64, None), (8, 2, 256, None)])
def test_what_lies_in_a_prompts_workspace_does_not_matter(hq, hkv, dim, engine):
    """NaN everywhere in the workspace, and in the pages behind the sequences' ends, against zeros."""
    cache = Cache4.filled(hkv, dim, 16, [75, 33], seed=231, poison=True)
    q = _queries(45, hq, dim, torch.bfloat16, 232)
    found = []
    for fill in (0.0, float("nan")):
        space, lse = torch.full((4 << 20,), fill, device="cuda"), torch.empty(45, hq, device="cuda")
        found.append((pk.prefill(q, cache.k, cache.v, "int4", cache.tables, [45, 18], 16, key_scales=cache.ks, value_scales=cache.vs, starts=[0, 30, 45],
                                 workspace=space, lse=lse, engine=engine), lse))
    assert found[0][0].isfinite().all() and torch.equal(found[0][0], found[1][0]) and torch.equal(found[0][1], found[1][1])
    nothing = pk.prefill(q[:0], cache.k, cache.v, "int4", cache.tables[0], 0, 16, key_scales=cache.ks, value_scales=cache.vs)
    assert nothing.shape == (0, hq, dim) and pk.status() == 0


def test_two_streams_at_once_with_a_workspace_each():
    """Steps of two owners on two streams, eager and as graphs, interleaved: each as alone."""
    caches = [Cache4.filled(8, 128, 16, [3000, 500], seed=241), Cache4.filled(8, 128, 16, [1200], seed=242)]
    queries = [_queries(2, 32, 128, torch.bfloat16, 243), _queries(6, 40, 128, torch.float16, 244)]
    i32 = dict(dtype=torch.int32, device="cuda")
    firsts = [torch.tensor([2999, 499], device="cuda"), torch.tensor([1194], device="cuda")]
    rows = [torch.arange(2, **i32), torch.zeros(1, **i32)]
    outs = [torch.empty_like(q) for q in queries]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def step(i, out):
        c = caches[i]
        pk.attend(queries[i], c.k, c.v, "int4", c.tables, rows[i], rows[i], firsts[i], 1 if i == 0 else 6, 16, key_scales=c.ks, value_scales=c.vs, out=out)
        pk.prefill(queries[i][:1], c.k, c.v, "int4", c.tables[0], firsts[i][:1], 16, key_scales=c.ks, value_scales=c.vs)
    want = [torch.empty_like(q) for q in queries]
    for i in (0, 1):
        step(i, want[i])
    torch.cuda.synchronize()
    graphs = []
    for i in (0, 1):
        with pk.owner(("stream", i)):
            with torch.cuda.stream(streams[i]):
                step(i, outs[i])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[i]):
                step(i, outs[i])
            graphs.append(graph)
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]), pk.owner(("stream", i)):
                graphs[i].replay()
                step(i, outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and pk.status() == 0
    del graphs
    for i in (0, 1):
        pk.release(("stream", i))


def test_pages_as_any_view_of_their_storage():
    """Pages of the other kinds given flat, which the slots' bound is counted from."""
    keys = _queries(5, 4, 128, torch.bfloat16, 251)
    slots = torch.tensor([0, 31, 16, 5, 63]).cuda()
    for kind, store in (("bf16", torch.bfloat16), ("fp8", torch.float8_e4m3fn)):
        shaped, flat = (torch.zeros(64, 4, 128, dtype=store, device="cuda") for _ in range(2))
        pk.write(keys, None, slots, shaped, None, kind)
        pk.write(keys, None, slots, flat.view(64, -1), None, kind)
        assert torch.equal(shaped.view(torch.uint8), flat.view(torch.uint8)) and shaped.view(torch.uint8).any()
    assert pk.status() == 0


def test_lists_are_kept_by_a_capture_and_short_tables_refused():
    cache = Cache4.filled(8, 128, 16, [64, 64], seed=261)
    q = _queries(10, 8, 128, torch.bfloat16, 262)
    args, kw = (q, cache.k, cache.v, "int4", cache.tables), dict(key_scales=cache.ks, value_scales=cache.vs)
    want = pk.prefill(*args, [3, 40], 16, starts=[0, 4, 10], **kw)
    out, graph, firsts = torch.empty_like(q), torch.cuda.CUDAGraph(), [3, 40]
    with torch.cuda.graph(graph):
        pk.prefill(*args, firsts, 16, starts=[0, 4, 10], out=out, **kw)
    firsts[0] = 9
    other = [torch.full((64,), -1, device="cuda") for _ in range(8)]       # (memory that a freed list would have been given to)
    for _ in range(2):
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, want)
    del other
    assert torch.equal(pk.prefill(*args, torch.tensor([3, 40], device="cuda"), 16, starts=[0, 4, 10], **kw), want)
    assert torch.equal(pk.prefill(q[:8], *args[1:], [3, 40], 16, **kw),                # equal counts: no starts
                       pk.prefill(q[:8], *args[1:], [3, 40], 16, starts=[0, 4, 8], **kw))
    with pytest.raises(ValueError, match="page table"):
        pk.prefill(*args, [3, 1 << 30], 16, starts=[0, 4, 10], **kw)
    with pytest.raises(ValueError, match="page table"):
        pk.gather(cache.k, "int4", 16, table=cache.tables[0], count=cache.tables.shape[1] * 16 + 1, scales=cache.ks)
    with pytest.raises(ValueError, match="page table"):
        pk.gather(cache.k, "int4", 16, table=cache.tables[0].long(), count=4, scales=cache.ks)
    with pytest.raises(ValueError, match="int64 slots"):
        pk.gather(cache.k, "int4", 16, slots=torch.zeros(4, dtype=torch.int32, device="cuda"), scales=cache.ks)
    assert pk.status() == 0


@pytest.mark.parametrize("columns,chunk", [(1, 64), (6, 128), (3, 1024)])
def test_states_that_stay_in_the_workspace_fold_to_the_same_bits(columns, chunk, monkeypatch):
    """The flag a sharded context's launches carry: every row's states kept, a row of one split too, and folded by the merge."""
    import ctypes
    from crit_b200 import _lib
    cache = Cache4.filled(8, 128, 16, [700 + columns, 40 + columns], seed=271)
    q, space = _queries(2 * columns, 32, 128, torch.bfloat16, 272), torch.full((1 << 21,), float("nan"), device="cuda")
    blocks, run = [], pk._run
    monkeypatch.setattr(pk, "_run", lambda name, what, device, *params: (blocks.extend(params), run(name, what, device, *params)))
    want, want_lse = _attend(cache, q, [0, 1], [0, columns], [700, 40], columns, chunk=chunk, engine="mma.sync", workspace=space)
    out, lse, p = torch.full_like(q, float("nan")), torch.full((2 * columns, 32), float("nan"), device="cuda"), blocks[-1]
    tensors = [torch.tensor(x, dtype=t, device="cuda") for x, t in (([0, 1], torch.int32), ([0, columns], torch.int32), ([700, 40], torch.int64))]
    p.rows, p.starts, p.firsts, p.counts = [x.data_ptr() for x in tensors] + [0]
    p.out, p.lse, p.workspace, p.workspace_floats, p.flags = out.data_ptr(), lse.data_ptr(), space.data_ptr(), space.numel(), p.flags | 32
    stream, lib = torch.cuda.current_stream().cuda_stream, _lib.load()
    assert lib.crit_b200_decode(ctypes.byref(p), stream) == 0
    assert out.isnan().all() and lse.isnan().all()
    assert lib.crit_b200_merge(ctypes.byref(p), stream) == 0
    if chunk < 700:
        assert torch.equal(out[:columns], want[:columns])                  # a row of several splits: the same states, the same fold
    # (a row of one split is divided by its sum in the fold instead: two FP32 roundings apart, one step of bf16 at most)
    assert ((out.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs()).all()
    assert (lse - want_lse).abs().max() <= 1e-5 and pk.status() == 0
