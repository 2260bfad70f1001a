"""norm_rope and norm_rope_write on a GPU against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

import crit_b200 as pk
from int4_oracle import Cache4

pytestmark = pytest.mark.gpu


def rotated(x, weight, positions, frequencies, eps=1e-6, offset=0.0, axes=None, interleaved=False, magnitude=1.0):
    """([tokens][heads][dim] in 64 bits, the sum of the magnitudes each result is made of)."""
    y = x.double().cpu().numpy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (offset + weight.double().cpu().numpy())
    f = frequencies.double().cpu().numpy()
    half = len(f)
    p = positions.double().cpu().numpy()
    at = p[:, None] if p.ndim == 1 else p[axes.cpu().numpy()].T
    angle = (at * f)[:, None]
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
    out, room = y.copy(), np.abs(y)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    room[..., a] = room[..., b] = (np.abs(y[..., a]) + np.abs(y[..., b])) * abs(magnitude)
    return out, room


def close(got, want, room, dtype):
    """FP32 work: the sum of squares (8 in a lane, up to 5 between lanes, halved by the root), root, quotient, mean and two
    weights, cosine and sine (2^-22 of a turn's part and two units), the pair's products and sum: below 24 * 2^-24 of the magnitudes;
    then one rounding to the type."""
    half = torch.finfo(dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    tol = 24 * 2.0 ** -24 * room + half * np.abs(want) * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    assert np.isfinite(err).all() and (err <= tol).all(), np.max(err / tol)


def inputs(tokens, hq, hkv, dim, rotary, dtype, seed, axes=1, far=5000):
    g = torch.Generator().manual_seed(seed)
    q, keys = (torch.randn(tokens, h, dim, generator=g).to(dtype).cuda() for h in (hq, hkv))
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2))
    half = rotary // 2
    frequencies = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
    positions = torch.randint(0, far, (tokens,) if axes == 1 else (axes, tokens), generator=g).cuda()
    return q, keys, qw, kw, positions, frequencies


CASES = [  # tokens, q_heads, kv_heads, dim, rotary, dtype
    (1, 1, 1, 64, 64, torch.bfloat16),
    (3, 5, 1, 32, 32, torch.float32),
    (7, 32, 8, 128, 128, torch.bfloat16),
    (33, 64, 8, 128, 64, torch.float16),
    (17, 6, 3, 96, 96, torch.bfloat16),
    (5, 24, 4, 256, 64, torch.bfloat16),
    (130, 2, 2, 64, 32, torch.float32),
    (9, 3, 1, 160, 40, torch.float16),
    (2, 1, 1, 224, 8, torch.float32),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rotary,dtype", CASES)
def test_norm_and_rotation(tokens, hq, hkv, dim, rotary, dtype, interleaved):
    q, keys, qw, kw, positions, frequencies = inputs(tokens, hq, hkv, dim, rotary, dtype, 1)
    for norm in (dict(q_weight=qw, key_weight=kw), dict(q_weight=qw, key_weight=None), dict(q_weight=qw.float(), key_weight=kw.float(), offset=1.0, eps=1e-5, magnitude=1.3), {}):
        got = pk.norm_rope(q, keys, positions, frequencies, interleaved=interleaved, **norm)
        rest = {k: v for k, v in norm.items() if not k.endswith("weight")}
        for x, out, weight in ((q, got[0], norm.get("q_weight")), (keys, got[1], norm.get("key_weight"))):
            close(out, *rotated(x, weight, positions, frequencies, interleaved=interleaved, **rest), dtype)
    only_q, none = pk.norm_rope(q, None, positions, frequencies, q_weight=qw, interleaved=interleaved)
    none_q, only_k = pk.norm_rope(None, keys, positions, frequencies, key_weight=kw, interleaved=interleaved)
    both = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw, interleaved=interleaved)
    assert none is None and none_q is None and torch.equal(only_q, both[0]) and torch.equal(only_k, both[1])
    a, b = q.clone(), keys.clone()                                              # in place
    same = pk.norm_rope(a, b, positions, frequencies, q_weight=qw, key_weight=kw, interleaved=interleaved, q_out=a, keys_out=b)
    assert same[0] is a and same[1] is b and torch.equal(a, both[0]) and torch.equal(b, both[1])
    assert pk.status() == 0


@pytest.mark.parametrize("order", [False, True])
def test_positions_of_several_axes(order):
    q, keys, qw, kw, positions, frequencies = inputs(11, 8, 2, 128, 128, torch.bfloat16, 2, axes=3)
    axes = pk.rope_axes([16, 24, 24], order)
    got = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw, axes=axes)
    close(got[0], *rotated(q, qw, positions, frequencies, axes=axes), q.dtype)
    close(got[1], *rotated(keys, kw, positions, frequencies, axes=axes), q.dtype)
    # text: the axes agree, and so does the form of one axis
    same = positions[:1].expand(3, -1).contiguous()
    text = pk.norm_rope(q, keys, same, frequencies, q_weight=qw, key_weight=kw, axes=axes)
    one = pk.norm_rope(q, keys, positions[0], frequencies, q_weight=qw, key_weight=kw)
    assert torch.equal(text[0], one[0]) and torch.equal(text[1], one[1])
    before = pk._status[str(q.device)].clone()
    pk.norm_rope(q, keys, positions, frequencies, axes=torch.full_like(axes, 3))
    assert pk.status() == 3                                                     # an axis that is not there: reported
    pk._status[str(q.device)].copy_(before)


def test_far_positions_and_odd_rows():
    q, keys, qw, kw, positions, frequencies = inputs(8, 4, 1, 128, 128, torch.float32, 3)
    positions = torch.tensor([0, 1, -5, 1 << 20, (1 << 31) - 1, 123456789, 1 << 35, 7], device="cuda")
    q[3] = 0
    q[4] *= 1e-12
    q[5] *= 1e15
    got = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw)
    close(got[0], *rotated(q, qw, positions, frequencies), q.dtype)
    close(got[1], *rotated(keys, kw, positions, frequencies), q.dtype)
    q[1, 2, 3] = float("nan")
    got = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw)[0]
    assert got[1, 2].isnan().all() and got[1, 1].isfinite().all() and got[0].isfinite().all()


def test_strided_and_unaligned_rows():
    q, keys, qw, kw, positions, frequencies = inputs(13, 4, 2, 64, 64, torch.bfloat16, 4)
    want = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw)
    packed = torch.cat([q, keys, keys], 1).flatten(1)                           # a packed projection, views of its heads
    views = packed[:, :256].unflatten(1, (4, 64)), packed[:, 256:384].unflatten(1, (2, 64))
    odd = torch.zeros(13, 4 * 64 + 3, dtype=q.dtype, device="cuda")
    odd[:, 1:257] = q.flatten(1)
    for a, b in (views, (odd[:, 1:257].unflatten(1, (4, 64)), keys.transpose(0, 1).contiguous().transpose(0, 1)),
                 (q.transpose(1, 2).contiguous().transpose(1, 2), keys)):
        got = pk.norm_rope(a, b, positions, frequencies, q_weight=qw, key_weight=kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = torch.zeros(13, 4 * 64 + 3, dtype=q.dtype, device="cuda")
    pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw, q_out=out[:, 1:257].unflatten(1, (4, 64)), keys_out=views[1])
    assert torch.equal(out[:, 1:257].unflatten(1, (4, 64)), want[0]) and torch.equal(views[1], want[1]) and not out[:, 0].any() and not out[:, 257:].any()
    empty = pk.norm_rope(q[:0], keys[:0], positions[:0], frequencies)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 2, 64)


STORE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn, "fp8:row": torch.float8_e4m3fn, "int8": torch.int8,
         "fp8:page": torch.float8_e4m3fn}


def pages_of(kind, heads, dim, value_dim, n, page=16):
    if kind == "int4":
        a, b = Cache4(heads, dim, page, n), Cache4(heads, value_dim, page, n)
        return [a.k, b.v, a.ks, b.vs]
    made = [torch.zeros(n, page, heads, w, dtype=STORE[kind], device="cuda") for w in (dim, value_dim)]
    shape = {"fp8:row": (n, page, heads), "int8": (n, page, heads), "fp8:page": (n, heads)}.get(kind)
    return made + [torch.zeros(shape, device="cuda") if shape else None for _ in range(2)]


@pytest.mark.parametrize("kind", ["int4", "bf16", "fp16", "fp8", "fp8:row", "int8", "fp8:page"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,value_dim,dtype", [(1, 8, 8, 128, 128, torch.bfloat16), (70, 32, 8, 128, 128, torch.bfloat16), (21, 3, 3, 64, 64, torch.float16),
                                                               (19, 4, 1, 96, 64, torch.bfloat16), (9, 8, 2, 256, 128, torch.float32), (12, 2, 1, 64, 256, torch.bfloat16)])
def test_rows_go_to_their_pages_in_the_same_pass(kind, tokens, hq, hkv, dim, value_dim, dtype):
    q, keys, qw, kw, positions, frequencies = inputs(tokens, hq, hkv, dim, min(dim, 64), dtype, 5)
    values = (3 * torch.randn(tokens, hkv, value_dim, generator=torch.Generator().manual_seed(6))).to(dtype).cuda()
    n = tokens // 16 + 3
    slots = torch.randperm(n * 16, generator=torch.Generator().manual_seed(7))[:tokens].cuda()
    if kind == "fp8:page":
        slots = torch.arange(tokens).cuda()
    if tokens > 5:
        slots[3] = -1
    rotation = dict(q_weight=qw, key_weight=kw)
    got, want = pages_of(kind, hkv, dim, value_dim, n), pages_of(kind, hkv, dim, value_dim, n)
    mult = (0.02, 0.05)
    turned = torch.empty_like(keys)
    out = pk.norm_rope_write(q, keys, values, positions, frequencies, slots, got[0], got[1], kind, got[2], got[3], multipliers=mult, keys_out=turned, **rotation)
    q_want, keys_want = pk.norm_rope(q, keys, positions, frequencies, **rotation)
    assert torch.equal(out, q_want) and torch.equal(turned, keys_want)
    # the same rows in two steps: the keys in FP32 between them (rounded to their type for fp8:page)
    between = keys_want if kind == "fp8:page" else pk.norm_rope(None, keys.float(), positions, frequencies, key_weight=kw)[1]
    pk.write(between, None, slots, want[0], None, kind, want[2], None, multipliers=mult)
    pk.write(None, values, slots, None, want[1], kind, None, want[3], multipliers=mult)
    for a, b in zip(got, want):
        if a is not None:
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), kind
    # keys alone, and no keys_out
    again = pages_of(kind, hkv, dim, value_dim, n)
    pk.norm_rope_write(q, keys, None, positions, frequencies, slots, again[0], None, kind, again[2], None, multipliers=mult, **rotation)
    assert torch.equal(again[0].view(torch.uint8), got[0].view(torch.uint8)) and not again[1].view(torch.uint8).any()
    assert pk.status() == 0


def test_the_steps_of_a_layer_captured_together():
    """norm_rope_write into int4 pages, then the attention that reads them: the run of a decode step, replayed."""
    cache = Cache4.filled(8, 128, 16, [60, 30], seed=141, spare=8)
    q, keys, qw, kw, positions, frequencies = inputs(2, 32, 8, 128, 128, torch.bfloat16, 8)
    values = torch.randn_like(keys)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = torch.arange(2, **i32)
    slots, out, lse = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.empty_like(q), torch.empty(2, 32, device="cuda")

    def step():
        turned = pk.norm_rope_write(q, keys, values, positions, frequencies, slots, cache.k, cache.v, "int4", cache.ks, cache.vs, q_weight=qw, key_weight=kw)
        pk.attend(turned, cache.k, cache.v, "int4", cache.tables, rows, rows, positions, 1, 16, key_scales=cache.ks, value_scales=cache.vs, out=out, lse=lse)
    place = lambda at: torch.cat([cache.slots(0, torch.tensor([at[0]])), cache.slots(1, torch.tensor([at[1]]))])
    positions.copy_(torch.tensor([60, 30]))
    slots.copy_(place([60, 30]))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    from int4_oracle import attention4, bounds4
    for i in range(3):
        at = [61 + i, 31 + i]
        positions.copy_(torch.tensor(at))
        slots.copy_(place(at))
        keys.normal_()
        graph.replay()
        turned, _ = pk.norm_rope(q, None, positions, frequencies, q_weight=qw)
        for r in (0, 1):
            want, want_lse, room = attention4(cache, turned[r], r, at[r], 0, 1, r)
            assert (np.abs(out[r].double().cpu().numpy() - want) <= bounds4(want, room, at[r] + 1, q.dtype)).all()
            assert (np.abs(lse[r].double().cpu().numpy() - want_lse) <= 3e-4).all()
    assert pk.status() == 0


def test_a_pool_takes_the_fused_step_and_keeps_a_prompts_rows_fresh():
    from crit_b200.attention import DeviceAttention
    from crit_b200.batch import StepBatch
    from crit_b200.pool import FreshBuffer, KVPool
    q, keys, qw, kw, positions, frequencies = inputs(40, 8, 2, 64, 64, torch.bfloat16, 9)
    values = torch.randn_like(keys)
    positions = torch.arange(40, device="cuda")
    found = []
    for fused in (True, False):
        pool = KVPool([0], 2, 64, 256, "cuda", "int4", window=16, fresh=FreshBuffer(torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")))
        pool.open("a")
        batch = StepBatch.build([("a", 0, 40)], "cuda")
        slots = pool.reserve(batch)
        if fused:
            turned = pool.norm_rope_write(0, slots, q, keys, values, positions, frequencies, q_weight=qw, key_weight=kw)
        else:
            turned, k = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw)
            pool.write(0, slots, k, values)
        fresh = pool.fresh_rows(0, 40)
        assert fresh is not None
        found.append((turned, fresh[0].clone(), fresh[1].clone(), DeviceAttention().forward(0, turned, pool, batch), *pool.gather(0, "a", 40)))
    for a, b in zip(found[0][:4], found[1][:4]):
        assert torch.equal(a, b)
    # The values' pages are the same.  A key went to its page with or without its rounding to bf16 (2^-8 of the largest of
    # its group at most); either code is within half a scale of what it was made of, and a scale within 17/16 of max / 7.
    assert torch.equal(found[0][5], found[1][5])
    a, b, exact = (x.double().unflatten(-1, (-1, 32)) for x in (found[0][4], found[1][4], found[0][1]))
    top = exact.abs().amax(-1, keepdim=True) * (1 + 2.0 ** -8)
    assert ((a - b).abs() <= top * (17 / 16 / 7 + 2.0 ** -8)).all() and (a != b).any()


def test_what_the_entry_points_refuse():
    q, keys, qw, kw, positions, frequencies = inputs(3, 4, 2, 64, 64, torch.bfloat16, 10)
    bad = [((None, None), {}, "takes q"), ((q, keys[:2]), {}, "one dtype"), ((q, keys.half()), {}, "one dtype"), ((q.double(), None), {}, "one dtype"),
           ((q, keys), {"positions": positions.int()}, "int64"), ((q, keys), {"positions": positions[:2]}, "int64"),
           ((q, keys), {"positions": positions.expand(2, 3)}, "several axes"), ((q, keys), {"frequencies": frequencies.double()}, "FP32"),
           ((q, keys), {"frequencies": frequencies.cpu()}, "FP32"), ((q, keys), {"axes": frequencies.long()}, "int32"),
           ((q, keys), {"q_weight": qw[:32]}, "contiguous"), ((q, keys), {"q_weight": qw, "key_weight": kw.float()}, "one bf16"),
           ((q, keys), {"q_out": q[:2]}, "shape"), ((q, keys), {"keys_out": keys.float()}, "shape"), ((q, None), {"keys_out": keys}, "no keys"), ((q[0], None), {}, "heads"),
           ((q, keys), {"frequencies": frequencies[:30].contiguous()}, "no kernel"), ((q, keys), {"frequencies": frequencies.repeat(2)}, "no kernel"),
           ((q[..., :40].contiguous(), None), {"frequencies": frequencies[:16].contiguous()}, "no kernel")]
    for (a, b), change, match in bad:
        kw_ = {"positions": positions, "frequencies": frequencies, **change}
        with pytest.raises(ValueError, match=match):
            pk.norm_rope(a, b, kw_.pop("positions"), kw_.pop("frequencies"), **kw_)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        pk.norm_rope(q.cpu(), keys.cpu(), positions.cpu(), frequencies.cpu())
    cache = Cache4(2, 64, 16, 2)
    with pytest.raises(ValueError, match="pass keys"):
        pk.norm_rope_write(q, None, keys, positions, frequencies, torch.arange(3).cuda(), cache.k, cache.v, "int4", cache.ks, cache.vs)
    with pytest.raises(ValueError, match="go to pages"):
        pk.norm_rope_write(q, keys, keys[..., :32], positions, frequencies, torch.arange(3).cuda(), cache.k, cache.v, "int4", cache.ks, cache.vs)
    with pytest.raises(ValueError, match="sections"):
        pk.rope_axes([])
    before = pk._status[str(q.device)].clone()
    pk.norm_rope_write(q, keys, keys, positions, frequencies, torch.tensor([0, 1 << 40, 5]).cuda(), cache.k, cache.v, "int4", cache.ks, cache.vs)
    assert pk.status() == 3
    pk._status[str(q.device)].copy_(before)


def test_a_refused_step_leaves_the_queries_as_they_were():
    q, keys, qw, kw, positions, frequencies = inputs(3, 4, 2, 64, 64, torch.bfloat16, 10)
    cache, slots, kept = Cache4(2, 64, 16, 2), torch.arange(3).cuda(), q.clone()
    pages, scales = torch.zeros(2, 16, 2, 64, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(2, 2, device="cuda")
    values = keys.clone()
    int4, fp8 = (cache.k, cache.v, "int4", cache.ks, cache.vs), (pages, pages.clone(), "fp8:page", scales, scales.clone())
    for store, change, match in ((int4, {"values": values[:2]}, "a row a token"), (int4, {"values": values[:, :1]}, "a row a token"),
                                 (int4, {"keys_out": values}, "values' place"), (int4, {"slots": slots[:2]}, "slots"), (fp8, {"slots": slots[:2]}, "slots"),
                                 (fp8, {"slots": slots.int()}, "slots"), (int4, {"slots": slots.cpu()}, "slots")):
        call = {"values": values, "slots": slots, "keys_out": None, **change}
        with pytest.raises(ValueError, match=match):
            pk.norm_rope_write(q, keys, call["values"], positions, frequencies, call["slots"], *store, q_weight=qw, key_weight=kw, q_out=q, keys_out=call["keys_out"])
        assert torch.equal(q, kept)
    # no tokens: nothing is launched, whatever the pages hold
    none = pk.norm_rope_write(q[:0], keys[:0], values[:0], positions[:0], frequencies, slots[:0], *int4)
    assert none.shape == (0, 4, 64) and not cache.k.any() and pk.status() == 0
