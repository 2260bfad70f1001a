"""norm_rope and norm_rope_write: calls at the borders of what their arguments say."""
import pytest
import torch

import crit_b200 as pk
from test_norm_rope_gpu import inputs, pages_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["int4", "bf16", "fp8:row", "fp8:page"])
def test_keys_and_values_without_queries(kind):
    q, keys, qw, kw, positions, frequencies = inputs(9, 4, 2, 64, 64, torch.bfloat16, 1)
    values, slots = torch.randn_like(keys), torch.arange(9).cuda()
    found = []
    for queries in (q, None):
        at, turned = pages_of(kind, 2, 64, 64, 2), torch.empty_like(keys)
        got = pk.norm_rope_write(queries, keys, values, positions, frequencies, slots, at[0], at[1], kind, at[2], at[3], q_weight=qw, key_weight=kw,
                                 keys_out=turned)
        assert (got is None) == (queries is None)
        found.append([x.view(torch.uint8) for x in (*at, turned) if x is not None])
    assert all(torch.equal(a, b) for a, b in zip(*found)) and found[0][0].any() and pk.status() == 0
    with pytest.raises(ValueError, match="no q"):
        pk.norm_rope_write(None, keys, values, positions, frequencies, slots, at[0], at[1], kind, at[2], at[3], q_out=q)
    with pytest.raises(ValueError, match="pass keys"):
        pk.norm_rope_write(None, None, values, positions, frequencies, slots, at[0], at[1], kind, at[2], at[3])


@pytest.mark.parametrize("kind", ["int4", "bf16", "fp8", "fp8:row", "int8", "fp8:page"])
def test_tensors_on_another_device_are_refused(kind):
    q, keys, qw, kw, positions, frequencies = inputs(3, 4, 2, 64, 64, torch.bfloat16, 2)
    kept, values, slots, at = q.clone(), torch.randn_like(keys), torch.arange(3).cuda(), pages_of(kind, 2, 64, 64, 2)
    for i in range(5):
        store, rows = list(at), values
        if i == 4:
            rows = values.cpu()
        elif store[i] is None:
            continue
        else:
            store[i] = store[i].cpu()
        with pytest.raises(ValueError):
            pk.norm_rope_write(q, keys, rows, positions, frequencies, slots, store[0], store[1], kind, store[2], store[3], q_out=q)
        with pytest.raises(ValueError):
            pk.write(keys, rows, slots, store[0], store[1], kind, store[2], store[3])
    assert torch.equal(q, kept) and pk.status() == 0


def test_values_of_fewer_pages_bound_the_slots():
    q, keys, qw, kw, positions, frequencies = inputs(2, 4, 2, 64, 64, torch.bfloat16, 3)
    before = pk._status[str(q.device)].clone()
    for kind in ("int4", "bf16"):
        k, _, ks, _ = pages_of(kind, 2, 64, 64, 6)
        _, v, _, vs = pages_of(kind, 2, 64, 64, 4)
        slots = torch.tensor([5, 70], device="cuda")                       # the keys' pages hold 96 slots, the values' 64
        for write in (lambda: pk.write(keys, keys, slots, k, v, kind, ks, vs),
                      lambda: pk.norm_rope_write(q, keys, keys, positions, frequencies, slots, k, v, kind, ks, vs)):
            write()
            assert pk.status() == 3
            pk._status[str(q.device)].copy_(before)
            assert k.view(torch.uint8).flatten(0, 1)[5].any() and not k.view(torch.uint8).flatten(0, 1)[70].any()


def test_outputs_that_meet_their_inputs_in_memory():
    q, keys, qw, kw, positions, frequencies = inputs(40, 4, 4, 64, 64, torch.bfloat16, 4)
    norm = dict(q_weight=qw, key_weight=kw)
    want = pk.norm_rope(q, keys, positions, frequencies, **norm)
    buffer = torch.zeros(41, 4, 64, dtype=q.dtype, device="cuda")
    for shift in (0, 1):                                                  # a token further on, and a token back
        buffer[1 - shift:41 - shift] = q
        pk.norm_rope(buffer[1 - shift:41 - shift], None, positions, frequencies, q_weight=qw, q_out=buffer[shift:40 + shift])
        assert torch.equal(buffer[shift:40 + shift], want[0])
    square = torch.empty(8, 8, 64, dtype=q.dtype, device="cuda")          # the same memory, the other way about
    square.copy_(torch.cat([q[:8], q[8:16]], 1))
    turned, p8 = square.transpose(0, 1), positions[:8]
    right = pk.norm_rope(square.clone(), None, p8, frequencies, q_weight=qw)[0]
    pk.norm_rope(square, None, p8, frequencies, q_weight=qw, q_out=turned)
    assert torch.equal(turned, right)
    packed = torch.cat([q, keys], 1)                                      # a packed projection, in place
    views = packed[:, :4], packed[:, 4:]
    pk.norm_rope(*views, positions, frequencies, q_out=views[0], keys_out=views[1], **norm)
    assert torch.equal(views[0], want[0]) and torch.equal(views[1], want[1])
    out = torch.empty_like(q)
    for bad in (dict(q_out=keys), dict(keys_out=q), dict(q_out=out, keys_out=out), dict(q_out=keys, keys_out=q)):
        with pytest.raises(ValueError, match="place"):
            pk.norm_rope(q, keys, positions, frequencies, **norm, **bad)
    for bad in (out[:1].expand(40, 4, 64), out[:, :1].expand(40, 4, 64)):
        with pytest.raises(ValueError, match="apart"):
            pk.norm_rope(q, keys, positions, frequencies, q_out=bad, **norm)
    assert pk.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_pools_step_gives_the_turned_keys_too(dtype):
    """keys_out through the pool, with a fresh buffer and without; a refused step leaves no fresh rows behind."""
    from crit_b200.batch import StepBatch
    from crit_b200.pool import FreshBuffer, KVPool
    q, keys, qw, kw, positions, frequencies = inputs(40, 8, 2, 64, 64, dtype, 5)
    values, positions = torch.randn_like(keys), torch.arange(40, device="cuda")
    want = pk.norm_rope(q, keys, positions, frequencies, q_weight=qw, key_weight=kw)
    for fresh in (None, FreshBuffer(torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"))):
        pool = KVPool([0], 2, 64, 256, "cuda", "int4", window=16, fresh=fresh)
        pool.open("a")
        slots, turned = pool.reserve(StepBatch.build([("a", 0, 40)], "cuda")), torch.empty_like(keys)
        found = pool.norm_rope_write(0, slots, q, keys, values, positions, frequencies, q_weight=qw, key_weight=kw, keys_out=turned)
        assert torch.equal(found, want[0]) and torch.equal(turned, want[1])
        if fresh is not None:
            rows = pool.fresh_rows(0, 40)
            assert torch.equal(rows[0], want[1].bfloat16()) and torch.equal(rows[1], values.bfloat16())
            with pytest.raises(ValueError):
                pool.norm_rope_write(0, slots[:3], q, keys, values, positions, frequencies, q_weight=qw, key_weight=kw)
            assert pool.fresh_rows(0, 40) is None
    assert pk.status() == 0


def test_cosines_and_sines_are_those_of_the_angle_in_64_bits():
    """Pairs of (1, 0) come out as (cos, sin).  The angle is reduced in FP64 and its part beyond FP32 put back, so what is left is
    sincospi's unit and two roundings: 2^-22 of each number (the reduction's own error is below 2^-33 of a turn here)."""
    _, _, _, _, _, frequencies = inputs(1, 1, 1, 128, 128, torch.float32, 6)
    positions = torch.cat([torch.arange(1, 2000), torch.randint(0, 1 << 20, (2000,), generator=torch.Generator().manual_seed(7))]).cuda()
    for interleaved in (False, True):
        q = torch.zeros(len(positions), 1, 128, device="cuda")
        first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 64), slice(64, 128))
        q[..., first] = 1.0
        out = pk.norm_rope(q, None, positions, frequencies, interleaved=interleaved)[0][:, 0].double()
        angle = positions.double()[:, None] * frequencies.double()
        for got, want in ((out[:, first], angle.cos()), (out[:, second], angle.sin())):
            assert bool(((got - want).abs() <= 2.0 ** -22 * want.abs() + 2.0 ** -30).all())
