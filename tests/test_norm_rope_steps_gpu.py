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
