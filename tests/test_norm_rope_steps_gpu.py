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
