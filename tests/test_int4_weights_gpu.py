"""Attention over "int4" pages where one position takes most of the weight and the others' small weights make the output: the
first token of most trained heads, whose own value is next to nothing.  Against 64 bits, whatever the values' magnitude."""
import math

import pytest
import torch

import crit_b200 as pk
from int4_oracle import Cache4

pytestmark = pytest.mark.gpu


def _cache(heads, dim, n, magnitude, mean, seed):
    """One sequence that every row of a launch reads (so that a block's run is thousands of positions of few pages): the
    first group of each key is zeros, but for position 0, whose other groups are zeros; position 0's value is zeros."""
    g = torch.Generator().manual_seed(seed)
    cache = Cache4(heads, dim, 16, n // 16 + 2)
    cache.tables = torch.randperm(n // 16 + 1, generator=g).to(torch.int32).cuda()[None]
    keys = torch.randn(n, heads, dim, generator=g)
    keys[:, :, :32] = 0
    keys[0] = 0
    keys[0, :, :32] = 7 / 8                                    # (held as it is: 7 codes of 1/8)
    values = (torch.randn(n, heads, dim, generator=g) + mean) * magnitude
    values[0] = 0
    cache.write(0, 0, keys.bfloat16().cuda(), values.bfloat16().cuda())
    return cache


def _queries(cache, tokens, heads, dim, n, share, dtype, seed):
    """Queries whose position 0 takes about `share` of the softmax over n positions of standard-normal logits."""
    q = torch.randn(tokens, heads, dim, generator=torch.Generator().manual_seed(seed))
    logit = math.log(share / (1 - share)) + math.log(n) + 0.5 * (dim - 32) / dim
    q[:, :, :32] = logit * math.sqrt(dim) / (32 * 7 / 8)
    return q.to(dtype).cuda()


def _close(cache, q, out, lse, tokens, lengths):
    """Beside half a step of the type: a weight rounded to FP16, 2^-12 of it; scores of sums |q k| below 30 summed in FP32, in the
    weight and in the total, 4.9e-4; FP32 sums of 2^10 products of 16 at the most, 2^-13: below 2^-9 of the weighted sum of
    |values|.  Weights below 2^-25 of the largest are rounded to steps of 2^-35 of it, 2^-36 a position."""
    k, v = (torch.from_numpy(cache.rows(which, 0, max(lengths))).cuda() for which in ("k", "v"))
    group = q.shape[1] // cache.heads
    for token, length in zip(tokens, lengths):
        for h in range(cache.heads):
            x = q[token, h * group:(h + 1) * group].double() @ k[:length, h].T * q.shape[-1] ** -0.5
            w = torch.softmax(x, -1)
            want, room = w @ v[:length, h], w @ v[:length, h].abs()
            tiny = length * 2.0 ** -36 * v[:length, h].abs().max() * w.max(-1, keepdim=True).values
            got = out[token, h * group:(h + 1) * group].double()
            tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -9 * room + tiny + (2.0 ** -25 if q.dtype == torch.float16 else 1e-30)
            assert bool(got.isfinite().all())
            worst = float(((got - want).abs() / tol).max())
            assert worst <= 1, f"token {token}, kv head {h}: {worst:.2f} of the bound (weight of position 0: {float(w[:, 0].mean()):.3f})"
            assert float((lse[token, h * group:(h + 1) * group].double() - torch.logsumexp(x, -1)).abs().max()) <= 3e-4


LAUNCHES = [  # rows, positions, q_heads, kv_heads, dim, columns, dtype, engine
    (256, 16384, 8, 1, 128, 1, torch.bfloat16, None),
    (64, 4096, 64, 8, 128, 1, torch.bfloat16, None),
    (200, 8000, 8, 2, 64, 1, torch.bfloat16, None),
    (40, 20000, 8, 2, 256, 1, torch.bfloat16, None),
    (256, 16384, 8, 1, 128, 1, torch.float16, None),
    (64, 8192, 15, 3, 128, 6, torch.float16, None),
    (64, 8192, 10, 5, 128, 3, torch.bfloat16, None),
    (6, 16384, 8, 1, 128, 1, torch.bfloat16, "mma.sync"),
    (6, 16384, 8, 1, 256, 2, torch.float16, "mma.sync"),
]


@pytest.mark.parametrize("share", [0.5, 0.9, 0.99, 0.9999])
@pytest.mark.parametrize("rows,n,hq,hkv,dim,columns,dtype,engine", LAUNCHES)
def test_small_weights_beside_a_dominant_one_are_kept(rows, n, hq, hkv, dim, columns, dtype, engine, share):
    i32 = dict(dtype=torch.int32, device="cuda")
    for magnitude, mean in ((1.0, 0.0), (0.1, 0.0), (0.02, 0.5), (3e-4, 0.0)):
        cache = _cache(hkv, dim, n, magnitude, mean, 1)
        q = _queries(cache, rows * columns, hq, dim, n, share, dtype, 2)
        out, lse = torch.full_like(q, float("nan")), torch.full((rows * columns, hq), float("nan"), device="cuda")
        starts = torch.arange(rows, **i32) * columns
        kw = dict(chunk=16384) if engine else {}
        pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.zeros(rows, **i32), starts, torch.full((rows,), n - columns, device="cuda"), columns, 16,
                  key_scales=cache.ks, value_scales=cache.vs, out=out, lse=lse, engine=engine, **kw)
        at = [0, rows // 2, rows - 1]
        _close(cache, q, out, lse, [r * columns + columns - 1 for r in at], [n] * 3)
        assert pk.status() == 0


def test_the_largest_values_with_every_weight_at_the_top():
    """Scales of 61,440 under weights that are all the largest there is."""
    cache = Cache4(1, 128, 16, 20)
    cache.tables = torch.arange(20, dtype=torch.int32, device="cuda")[None]
    n = 300
    keys, values = torch.zeros(n, 1, 128), torch.full((n, 1, 128), 4e5)
    values[:, :, 1::2] = -4e5
    cache.write(0, 0, keys.cuda(), values.cuda())
    i32 = dict(dtype=torch.int32, device="cuda")
    for columns in (1, 4):
        q = torch.randn(columns, 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
        for engine in (None, "mma.sync"):
            out = pk.attend(q, cache.k, cache.v, "int4", cache.tables, torch.zeros(1, **i32), torch.zeros(1, **i32), torch.tensor([n - columns], device="cuda"),
                            columns, 16, key_scales=cache.ks, value_scales=cache.vs, engine=engine)
            want = torch.from_numpy(cache.rows("v", 0, 1)[0, 0]).cuda()
            assert bool((out.double() - want).abs().le(2.0 ** -8 * want.abs()).all())
    assert pk.status() == 0
