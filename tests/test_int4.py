"""The 4-bit page kind without a GPU: the format's definition, and what the C ABI refuses before any launch."""
import ctypes

import numpy as np
import pytest

from int4_oracle import SCALES, quantise4, scale_byte, values4


def test_scales_are_the_top_bytes_of_fp16_numbers():
    assert np.array_equal(SCALES, (np.arange(248, dtype=np.uint16) << 7).view(np.float16).astype(np.float64))
    assert np.array_equal(scale_byte(SCALES), np.arange(248))
    middle = (SCALES[1:] + SCALES[:-1]) / 2                                     # half to even
    assert np.array_equal(scale_byte(middle), np.arange(247) + np.arange(247) % 2)
    assert scale_byte(np.array([1e9]))[0] == 247


def test_every_value_is_exact_in_sixteen_bits():
    codes, byte = np.meshgrid(np.arange(1, 16, dtype=np.uint8), np.arange(248, dtype=np.uint8), indexing="ij")
    x = values4(np.repeat(codes[..., None], 32, -1), byte[..., None])[..., 0]
    import torch
    assert torch.equal(torch.from_numpy(x).bfloat16().double(), torch.from_numpy(x))
    inside = np.abs(x) <= 65504
    assert np.array_equal(x[inside].astype(np.float16).astype(np.float64), x[inside])


def test_a_row_quantised_twice_is_itself():
    x = np.random.default_rng(0).standard_normal((50, 2, 128))
    codes, byte = quantise4(x)
    again = quantise4(values4(codes, byte))
    assert np.array_equal(values4(*again), values4(codes, byte))


@pytest.fixture(scope="module")
def lib():
    from crit_b200 import _lib, build
    build.build()
    return _lib.load()


def test_bad_parameters_are_refused_before_any_launch(lib):
    from crit_b200 import _lib
    a = _lib.AppendParams()
    a.keys = a.slots = a.key_pages = a.key_scales = 4096
    a.tokens, a.kv_heads, a.head_dim, a.value_dim, a.page, a.kind = 1, 1, 128, 128, 16, _lib.KIND_INT4
    for field, bad, code in (("key_scales", None, -1), ("key_pages", 4098, -4), ("head_dim", 48, -2), ("kind", 6, -2), ("in_dtype", 7, -1),
                             ("values", 4096, -1)):
        before = getattr(a, field)
        setattr(a, field, bad)
        assert lib.crit_b200_append(ctypes.byref(a), None) == code, field
        setattr(a, field, before)
    g = _lib.GatherParams()
    g.pages = g.scales = g.slots = g.out = 4096
    g.count, g.kv_heads, g.dim, g.page, g.kind = 1, 1, 128, 16, _lib.KIND_INT4
    for field, bad, code in (("scales", None, -1), ("out", 4104, -4), ("dim", 40, -2), ("kind", 6, -2), ("out_dtype", 5, -1)):
        before = getattr(g, field)
        setattr(g, field, bad)
        assert lib.crit_b200_gather(ctypes.byref(g), None) == code, field
        setattr(g, field, before)
    p = _lib.AttendParams()
    p.q = p.out = p.key_pages = p.value_pages = p.key_scales = p.value_scales = p.tables = p.rows = p.starts = p.firsts = 4096
    p.n_rows = p.columns = p.partial_rows = p.max_splits = 1
    p.q_heads, p.kv_heads, p.head_dim, p.value_dim, p.page, p.kind, p.chunk, p.slots = 8, 8, 128, 128, 16, _lib.KIND_INT4, 1024, 64
    for field, bad, code in (("key_scales", None, -1), ("value_scales", None, -1), ("key_scales", 4104, -4), ("value_dim", 64, -2), ("head_dim", 96, -2),
                             ("slots", 0, -2), ("page", 24, -2), ("flags", 8, -2), ("flags", 64, -2), ("flags", 128, -2), ("q", 4098, -4)):
        before = getattr(p, field)
        setattr(p, field, bad)
        assert lib.crit_b200_attend(ctypes.byref(p), None) == code, (field, bad)
        setattr(p, field, before)
