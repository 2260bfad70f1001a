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


def test_an_even_launch_names_its_workspace_and_what_it_does_not_take(lib):
    from crit_b200 import _lib
    p = _lib.AttendParams()
    p.q = p.out = p.key_pages = p.value_pages = p.key_scales = p.value_scales = p.tables = p.rows = p.starts = p.firsts = 4096
    p.n_rows = p.columns = p.partial_rows = p.max_splits = 1
    p.q_heads, p.kv_heads, p.head_dim, p.value_dim, p.page, p.kind, p.chunk, p.slots = 8, 8, 128, 128, 16, _lib.KIND_INT4, 1024, 64
    assert lib.crit_b200_attend_floats(None) == -1
    assert lib.crit_b200_attend_floats(ctypes.byref(p)) == 8 * 130                     # a launch of splits: every state of one split
    for field, bad in (("n_rows", 0), ("columns", 65), ("q_heads", 7), ("kv_heads", 0), ("value_dim", 0), ("max_splits", 0), ("partial_rows", 0)):
        before = getattr(p, field)
        setattr(p, field, bad)
        assert lib.crit_b200_attend_floats(ctypes.byref(p)) == -1, field
        setattr(p, field, before)
    p.max_splits = p.partial_rows = p.q_heads = p.kv_heads = 2 ** 31 - 1
    assert lib.crit_b200_attend_floats(ctypes.byref(p)) == -1                          # (no product of the four wraps)
    p.max_splits = p.partial_rows = 1
    p.q_heads = p.kv_heads = 8
    p.flags = 512
    for field, bad in (("kind", _lib.KIND_FP8), ("value_dim", 64), ("head_dim", 96), ("flags", 512 | 32)):
        before = getattr(p, field)
        setattr(p, field, bad)
        assert lib.crit_b200_attend_floats(ctypes.byref(p)) == -2, field
        assert lib.crit_b200_attend(ctypes.byref(p), None) == -2, field
        setattr(p, field, before)


def test_bad_blocks_of_expand_and_norm_rope_are_refused_before_any_launch(lib):
    from crit_b200 import _lib
    e = _lib.ExpandParams()
    for name in ("key_pages", "value_pages", "key_scales", "value_scales", "tables", "out_keys", "out_values", "out_tables"):
        setattr(e, name, 4096)
    e.sequences, e.width, e.tokens, e.kv_heads, e.dim, e.page, e.slots_total = 1, 2, 5, 8, 128, 16, 64
    assert lib.crit_b200_expand(None, None) == -1
    for field, bad, code in (("key_scales", None, -1), ("tables", None, -1), ("out_tables", None, -1), ("sequences", -1, -1), ("sequences", 70000, -1),
                             ("sequences", 2, -1), ("width", -1, -1), ("tokens", -1, -1), ("position", -1, -1), ("slots_total", 8, -1), ("page", 0, -1),
                             ("dim", 48, -2), ("dim", 0, -2), ("out_dtype", 2, -2), ("out_dtype", -1, -2), ("key_pages", 4098, -4), ("out_values", 4104, -4)):
        before = getattr(e, field)
        setattr(e, field, bad)
        assert lib.crit_b200_expand(ctypes.byref(e), None) == code, (field, bad)
        setattr(e, field, before)
    e.width = 0
    assert lib.crit_b200_expand(ctypes.byref(e), None) == 0                            # no pages: no launch
    n, a = _lib.NormRopeParams(), _lib.AppendParams()
    for name in ("q", "keys", "q_out", "keys_out", "positions", "frequencies"):
        setattr(n, name, 4096)
    n.tokens, n.q_heads, n.kv_heads, n.head_dim, n.rotary, n.n_axes = 3, 4, 2, 64, 64, 1
    n.q_stride_token = n.q_out_stride_token = 256
    n.key_stride_token = n.key_out_stride_token = 128
    n.q_stride_head = n.q_out_stride_head = n.key_stride_head = n.key_out_stride_head = 64
    assert lib.crit_b200_norm_rope(None, None, None) == -1
    for field, bad, code in (("positions", None, -1), ("frequencies", None, -1), ("q", None, -1), ("q_out", None, -1), ("keys", None, -1), ("keys_out", None, -1),
                             ("tokens", -1, -1), ("n_axes", 0, -1), ("n_axes", 3, -1), ("q_heads", -1, -1), ("dtype", 3, -1), ("weight_dtype", -1, -1),
                             ("head_dim", 48, -2), ("head_dim", 288, -2), ("rotary", 0, -2), ("rotary", 12, -2), ("rotary", 72, -2),
                             ("q", 4100, -4), ("keys_out", 4098, -4), ("q_stride_head", 66, -4), ("key_out_stride_token", 130, -4)):
        before = getattr(n, field)
        setattr(n, field, bad)
        assert lib.crit_b200_norm_rope(ctypes.byref(n), None, None) == code, (field, bad)
        setattr(n, field, before)
    for name in ("slots", "key_pages", "value_pages", "key_scales", "value_scales", "values"):
        setattr(a, name, 4096)
    a.tokens, a.kv_heads, a.head_dim, a.value_dim, a.page, a.kind, a.value_stride_token, a.value_stride_head = 3, 2, 64, 64, 16, _lib.KIND_INT4, 128, 64
    for field, bad, code in (("tokens", 2, -1), ("kv_heads", 3, -1), ("head_dim", 32, -1), ("in_dtype", 1, -1), ("slots", None, -1), ("key_scales", None, -1),
                             ("value_pages", None, -1), ("value_dim", 48, -2), ("kind", _lib.KIND_FP8_PAGE, -2), ("kind", 6, -2), ("key_pages", 4104, -4),
                             ("value_pages", 4104, -4), ("values", 4100, -4), ("value_stride_head", 66, -4)):
        before = getattr(a, field)
        setattr(a, field, bad)
        assert lib.crit_b200_norm_rope(ctypes.byref(n), ctypes.byref(a), None) == code, (field, bad)
        setattr(a, field, before)
    n.tokens = 0
    assert lib.crit_b200_norm_rope(ctypes.byref(n), None, None) == 0                   # no tokens: no launch


def test_numbers_for_the_device_are_checked(lib):
    numbers = (ctypes.c_int64 * 2)(1, 2)
    assert lib.crit_b200_put(None, None, 0, None) == 0
    for to, n, code in ((None, 2, -1), (4096, -1, -1), (4100, 2, -4)):
        assert lib.crit_b200_put(to, numbers, n, None) == code
    assert lib.crit_b200_put(4096, None, 2, None) == -1


def test_splits_past_a_page_table_and_tables_past_32_bits_are_refused(lib):
    from crit_b200 import _lib
    p = _lib.AttendParams()
    p.q = p.out = p.key_pages = p.value_pages = p.key_scales = p.value_scales = p.tables = p.rows = p.starts = p.firsts = p.workspace = 4096
    p.n_rows = p.columns = p.partial_rows = 1
    p.q_heads, p.kv_heads, p.head_dim, p.value_dim, p.page, p.kind, p.chunk, p.slots = 8, 8, 128, 128, 16, _lib.KIND_INT4, 64, 64
    p.workspace_floats, p.table_pages = 1 << 20, 5
    for splits in (3, 100):                                                      # the table's 80 positions are two splits of 64
        p.max_splits = splits
        assert lib.crit_b200_attend(ctypes.byref(p), None) == -1
    p.max_splits, p.flags = 1, 512
    for pages in (-1, 1 << 28):
        p.table_pages = pages
        assert lib.crit_b200_attend(ctypes.byref(p), None) == -2


def test_the_pages_of_prompt_chunks():
    import crit_b200 as pk
    assert pk._pages_of([0, 5, 16, 7], [1, 21, 16, 7], 9, 4, 16) == [1, 2, 1, 1]
    assert pk._pages_of(None, None, 64, 4, 16) is None
    for positions, ends, tokens in (([0], [65], 65), (None, None, 65), ([-1], [3], 4), ([3, -5], [5, 2], 7)):
        with pytest.raises(ValueError):
            pk._pages_of(positions, ends, tokens, 4, 16)
