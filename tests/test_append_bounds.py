"""What the append is told of the pages' and scales' room, without a GPU: the parameter block made of CPU tensors, never launched."""
import pytest
import torch

import crit_b200 as pk

KINDS = ["bf16", "fp8", "fp8:row", "int8", "fp8:page", "int4"]


@pytest.fixture
def params(monkeypatch):
    monkeypatch.setattr(pk, "_status_word", lambda device: None)
    return lambda *args: pk._append_params(*args, (1.0, 1.0))[0]


def _store(kind, pages, heads, dim, page=16):
    """(pages, scales) of `pages` pages."""
    if kind == "int4":
        return torch.zeros(pages, page, heads, dim // 2, dtype=torch.uint8), torch.zeros(pages, page, heads, dim // 32, dtype=torch.uint8)
    made = torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16 if kind == "bf16" else torch.int8 if kind == "int8" else torch.float8_e4m3fn)
    shape = {"fp8:row": (pages, page, heads), "int8": (pages, page, heads), "fp8:page": (pages, heads)}.get(kind)
    return made, torch.zeros(shape) if shape else None


@pytest.mark.parametrize("kind", KINDS)
def test_slots_are_bound_by_whatever_holds_the_fewest(params, kind):
    keys, values, slots = torch.zeros(3, 2, 64).bfloat16(), torch.zeros(3, 2, 96).bfloat16(), torch.zeros(3, dtype=torch.int64)
    (k, ks), (v, vs) = _store(kind, 6, 2, 64), _store(kind, 4, 2, 96)
    assert params(keys, values, slots, k, v, kind, ks, vs).slots_total == 64                 # the values' pages
    assert params(keys, None, slots, k, None, kind, ks, None).slots_total == 96
    (k, ks), (v, vs) = _store(kind, 4, 2, 64), _store(kind, 6, 2, 96)
    assert params(keys, values, slots, k, v, kind, ks, vs).slots_total == 64
    if kind in ("fp8:row", "int8", "fp8:page"):
        assert params(keys, values, slots, k, v, kind, ks[:3], vs).slots_total == 48          # fewer scales than pages
        assert params(keys, values, slots, k, v, kind, ks, vs[:2]).slots_total == 32
    none, none_scales = _store(kind, 0, 2, 64)
    with pytest.raises(ValueError, match="no slot"):                                          # (0 would say: any)
        params(keys, None, slots, none, None, kind, none_scales, None)


@pytest.mark.parametrize("kind", KINDS)
def test_tensors_that_do_not_fit_together_are_refused(params, kind):
    keys, values, slots = torch.zeros(3, 2, 64).bfloat16(), torch.zeros(3, 2, 64).bfloat16(), torch.zeros(3, dtype=torch.int64)
    (k, ks), (v, vs) = _store(kind, 4, 2, 64), _store(kind, 4, 2, 64)
    assert params(keys, values, slots, k, v, kind, ks, vs).slots_total == 64
    for change in ({3: None}, {4: None}, {1: values[:2]}, {1: values[:, :1]}):
        args = [keys, values, slots, k, v, kind, ks, vs]
        for i, x in change.items():
            args[i] = x
        with pytest.raises(ValueError):
            params(*args)
    if kind in ("fp8:row", "int8", "fp8:page"):
        for bad in (ks.half(), ks.double(), torch.zeros(*ks.shape, 2)[..., 0]):
            with pytest.raises(ValueError, match="scales"):
                params(keys, values, slots, k, v, kind, bad, vs)
            with pytest.raises(ValueError, match="scales"):
                params(keys, values, slots, k, v, kind, ks, bad)
        with pytest.raises(ValueError, match="scales"):
            params(keys, values, slots, k, v, kind, ks, None)
