"""crit_b200: the paged KV-cache hot path of crit, hand-written for B200 (sm_100a).

This module is the kernel-module boundary: the object crit's KVPool and DeviceAttention take as `kernels=`
(reference: kernels/techniques/attention/paged-kv-attention/torch-ext/paged_kv_attention/__init__.py, loaded by
crit_plugins.kernels.load_kernel("paged-kv-attention")).  It keeps that module's names, argument meanings and errors
for write / attend / prefill / partitions / piece_size / tile_for / workspace_floats / owner / release, and reaches
the CUDA kernels through the C ABI of include/crit_b200.h (ctypes, as the reference binds its own CUDA tile).  There
is no Triton, no torch fallback and no CPU path: without the native library, or on a tensor that is not on a CUDA
device, every entry point raises.

Page kinds: the reference's "bf16", "fp16", "fp8", "fp8:row", "int8", and "fp8:page": E4M3 codes with one FP32 scale
per (page, kv head), scales [pages][kv_heads] (scale = amax / 448 over the page's rows of that head); and "int4": 4-bit
codes, pages uint8 [pages][page][kv_heads][dim / 2] (element 2 i in the low half of byte i), with one byte of scale for
each group of 32 elements, scales uint8 [pages][page][kv_heads][dim / 32].  The byte is an unsigned float, bits 14..7 of
an FP16 number: the one nearest to the group's max |x| / 7 (61,440 at most); a code is 8 + rint(x / scale) and stands for
(code - 8) * scale, at most half a scale from x (scales of 2^-14 and above), exact in 16-bit types.  A group that holds a NaN reads as NaN.

A row's positions are read in contiguous splits of `chunk` positions (one per cache geometry, chunk_for()); the splits'
states are folded in split order.  This is the reference's "flash" split shape (contiguous splits, __init__.py:580-612)
rather than its interleaved pieces; attention outputs agree with the reference's within its own kernel-vs-torch
tolerance, integer and byte results (slots, codes, scales) bit for bit.
"""
import contextlib
import ctypes
import itertools
import struct
import math
import threading

import torch

from . import _lib

__all__ = ["KINDS", "MAX_COLUMNS", "attend", "chunk_for", "gather", "merge_shards", "move_rows", "norm_rope", "norm_rope_write", "owner",
           "partitions", "parts_for", "rope_axes", "engine_for", "piece_size", "plan", "prefill", "prefill_serves", "release", "slots_at", "states_for", "status", "tcgen05_serves",
           "tcgen05p_serves", "tile_for", "workspace_floats", "write"]

_STAGINGS = {None: 0, "cp.async": 1, "tma": 2}
_ENGINES = {"tcgen05": 8, "mma.sync": 16, "tcgen05t": 64, "tcgen05p": 128, "even": 512}
_PREFILL_ENGINES = {None: 0, "mma.sync": 1, "tcgen05": 2, "tcgen05:single": 2 | 4, "tcgen05:pair": 2 | 8}
KINDS = {"bf16": 0, "fp16": 0, "fp8": 1, "fp8:row": 2, "int8": 3, "fp8:page": 4, "int4": 5}
GROUP4 = 32                 # elements of an "int4" row that share a scale
MAX_COLUMNS = 64            # columns of one row a launch reads
TILE = 16                   # positions a warp reads per step: chunks and pages are multiples of it
DEFAULT_CHUNK = 1024

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
_PAGE_DTYPES = {"bf16": _lib.DTYPE_BF16, "fp16": _lib.DTYPE_FP16}


def _check_kind(kind, key_scales):
    if kind not in KINDS:
        raise ValueError(f"page kinds are {', '.join(KINDS)}, not {kind!r}")
    if (KINDS[kind] >= 2) != (key_scales is not None):
        raise ValueError(f"{kind} pages {'take' if KINDS[kind] >= 2 else 'have no'} scales beside their codes")
    return KINDS[kind]


def _check4(pages, scales, what):
    """An "int4" page tensor [...][kv_heads][dim / 2] and its scales [...][kv_heads][dim / 32]: (kv_heads, dim)."""
    shape = pages.shape
    hkv, half = shape[-2], shape[-1]
    if pages.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise ValueError(f"int4 pages and their scales are uint8 tensors: {what} are {pages.dtype} with scales of {scales.dtype}")
    if half % (GROUP4 // 2) or scales.numel() * (GROUP4 // 2) != pages.numel() or not scales.is_contiguous() or not pages.is_contiguous():
        raise ValueError(f"int4 {what} of [{hkv}][{2 * half}] rows have contiguous scales [...][{hkv}][{2 * half // GROUP4}], a byte for "
                         f"each group of {GROUP4} elements")
    if scales.get_device() != pages.get_device():
        raise ValueError(f"int4 {what} and their scales are on one device")
    return hkv, 2 * half


def _cuda(tensor, what):
    if not tensor.is_cuda:
        raise RuntimeError(f"crit_b200 runs on CUDA devices only: {what} is on {tensor.device} (there is no CPU path)")
    return tensor


def _ptr(tensor):
    return tensor.data_ptr() if tensor is not None else 0


# (the handle alone: a Stream object takes longer to make than a launch's other host work)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(name, what, device, *params):
    """The library's entry point `name` on the device's current stream, with that device current; errors raised."""
    call, index, current = getattr(_lib.load(), name), device.index, torch.cuda.current_device()
    if index is None or index == current:
        code = call(*params, _raw_stream(current))
    else:
        with torch.cuda.device(index):
            code = call(*params, _raw_stream(index))
    if code:
        _lib.check(code, what)


def _page_dtype(kind, pages):
    if KINDS[kind] != 0:
        return _lib.DTYPE_BF16
    if pages.dtype not in _DTYPES:
        raise ValueError(f"{kind} pages are 16-bit tensors, not {pages.dtype}")
    return _DTYPES[pages.dtype]


# -- workspaces -----------------------------------------------------------------------------------------------------------
# One per (device, owner): a launch writes its partials and the merge reads them back, so two engines of one process
# never share one (reference: paged_kv_attention/__init__.py:129-171).  A workspace a launch outgrew is kept: a CUDA
# graph captured over it replays into it.
_workspaces, _retired = {}, []
_owner = threading.local()


@contextlib.contextmanager
def owner(key):
    """Launches inside this block take a workspace of their own, apart from every other owner's."""
    before = getattr(_owner, "key", None)
    _owner.key = key
    try:
        yield
    finally:
        _owner.key = before


def release(key):
    """Drop an owner's workspaces (its captured graphs must be gone: they replay into them)."""
    for at in [at for at in _workspaces if at[1] == key]:
        del _workspaces[at]
    _retired[:] = [(k, found) for k, found in _retired if k != key]


def _workspace(device, floats, given):
    if given is not None:
        if given.dtype != torch.float32 or given.numel() < floats or not given.is_contiguous() or given.device != device:
            raise ValueError(f"attend's workspace holds {given.numel()} floats on {given.device}; this launch needs {floats} "
                             f"contiguous FP32 ones on {device} (workspace_floats)")
        return given
    at = (device.index, getattr(_owner, "key", None))
    found = _workspaces.get(at)
    if found is None or found.numel() < floats:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("crit_b200.attend: run a launch of this size once before capturing it (its partials' "
                               "workspace is allocated outside the capture)")
        if found is not None:
            _retired.append((at[1], found))
        found = _workspaces[at] = torch.empty(max(floats, 1 << 20), dtype=torch.float32, device=device)
    return found


_status, _status_at = {}, {}
_even_floats = {}           # an even launch's workspace, by device and shape (the library's answer)


def _status_word(device):
    """One int32 a device: a kernel sets it (and never clears it) when one of its bounded waits gave up."""
    found = _status_at.get(device.index)
    if found is not None:
        return found
    found = _status.get(str(device))
    if found is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        found = _status[str(device)] = torch.zeros(1, dtype=torch.int32, device=device)
    if device.index is not None:
        _status_at[device.index] = found
    return found


def status(device=None):
    """0, or what a kernel recorded on `device` since load, when one of its bounded waits ran out (the block concerned
    wrote nothing): 1 = a TMA copy of the m16n8k16 decode kernel; 0x110 / 0x120 / 0x140 = the producer / MMA / softmax
    warps of the tcgen05 prefill kernel (0x1ff: its shared memory was not 1 KB aligned); 0x410 / 0x420 / 0x440 = the
    producer / MMA / softmax warps of the tcgen05 decode kernel; 0x800 + rank = the peer exchange of the shards' partials
    waited in vain for another rank's message.  Reads the device word (one synchronisation)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    found = _status.get(str(device))
    return 0 if found is None else int(found.item())


# -- geometry rules -----------------------------------------------------------------------------------------------------
def chunk_for(head_dim, value_dim, heads, kv_heads, page, kind="bf16", engine=None, columns=1):
    """Positions per split of a launch over a cache of this geometry (a multiple of 16).  One per cache for the
    m16n8k16 kernel, never by the batch, so a column's bits are the same alone and in any window.  Launches of the
    tcgen05 kernel that gives a unit one kv head (engine "tcgen05", or attend's own choice for windows of several columns
    over E4M3 pages) use splits of 2,048: a unit's fold of its lane replicas is paid once per split."""
    if engine is None:
        engine = engine_for(kind, head_dim, value_dim, heads, kv_heads, columns)
    return 2 * DEFAULT_CHUNK if engine in ("tcgen05", "tcgen05t") else DEFAULT_CHUNK


def tcgen05_serves(kind, head_dim, value_dim, heads, kv_heads, columns, chunk, rows=1):
    """Whether the tcgen05 kernel takes a launch: E4M3 pages of 128-wide heads, at most 32 query rows a unit (columns
    x heads of a kv head's group), splits of whole 128-position tiles up to 2,048 positions, up to 256 window rows (the
    same test the library makes: decode.cu, tc_serves)."""
    return (str(kind).startswith("fp8") and head_dim == 128 and value_dim == 128 and columns * (heads // kv_heads) <= 32
            and chunk % 128 == 0 and chunk <= 2048 and rows <= 256)


def tcgen05p_serves(kind, head_dim, value_dim, heads, kv_heads, columns, chunk, rows=1):
    """Whether the tcgen05 kernel over whole page rows takes a launch: E4M3 pages of 128-wide heads, 8 kv heads, at most 8
    query rows a kv head (columns x heads of a group), splits of whole 16-position tiles up to 2,048 positions, up to 256
    window rows (the same test the library makes: decode.cu, ph_serves)."""
    return (str(kind).startswith("fp8") and head_dim == 128 and value_dim == 128 and kv_heads == 8 and
            columns * (heads // kv_heads) <= 8 and chunk % 16 == 0 and chunk <= 2048 and rows <= 256)


# Launches below this many positions (window rows x the positions their tables hold) stay on the m16n8k16 kernel: the
# whole-page-rows kernel deals whole splits to its blocks, and a small launch has too few to fill the device.
PAGE_ROWS_FROM = 1 << 16
EVEN_ROWS = 256             # window rows an even launch takes (decode4.cu, D4_MAX_ROWS)
_LISTED_ROWS = {"even": EVEN_ROWS, "tcgen05": 256, "tcgen05p": 256, "tcgen05t": 128}      # window rows the kernels take that list them


def engine_for(kind, head_dim, value_dim, heads, kv_heads, columns, rows=1, positions=None, engine=None):
    """The kernel a launch runs on: `engine` when one is named, else attend's own choice: "tcgen05p" (whole page rows:
    every kv head of a position in one contiguous read) for E4M3 pages of 8 kv heads x 128 with at most 8 query rows a
    kv head, when the launch is large enough to fill the device that way; "tcgen05" for other windows of several
    columns over E4M3 pages of 128-wide heads; "even" for int4 pages, up to 256 window rows (the m16n8k16 kernel of 4-bit
    pages with the launch's positions dealt out evenly to the device's blocks, not cut into splits); "mma.sync" (m16n8k16)
    for everything else.  Only the last gives a column the same bits alone and in any window or batch."""
    if engine is not None:
        return engine
    if kind == "int4":
        return "even" if rows <= EVEN_ROWS else "mma.sync"
    if tcgen05p_serves(kind, head_dim, value_dim, heads, kv_heads, columns, DEFAULT_CHUNK, rows) and \
            positions is not None and rows * positions >= PAGE_ROWS_FROM:
        return "tcgen05p"
    if columns > 1 and tcgen05_serves(kind, head_dim, value_dim, heads, kv_heads, columns, 2 * DEFAULT_CHUNK, rows):
        return "tcgen05"
    return "mma.sync"


def states_for(parts, engine):
    """Split states a partial row takes in the workspace for `parts` splits: the whole-page-rows kernel deals the
    launch's tiles out evenly, so a split may be shared by two blocks and has two states (its head and its tail)."""
    return 2 * parts if engine == "tcgen05p" else parts


def parts_for(positions, chunk):
    """Splits a partial row takes over page tables holding `positions` positions a row."""
    return max(1, -(-int(positions) // int(chunk)))


_plans = {}


def plan(heads, kv_heads, head_dim, value_dim, page, kind="bf16", columns=1, device=None):
    """What the library would launch for a cache of this geometry on `device`: a dict of chunk (positions per split),
    smem (bytes of shared memory a block takes), rows (query rows a block's tile holds), per_sm (blocks resident per
    SM) and sms.  Asked of the library once per geometry and device (crit_b200_attend_plan)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    key = (str(device), heads, kv_heads, head_dim, value_dim, page, kind, columns)
    found = _plans.get(key)
    if found is None:
        out = (ctypes.c_int32 * 5)()
        dtype = _lib.DTYPE_FP16 if kind == "fp16" else _lib.DTYPE_BF16
        with torch.cuda.device(device):
            _lib.check(_lib.load().crit_b200_attend_plan(heads, kv_heads, head_dim, value_dim, page, KINDS[kind], dtype, columns, out),
                       "crit_b200.plan")
        found = _plans[key] = dict(chunk=out[0], smem=out[1], rows=out[2], per_sm=out[3], sms=out[4])
    return found


def partitions(device, kv_heads, kind, head_dim=None, value_dim=None):
    """The most splits a partial row takes in a launch whose caller sizes the workspace by a count per cache
    (reference: paged_kv_attention/__init__.py:260-273, a rule over the device's SMs, the kv heads and the code width).
    Here: enough splits for two waves of the device's resident blocks from ONE row (its splits x kv_heads blocks), as
    a power of two in 8..128.  attend(partitions=P) never makes more than P splits: it raises the chunk where a row's
    tables hold more than P * chunk positions."""
    head_dim = head_dim or 128
    value_dim = value_dim or head_dim
    found = plan(kv_heads, kv_heads, head_dim, value_dim, TILE, kind, 1, device)
    want = max(1, 2 * found["sms"] * max(found["per_sm"], 1) // max(kv_heads, 1))
    return min(128, max(8, 1 << (want.bit_length() - 1)))


def piece_size(head_dim, value_dim, kind="bf16", kv_heads=None):
    """Positions a warp reads per step (reference: __init__.py:276-286; here the tile is 16 for every geometry)."""
    return TILE


def tile_for(columns, group, capability, fused=False):
    """(rows, warps, stages) of a launch's query tile (reference: __init__.py:335-356): 8, 16 or 32 query rows (columns
    x the group's heads, in tiles of 8), four warps, each with its own ring of 3 or 4 stages (4 where a warp's
    iteration takes two 16-position tiles, which 8-bit pages of heads up to 128 wide do; the width is not an argument
    here, so the deeper ring is reported)."""
    rows = columns * group
    return (8 if rows <= 8 else (16 if rows <= 16 else 32)), 4, 4


def workspace_floats(tokens, heads, partitions, value_dim):
    """FP32 floats of the partials a launch needs for `tokens` partial rows (reference: __init__.py:359-362)."""
    return tokens * heads * partitions * (value_dim + 2)


# -- KV append ----------------------------------------------------------------------------------------------------------
def write(keys, values, slots, key_pages, value_pages, kind, key_scales=None, value_scales=None,
          multipliers=(1.0, 1.0)):
    """A step's keys [tokens][kv_heads][dim] and values [tokens][kv_heads][value_dim] (bf16, fp16 or fp32) into their
    slots ([tokens] int64; a slot below 0 is skipped; a slot at most once a call) of one layer's pages (any view whose
    storage is [slots][kv_heads][dim]; "int4": two elements a byte), encoded for the page kind, in one launch.  values and value_pages None: keys only; keys
    and key_pages None: values only, at the value multiplier.  "fp8:page" takes scales [pages][kv_heads] and the page
    size from the pages' shape ([pages][page][kv_heads][dim]).  Reference: paged_kv_attention/__init__.py:289-324."""
    if keys is None:
        if values is None:
            raise ValueError("write takes keys, values or both")
        return write(values, None, slots, value_pages, None, kind, value_scales, None,
                     multipliers=(multipliers[1], multipliers[1]))
    _cuda(keys, "keys")
    if keys.shape[0] == 0:
        _check_kind(kind, key_scales)
        return
    p, _held = _append_params(keys, values, slots, key_pages, value_pages, kind, key_scales, value_scales, multipliers)
    _run("crit_b200_append", "crit_b200.write", keys.device, p)


def _append_params(keys, values, slots, key_pages, value_pages, kind, key_scales, value_scales, multipliers):
    """The append's parameter block, its arguments checked, and the tensors it points at that were made here."""
    k_kind = _check_kind(kind, key_scales)
    T, hkv, d = keys.shape
    in_dtype, place = _DTYPES.get(keys.dtype), keys.get_device()
    if in_dtype is None or (values is not None and values.dtype != keys.dtype):
        raise ValueError("keys and values are bf16, fp16 or fp32 tensors of one dtype")
    if keys.stride(-1) != 1:
        keys = keys.contiguous()
    if values is not None and values.stride(-1) != 1:
        values = values.contiguous()
    if slots.dtype is not torch.int64 or not slots.is_contiguous() or slots.numel() != T or slots.get_device() != place:
        raise ValueError(f"slots are contiguous int64 [{T}] on the keys' device")
    if key_pages is None or (values is not None and value_pages is None and k_kind != 5):
        raise ValueError("write stores rows in pages: pass them beside the rows")
    if not key_pages.is_contiguous() or (value_pages is not None and not value_pages.is_contiguous()):
        raise ValueError("pages are contiguous [slots][kv_heads][dim] storage")
    page, dv = 1, d
    if k_kind == 5:
        if (hkv, d) != _check4(key_pages, key_scales, "keys") or key_pages.get_device() != place:
            raise ValueError(f"int4 keys [{T}][{hkv}][{d}] go to pages [...][{hkv}][{d // 2}] on their device")
        if values is not None:
            if value_pages is None or value_scales is None:
                raise ValueError("write stores int4 values in pages with scales beside them")
            if values.shape != (T, *_check4(value_pages, value_scales, "values")) or value_pages.get_device() != place or values.get_device() != place:
                raise ValueError(f"int4 values {list(values.shape)} go to pages [...][{hkv}][{values.shape[-1] // 2}] on their device, a row a token")
    elif k_kind == 4:
        if key_pages.dim() != 4:
            raise ValueError("fp8:page pages are given as [pages][page][kv_heads][dim]")
        page = key_pages.shape[1]
    value_at = value_token = value_head = 0
    if values is not None:
        value_at, (value_token, value_head, _), dv = values.data_ptr(), values.stride(), values.shape[-1]
    if k_kind == 5:                              # (checked above)
        held = key_pages.numel() * 2 // (hkv * d)
        if values is not None:
            held = min(held, value_pages.numel() * 2 // (hkv * dv))
    else:
        held = _slots_held(key_pages, key_scales, k_kind, hkv, d, page, place)
        if values is not None:
            if values.shape[0] < T or values.shape[1] != hkv or values.get_device() != place:
                raise ValueError(f"values are [{T}][{hkv}][value_dim] on the keys' device, not {list(values.shape)}")
            held = min(held, _slots_held(value_pages, value_scales, k_kind, hkv, dv, page, place))
    if T and held < 1:
        raise ValueError("the pages (and their scales) hold no slot")
    key_token, key_head, _ = keys.stride()
    p = _lib.block(_lib.AppendParams, keys.data_ptr(), value_at, slots.data_ptr(), key_pages.data_ptr(), _ptr(value_pages), _ptr(key_scales), _ptr(value_scales),
                   _ptr(_status_word(keys.device)), T, held, key_token, key_head, value_token, value_head,
                   hkv, d, dv, page, k_kind, in_dtype, _page_dtype(kind, key_pages), multipliers[0], multipliers[1])
    return p, (keys, values)


def _slots_held(pages, scales, k_kind, heads, dim, page, place):
    """The slots that a page tensor (of another kind than "int4") and its scales have room for: the append writes to none beyond."""
    if pages.get_device() != place:
        raise ValueError("pages are on the keys' device")
    if k_kind < 2:
        return pages.numel() // (heads * dim)
    if scales is None or scales.dtype is not torch.float32 or not scales.is_contiguous() or scales.get_device() != place:
        raise ValueError("scales are contiguous FP32 on the keys' device, a tensor beside each of the page tensors")
    return min(pages.numel() // (heads * dim), scales.numel() // heads * (page if k_kind == 4 else 1))


# -- norm and rotation ----------------------------------------------------------------------------------------------------
def rope_axes(sections, interleaved=False, device="cuda"):
    """The axis each pair of a head turns with, int32 [sum(sections)]: norm_rope's `axes` for positions of several axes
    (time, height, width).  sections: the pairs each axis turns.  interleaved False: one axis' pairs after another's; True:
    the axes take turns, pair by pair, each until its pairs are used up."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0:
        raise ValueError("sections are the numbers of pairs each axis turns")
    if interleaved:
        order = sorted((turn, axis) for axis, n in enumerate(sections) for turn in range(n))
        found = [axis for _, axis in order]
    else:
        found = [axis for axis, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(found, dtype=torch.int32, device=device)


def _vectors_fit(x):
    """Whether rows are read or written in the kernel's vectors of four elements as they lie."""
    token, head, element = x.stride()
    return element == 1 and not (token | head) & 3 and not x.data_ptr() % (4 * x.element_size())


def _like(x):
    """An uninitialised contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _vectors(x):
    """x where the kernel's vectors fit it, else a copy."""
    return x if _vectors_fit(x) else x.clone(memory_format=torch.contiguous_format)


def _bytes(x):
    """The addresses a tensor lies between."""
    at = x.data_ptr()
    return at, at + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size() if x.numel() else at


def _in_place(out, x):
    """Whether rows may be written to `out` as they are made of x's: its own place, or memory apart from it."""
    if out.data_ptr() == x.data_ptr() and out.stride() == x.stride():
        return True
    (a, b), (c, d) = _bytes(out), _bytes(x)
    return b <= c or d <= a


def _norm_rope_params(q, keys, positions, frequencies, q_weight, key_weight, eps, offset, axes, interleaved, magnitude, q_out, keys_out, writes):
    """norm_rope's arguments checked: (parameter block, [q, keys] as they are read, [q, keys] outputs, outputs to copy)."""
    given = q if q is not None else keys
    if given.dim() != 3:
        raise ValueError("q and keys are [tokens][heads][dim]")
    (T, _, d), device, place, dtype = given.shape, given.device, given.get_device(), given.dtype
    half, n_axes, axis_stride, weight_dtype = frequencies.numel(), 1, 0, None
    if dtype not in _DTYPES or (q is not None and keys is not None and
                                (keys.dim() != 3 or keys.shape[0] != T or keys.shape[-1] != d or keys.dtype != dtype or keys.get_device() != place)):
        raise ValueError("q and keys are bf16, fp16 or fp32 tensors [tokens][heads][dim] of one dtype, width and device")
    if frequencies.dtype is not torch.float32 or frequencies.dim() != 1 or not frequencies.is_contiguous() or frequencies.get_device() != place:
        raise ValueError("frequencies are contiguous FP32 [rotary / 2] on the queries' device")
    ways = positions.dim()
    if ways == 2:
        n_axes, axis_stride = positions.shape[0], positions.stride(0)
    if positions.dtype is not torch.int64 or ways not in (1, 2) or positions.shape[-1] != T or positions.get_device() != place or \
            (T > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions are int64 [{T}], or [axes][{T}], on the queries' device")
    if axes is not None:
        if axes.dtype is not torch.int32 or axes.numel() != half or not axes.is_contiguous() or axes.get_device() != place:
            raise ValueError("axes are contiguous int32, one for each frequency (rope_axes)")
    elif n_axes > 1:
        raise ValueError("positions of several axes come with the axis of each pair: axes (rope_axes)")
    for w in (q_weight if q is not None else None, key_weight if keys is not None else None):
        if w is not None:
            weight_dtype = weight_dtype or w.dtype
            if w.dtype not in _DTYPES or w.dtype != weight_dtype or w.numel() != d or not w.is_contiguous() or w.get_device() != place:
                raise ValueError(f"q_weight and key_weight are contiguous [{d}] of one bf16, fp16 or fp32 type, on the queries' device")
    reads, outs, copies, at, strides = [], [], [], [], []
    for x, out, what in ((q, q_out, "q"), (keys, keys_out, "keys")):
        if x is None:
            if out is not None:
                raise ValueError(f"there are no {what} for the {what} output, whose shape, dtype and device are theirs")
            reads.append(None), outs.append(None), at.append((0, 0)), strides.append((0, 0, 0, 0, 0, 0))
            continue
        read, into = _vectors(x), out
        if out is None and not (writes and what == "keys"):
            out = into = _like(x)
        elif out is not None:
            if out.shape != x.shape or out.dtype != dtype or out.get_device() != place:
                raise ValueError(f"the {what} output has the shape, dtype and device of {what}")
            if out.numel() and any(n > 1 and not s for n, s in zip(out.shape, out.stride())):
                raise ValueError(f"the {what} output's rows lie apart from one another")
            if not _vectors_fit(out) or not _in_place(out, x):         # made beside it and copied
                into = _like(x)
                copies.append((out, into))
        reads.append(read), outs.append(out), at.append((read.data_ptr(), _ptr(into)))
        strides.append(read.stride() + (into.stride() if into is not None else (0, 0, 0)))
    # (the launch's warps read one tensor's rows while others write the other's)
    if T and q is not None and keys is not None and ((q_out is not None and (q_out.data_ptr() == keys.data_ptr() or keys_out is not None and
            q_out.data_ptr() == keys_out.data_ptr())) or (keys_out is not None and keys_out.data_ptr() == q.data_ptr())):
        raise ValueError("the queries' and the keys' outputs are in each other's or the other input's place")
    (q_at, q_to), (k_at, k_to) = at
    a, b = strides
    p = _lib.block(_lib.NormRopeParams, q_at, k_at, q_to, k_to, positions.data_ptr(), frequencies.data_ptr(), _ptr(axes), _ptr(q_weight), _ptr(key_weight),
                   _ptr(_status_word(device)), T, axis_stride, a[0], a[1], b[0], b[1], a[3], a[4], b[3], b[4],
                   q.shape[1] if q is not None else 0, keys.shape[1] if keys is not None else 0, d, 2 * half, n_axes, bool(interleaved),
                   _DTYPES[dtype], _DTYPES[weight_dtype] if weight_dtype else 0, eps, offset, magnitude)
    return p, reads, outs, copies


def norm_rope(q, keys, positions, frequencies, *, q_weight=None, key_weight=None, eps=1e-6, offset=0.0, axes=None, interleaved=False,
              magnitude=1.0, q_out=None, keys_out=None):
    """A step's queries [tokens][heads][dim] and keys [tokens][kv_heads][dim] (bf16, fp16 or fp32; either may be None), each
    head normed and turned, in one launch -> (queries, keys).

    y = x / sqrt(mean x^2 + eps) * (offset + weight) over each head where its weight [dim] is given; then the first rotary =
    2 * len(frequencies) elements (a multiple of 8) in pairs, (a, b) -> magnitude * (a cos - b sin, b cos + a sin): pairs
    (i, rotary / 2 + i), or (2 i, 2 i + 1) with interleaved.  The angle of pair i is position * frequencies[i], made in FP64;
    positions int64 [tokens], or [axes][tokens] with axes int32 [rotary / 2] naming the axis each pair turns with
    (rope_axes).  Sums are FP32, a result is rounded once.  q_out / keys_out: where to put them (q and keys themselves for
    in place; in no other argument's memory).  Heads of 32..256 in steps of 32."""
    if q is None and keys is None:
        raise ValueError("norm_rope takes q, keys or both")
    _cuda(q if q is not None else keys, "q")
    p, reads, outs, copies = _norm_rope_params(q, keys, positions, frequencies, q_weight, key_weight, eps, offset, axes, interleaved,
                                               magnitude, q_out, keys_out, False)
    _launch_norm_rope(p, None, reads, copies, "crit_b200.norm_rope")
    return outs[0], outs[1]


def _launch_norm_rope(p, append, reads, copies, what):
    if p.tokens == 0:
        return
    device = (reads[0] if reads[0] is not None else reads[1]).device
    _run("crit_b200_norm_rope", what, device, p, append)
    for out, made in copies:
        out.copy_(made)


def norm_rope_write(q, keys, values, positions, frequencies, slots, key_pages, value_pages, kind, key_scales=None, value_scales=None, *,
                    multipliers=(1.0, 1.0), q_weight=None, key_weight=None, eps=1e-6, offset=0.0, axes=None, interleaved=False,
                    magnitude=1.0, q_out=None, keys_out=None):
    """norm_rope with write() in the same launch: the queries and keys normed and turned, the keys and the values [tokens]
    [kv_heads][value_dim] (None: keys only) stored at their slots of one layer's pages -> the queries (q None: None).  The keys go
    to the pages from their FP32 values, with no rounding to their type on the way (16-bit pages of that type hold what
    norm_rope + write would put there); keys_out takes them too when given (no output lies in the values' memory).  "fp8:page"
    pages, whose scales are a page's rows together, take two launches, the keys rounded to their type between them.  Arguments
    as norm_rope's and write's."""
    if keys is None:
        raise ValueError("norm_rope_write stores keys (and values): pass keys")
    _cuda(q if q is not None else keys, "q")
    if values is not None and values.shape[:2] != keys.shape[:2]:
        raise ValueError(f"values are a row a token and kv head, like the keys' {list(keys.shape[:2])}, not {list(values.shape[:2])}")
    if values is not None and values.numel() and any(x is not None and x.data_ptr() == values.data_ptr() for x in (q_out, keys_out)):
        raise ValueError("an output in the values' place would be stored as the values: pass values of their own")
    if kind == "fp8:page":
        if keys.shape[0]:                      # (what write() would refuse, before the queries are turned)
            _append_params(keys, values, slots, key_pages, value_pages, kind, key_scales, value_scales, multipliers)
        found, turned = norm_rope(q, keys, positions, frequencies, q_weight=q_weight, key_weight=key_weight, eps=eps, offset=offset,
                                  axes=axes, interleaved=interleaved, magnitude=magnitude, q_out=q_out, keys_out=keys_out)
        write(turned, values, slots, key_pages, value_pages, kind, key_scales, value_scales, multipliers)
        return found
    p, reads, outs, copies = _norm_rope_params(q, keys, positions, frequencies, q_weight, key_weight, eps, offset, axes, interleaved,
                                               magnitude, q_out, keys_out, True)
    a, _held = _append_params(reads[1], None if values is None else _vectors(values), slots, key_pages, value_pages, kind, key_scales,
                              value_scales, multipliers)
    _launch_norm_rope(p, a, reads, copies, "crit_b200.norm_rope_write")
    return outs[0]


# -- gather and slots ---------------------------------------------------------------------------------------------------
def gather(pages, kind, page, *, table=None, slots=None, count=None, scales=None, multiplier=1.0, dtype=torch.bfloat16, out=None):
    """Rows of one page tensor ([pages][page][kv_heads][dim] or [slots][kv_heads][dim]; "int4": two elements a byte)
    dequantised to `dtype`: the first `count` positions of the page table `table` (int32), or the rows at `slots` (int64,
    any shape).  -> [count][kv_heads][dim] (or slots' shape + [kv_heads][dim]); into `out` (contiguous, of that size, its
    type in dtype's place) when given.  Reference: pages.py:455-493."""
    _cuda(pages, "pages")
    k_kind = _check_kind(kind, scales)
    hkv, dim = _check4(pages, scales, "rows") if k_kind == 5 else pages.shape[-2:]
    place = pages.get_device()
    if slots is not None:
        shape = (*slots.shape, hkv, dim)
        if slots.dim() != 1 or not slots.is_contiguous():
            slots = slots.reshape(-1).contiguous()
        count, listed = slots.numel(), slots
    elif table is None or count is None:
        raise ValueError("gather reads a page table's first `count` positions, or rows at `slots`")
    else:
        table = listed = table.contiguous()
        shape = (count, hkv, dim)
    if listed.get_device() != place:
        raise ValueError("gather's slots or page table are on the pages' device")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=pages.device)
    elif out.numel() != count * hkv * dim or not out.is_contiguous() or out.dtype not in _DTYPES or out.get_device() != place:
        raise ValueError(f"gather's out is a contiguous bf16, fp16 or fp32 tensor of [{count}][{hkv}][{dim}] on the pages' device")
    elif out.shape != shape:
        out = out.view(shape)
    if k_kind == 5 and (listed.dtype is not (torch.int32 if slots is None else torch.int64) or (slots is None and listed.numel() * page < count)):
        raise ValueError(f"int4 rows are read through an int32 page table that holds the {count} positions, or at int64 slots")
    if count == 0:
        return out
    if k_kind == 5 and out.data_ptr() % 16:            # (the kernel stores 16 bytes at once: made beside it)
        return out.copy_(gather(pages, kind, page, table=table, slots=slots, count=count, scales=scales, dtype=out.dtype).view(out.shape))
    if not pages.is_contiguous():
        raise ValueError("pages are contiguous [slots][kv_heads][dim] storage")
    p = _lib.block(_lib.GatherParams, pages.data_ptr(), _ptr(scales), _ptr(table), _ptr(slots), out.data_ptr(), _ptr(_status_word(pages.device)), count,
                   pages.numel() // (hkv * pages.shape[-1]), hkv, dim, int(page), k_kind, _page_dtype(kind, pages), _DTYPES[out.dtype], multiplier)
    _run("crit_b200_gather", "crit_b200.gather", pages.device, p)
    return out


def slots_at(tables, rows, positions, page, dump, capacity=None, out=None):
    """Each position's slot through its table row, on the device: tables [S][width] int32, rows and positions int64 of
    one shape; with capacity [S] int64 a position outside [0, capacity[row]) gets the dump page's first slot.
    Reference: pages.py:653-660."""
    _cuda(tables, "tables")
    shape = tuple(positions.shape)
    rows, positions = rows.reshape(-1).contiguous(), positions.reshape(-1).contiguous()
    if rows.dtype != torch.int64 or positions.dtype != torch.int64 or tables.dtype != torch.int32:
        raise ValueError("tables are int32, rows and positions int64")
    out = torch.empty(positions.numel(), dtype=torch.int64, device=tables.device) if out is None else out
    p = _lib.SlotsParams()
    p.tables, p.rows, p.positions, p.capacity, p.slots = _ptr(tables), _ptr(rows), _ptr(positions), _ptr(capacity), _ptr(out)
    p.n, p.table_stride, p.table_width = positions.numel(), tables.stride(0), tables.shape[1]
    p.page, p.dump = int(page), int(dump)
    _run("crit_b200_slots", "crit_b200.slots_at", tables.device, p)
    return out.view(shape)


def move_rows(store, source, target):
    """Rows of one store moved between slots, in place: store [layers][slots][...] (keys, values or their row scales),
    source / target [lists][width] int64 slots; for every list, in order j = 0 .. width - 1, the row at source[l][j] of
    every layer goes to target[l][j] (nothing where the two are equal).  A list's moves happen one after another; lists
    are independent.  What the pool's commit_round brings an accepted draft-tree path's KV together with
    (reference: inference/attention-state/code/pages.py:662-684)."""
    _cuda(store, "store")
    if not store.is_contiguous() or store.dim() < 2:
        raise ValueError("a store is contiguous [layers][slots][...]")
    if source.dtype != torch.int64 or target.dtype != torch.int64 or source.shape != target.shape or source.dim() != 2:
        raise ValueError("source and target are int64 [lists][width]")
    source, target = source.contiguous(), target.contiguous()
    layers, slots = store.shape[0], store.shape[1]
    row_bytes = store[0, 0].numel() * store.element_size()
    p = _lib.MoveParams()
    p.store, p.source, p.target = _ptr(store), _ptr(source), _ptr(target)
    p.lists, p.width, p.slots, p.row_bytes, p.layers = source.shape[0], source.shape[1], slots, row_bytes, layers
    p.status = _ptr(_status_word(store.device))
    _run("crit_b200_move_rows", "crit_b200.move_rows", store.device, p)


def _listed_rows(tables, rows, starts, counts, firsts, blocks, block_size, page, columns, out, lse):
    """Block lists as page tables of their own (crit_b200_compact_blocks): (tables, rows, starts, firsts, counts) of
    one-column rows, a row a token, whose tables hold the pages of the token's listed blocks only; tokens that see
    nothing get zeros in out (and -inf in lse) here."""
    device = tables.device
    R = int(starts.shape[0])
    n, per = R * columns, block_size // page
    t2 = torch.empty(n, blocks.shape[1] * per, dtype=torch.int32, device=device)
    c2 = torch.empty(n, dtype=torch.int32, device=device)
    f2 = torch.empty(n, dtype=torch.int64, device=device)
    p = _lib.CompactParams()
    p.tables, p.rows, p.starts, p.counts, p.firsts, p.blocks = (_ptr(x) for x in (tables, rows, starts, counts, firsts, blocks))
    p.out_tables, p.out_counts, p.out_firsts, p.out, p.lse = _ptr(t2), _ptr(c2), _ptr(f2), _ptr(out), _ptr(lse)
    p.n_rows, p.table_stride, p.table_width = R, tables.stride(0), tables.shape[1]
    p.out_stride_token, p.out_stride_head = out.stride(0), out.stride(1)
    p.columns, p.blocks_k, p.block_size, p.page = columns, blocks.shape[1], block_size, page
    p.dump = 0              # (entries past a row's listed pages are never read: its last position ends before them)
    p.q_heads, p.value_dim, p.out_dtype = out.shape[1], out.shape[2], _DTYPES[out.dtype]
    _run("crit_b200_compact_blocks", "crit_b200.attend (block lists)", device, p)
    tokens = (starts[:, None] + torch.arange(columns, dtype=torch.int32, device=device)[None, :]).reshape(-1).contiguous()
    return t2, torch.arange(n, dtype=torch.int32, device=device), tokens, f2, c2


# -- decode and verify windows ------------------------------------------------------------------------------------------
def _refuse(**given):
    asked = [name for name, value in given.items()
             if value is not None and value is not False and not (isinstance(value, int) and value == 0)]
    if asked:
        raise NotImplementedError(f"crit_b200.attend does not serve {', '.join(asked)} yet: causal windows over the "
                                  "whole context only")


def attend(q, key_pages, value_pages, kind, tables, rows, starts, firsts, columns, page, *, counts=None,
           offsets=None, tokens=None, key_scales=None, value_scales=None, multipliers=(1.0, 1.0), scale=None,
           partitions=None, parents=None, blocks=None, block_size=None, out=None, lse=None, workspace=None, piece=None,
           fused=False, fresh=None, vsplit=None, tile=None, num_warps=None, num_stages=None, maxnreg=None,
           flash=False, chunk=None, ramp=None, sinks=None, sliding=0, derive=None, launch="both", staging=None,
           persistent=False, engine=None, shards=None, context=False):
    """Decode and verify windows over paged KV (reference: paged_kv_attention/__init__.py:396-445, same arguments).

    q [tokens][heads][dim] bf16 or fp16 (fp16 for "fp16" pages); key_pages / value_pages one layer's pages
    ([pages][page][kv_heads][dim]), key_scales / value_scales their scales; tables [S][width] int32; rows [R] int32 the
    table row of each batch row; starts [R] int32 its first token in q; firsts [R] int64 its column 0's position;
    counts [R] int32 its columns (None: `columns` each; more read as `columns`); columns the widest row (<= 64).
    offsets [R] int32 and tokens: each row's first partial row and the partial rows the launch takes.  Writes
    out [tokens][heads][value_dim] (q's dtype) at the rows' tokens and lse [tokens][heads] FP32 when given; returns out.
    chunk: positions per split (default chunk_for()); partitions: the most splits a partial row may take (the
    workspace's, see partitions()).  piece, fused, vsplit, tile, num_warps, num_stages, maxnreg, flash and ramp are
    accepted and change nothing (one launch shape per geometry).  parents [tokens]: each token's parent column in its
    row, -1 for none (a draft tree in topological order): a column then sees the context before its row's first position,
    itself and its ancestors.  sinks [heads] FP32: a logit a query head that joins the softmax's maximum and sum (and
    the lse) without a value; sliding: the positions a column sees up to its own, 0 for all (all three on the m16n8k16
    kernel).  blocks [tokens][k] int32 with block_size: the KV blocks (block_size positions each, -1 for none) a token
    sees.  Where block_size is a multiple of the page (and no tree, sink or sliding window is asked for) the launch
    reads the listed blocks only: every token becomes a one-column row over a page table of its blocks, built on the
    device, on whichever kernel serves it; otherwise the lists are a mask over the m16n8k16 kernel's tiles (every
    position is read).  context: every column of a row sees the positions before firsts[r] and none from there on (the
    part of a prompt chunk's attention that reads the pages when its own keys and values are read fresh; an extension
    of this module).  fresh (the reference's in-kernel fresh rows) and derive are not served: DeviceAttention reads a
    pool's fresh rows as context rows + a prefill over the fresh chunk + merge_shards.  launch: "both", or "decode" / "merge" alone (a measurement's).  staging: how pages reach shared memory:
    None (TMA tiled loads for 16-bit pages of 128- or 256-wide heads, cp.async otherwise: what measured faster), "tma"
    (TMA wherever the geometry allows it) or "cp.async" (never TMA); the same bits either way.  persistent: a fixed
    number of blocks walk a work list built on the device from the rows' lengths, instead of one block per (split, kv
    head, row) of a 3-D grid (the same bits; measured slower on the bench workloads, hence off).  engine: None (the
    library's choice), "mma.sync" (the m16n8k16 kernel), "even" (int4 pages: no splits, the launch's positions dealt out
    evenly; the choice for them where the caller names no chunk, partitions or workspace) or "tcgen05" (E4M3 page bytes straight into tcgen05.mma: E4M3
    pages of 128-wide heads, columns x group heads <= 32, chunk a multiple of 128; refused elsewhere).
    shards: a crit_b200.dist.ShardMerge: these pages hold one KV range of a context sharded over the ranks; every
    split state stays in the workspace, the fold of this rank's splits is stored into every rank's exchange buffer and
    out / lse get the merge over all ranks (three launches: decode, fold + push, wait + merge).
    workspace: the states' (FP32; else the owner's): launches that may run at the same time, on two streams or as two graphs,
    take one each (`owner`).  "int4" pages: nothing is read past the tables' width; of a row that ends there the columns past it
    see the table's positions, a row that begins past it is reported (status) and, evenly, left out."""
    _refuse(fresh=fresh, derive=derive)
    # masks are served by the m16n8k16 kernels: of 4-bit pages under either engine, else "mma.sync"
    plain = (None, "mma.sync", "even") if kind == "int4" else (None, "mma.sync")
    masked = engine if kind == "int4" else "mma.sync"
    if context and (parents is not None or blocks is not None or sinks is not None or sliding or shards is not None or
                    engine not in plain):
        raise NotImplementedError("context rows (every column sees the positions before its row's first only) are the "
                                  "m16n8k16 kernel's plain rows")
    k_kind = _check_kind(kind, key_scales)
    _cuda(q, "q")
    T, hq, d = q.shape
    hkv, dv, place = key_pages.shape[-2], value_pages.shape[-1], q.get_device()
    if k_kind == 5:
        if value_scales is None:
            raise ValueError("int4 pages take scales beside their codes, keys and values alike")
        if _check4(key_pages, key_scales, "keys") != (hkv, d) or _check4(value_pages, value_scales, "values") != (hkv, d):
            raise ValueError(f"int4 pages hold keys and values of q's width, [...][kv_heads][{d // 2}]")
        if key_pages.numel() != value_pages.numel() or key_pages.get_device() != place or value_pages.get_device() != place:
            raise ValueError("int4 keys and values are as many pages each, on q's device")
        dv = d
    R = int(starts.shape[0])
    if hq % hkv or not 1 <= columns <= MAX_COLUMNS or R == 0:
        raise ValueError("query heads a multiple of the KV heads, 1..64 columns a row, one row or more")
    (q_token, q_head, q_element), q_dtype = q.stride(), q.dtype
    if q_element != 1:
        raise ValueError("q's last dimension is contiguous")
    if q_dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q is bf16 or fp16")
    if (offsets is None) != (tokens is None):
        raise ValueError("offsets come with the partial rows they take (tokens)")
    if k_kind == 5:
        for x in (tables, rows, starts, firsts, counts, offsets, out, lse):
            if x is not None and x.get_device() != place:
                raise ValueError("attend's tensors are on q's device")
        for x in (rows, starts, firsts, counts, offsets):
            if x is not None and (x.numel() < R or not x.is_contiguous()):
                raise ValueError(f"rows, starts, firsts, counts and offsets are contiguous, an entry each of the {R} rows")
        if workspace is not None and workspace.get_device() != place:
            raise ValueError("attend's workspace is on q's device")
        if (counts is not None and counts.dtype is not torch.int32) or (offsets is not None and offsets.dtype is not torch.int32):
            raise ValueError("counts and offsets are int32")
        if out is not None and out.shape != q.shape:
            raise ValueError(f"out is [{T}][{hq}][{d}], as q")
    if tables.dtype != torch.int32 or tables.stride(-1) != 1 or rows.dtype != torch.int32 or \
            starts.dtype != torch.int32 or firsts.dtype != torch.int64:
        raise ValueError("tables, rows and starts are int32, firsts int64")
    page = int(page)
    if page % TILE:
        raise ValueError(f"crit_b200 reads pages of a multiple of {TILE} positions, not {page}")
    if k_kind != 5 and (not key_pages.is_contiguous() or not value_pages.is_contiguous()):       # (int4: checked above)
        raise ValueError("pages are contiguous [slots][kv_heads][dim] storage")
    device = q.device
    positions = tables.shape[1] * page
    if parents is not None:
        # a draft tree: parents [tokens] is each token's parent column in its row, -1 for none (topological order)
        if engine not in plain:
            raise NotImplementedError("draft trees (parents) are served by the m16n8k16 kernel: engine None or mma.sync")
        parents = parents.reshape(-1)
        if parents.dtype not in (torch.int32, torch.int64) or parents.numel() != T:
            raise ValueError("parents are int32 or int64, one per token of q")
        parents = _cuda(parents, "parents").to(torch.int32).contiguous()
        engine = masked
    if blocks is not None:
        # block lists: blocks [tokens][k] KV block ids (-1 for none) of block_size positions: a token sees only those
        if blocks.dim() != 2 or blocks.shape[0] != T or not block_size or int(block_size) < 1:
            raise ValueError("blocks are [tokens][k] block ids, with the positions a block holds (block_size)")
        blocks = _cuda(blocks, "blocks").to(torch.int32).contiguous()
        if (int(block_size) % page == 0 and parents is None and sinks is None and not sliding and offsets is None and
                shards is None and launch == "both" and not torch.cuda.is_current_stream_capturing()):
            # the sparse reader: every token becomes a row of one column over a page table of its listed blocks only
            # (built on the device), so the launch reads those blocks and nothing else, on whichever kernel serves it
            out = torch.empty(T, hq, dv, dtype=q.dtype, device=q.device) if out is None else out
            listed = _listed_rows(tables, rows, starts, counts, firsts, blocks, int(block_size), page, int(columns), out, lse)
            if engine in _LISTED_ROWS and listed[2].numel() > _LISTED_ROWS[engine]:
                engine = "mma.sync"           # (named for the caller's rows; the tokens are more than it lists)
            return attend(q, key_pages, value_pages, kind, listed[0], listed[1], listed[2], listed[3], 1, page,
                          counts=listed[4], key_scales=key_scales, value_scales=value_scales, multipliers=multipliers,
                          scale=scale, partitions=partitions, out=out, lse=lse, workspace=workspace, chunk=chunk,
                          engine=engine)
        if engine not in plain:
            raise NotImplementedError("block lists of blocks that are no multiple of the page, or with a tree, sinks or a "
                                      "sliding window, are a mask of the m16n8k16 kernel: engine None or mma.sync")
        engine = masked             # as a mask over the m16n8k16 kernel's tiles: every position is read
    sliding = int(sliding or 0)
    if sinks is not None or sliding:
        # a sink logit a query head (joins the softmax's maximum and sum, and the lse, in the fold of the splits), and a
        # window of the `sliding` positions up to a column's own: the m16n8k16 kernel's
        if engine not in plain:
            raise NotImplementedError("sinks and sliding windows are served by the m16n8k16 kernel: engine None or mma.sync")
        if shards is not None and sinks is not None:
            raise NotImplementedError("a sharded context's merge does not take sinks")
        if sliding < 0:
            raise ValueError("sliding is the number of positions a column sees, 0 for all")
        if sinks is not None:
            sinks = _cuda(sinks, "sinks").reshape(-1)
            if sinks.numel() != hq:
                raise ValueError(f"sinks are one logit a query head ({hq}), not {sinks.numel()}")
            sinks = sinks.float().contiguous()
        engine = masked
    if context:
        engine = masked
    chosen = engine is None
    if chosen and (shards is not None or persistent or staging is not None):
        engine = "mma.sync"               # what those arguments are about
    if chosen and k_kind == 5 and (chunk or partitions or offsets is not None or workspace is not None):
        engine = "mma.sync"               # the caller cuts the launch itself
    engine = engine_for(kind, d, dv, hq, hkv, int(columns), R, positions, engine)
    chunk = int(chunk or chunk_for(d, dv, hq, hkv, page, kind, engine, int(columns)))
    if partitions:
        chunk = max(chunk, -(-positions // int(partitions)))
    chunk = -(-chunk // TILE) * TILE
    if chosen and ((engine == "tcgen05p" and not tcgen05p_serves(kind, d, dv, hq, hkv, int(columns), chunk, R)) or
                   (engine == "tcgen05" and not tcgen05_serves(kind, d, dv, hq, hkv, int(columns), chunk, R))):
        engine = "mma.sync"               # the caller's chunk is not one the chosen kernel takes
    splits = states_for(parts_for(positions, chunk), engine)
    partial_rows = R * columns if offsets is None else int(tokens)
    if out is None:
        out = _like(q) if dv == d else torch.empty(T, hq, dv, dtype=q_dtype, device=device)
    (out_token, out_head, out_element) = out.stride()
    if out.dtype != q_dtype or out_element != 1:
        raise ValueError("out is in q's dtype, its last dimension contiguous")
    if engine == "even" and k_kind != 5:
        raise NotImplementedError("the even engine reads int4 pages")
    if lse is not None and (lse.dtype != torch.float32 or not lse.is_contiguous() or lse.shape != (T, hq)):
        raise ValueError(f"lse is contiguous FP32 [{T}][{hq}]")
    if staging not in (None, "tma", "cp.async"):
        raise ValueError("staging is None, tma or cp.async")
    space = None
    if engine != "even" and (splits > 1 or shards is not None or sinks is not None):
        space = _workspace(device, workspace_floats(partial_rows, hq, splits, dv), workspace)
    columns = int(columns)
    flags = (_STAGINGS[staging] | (4 if persistent else 0) | _ENGINES[engine] | (32 if shards is not None else 0) | (256 if context else 0))
    p = _lib.block(_lib.AttendParams, q.data_ptr(), out.data_ptr(), _ptr(lse), key_pages.data_ptr(), value_pages.data_ptr(), _ptr(key_scales), _ptr(value_scales),
                   tables.data_ptr(), rows.data_ptr(), starts.data_ptr(), _ptr(counts), firsts.data_ptr(), _ptr(offsets), _ptr(space), _ptr(_status_word(device)),
                   space.numel() if space is not None else 0, key_pages.numel() * (2 if k_kind == 5 else 1) // (hkv * d), q_token, q_head,
                   out_token, out_head, tables.stride(0), R, columns, partial_rows, hq, hkv, d, dv, page, k_kind,
                   _page_dtype(kind, key_pages), _DTYPES[q_dtype], chunk, splits, flags, float(scale if scale is not None else d ** -0.5),
                   float(multipliers[0]), float(multipliers[1]), _ptr(parents), _ptr(sinks), sliding,
                   blocks.shape[1] if blocks is not None else 0, int(block_size) if blocks is not None else 0, tables.shape[1] if k_kind == 5 else 0,
                   _ptr(blocks))
    lib = _lib.load()
    if engine == "even":
        key = (place, R, columns, hq, hkv, d, q_dtype, parents is not None or sliding > 0 or blocks is not None)
        floats = _even_floats.get(key)
        if floats is None:
            with torch.cuda.device(device):
                floats = lib.crit_b200_attend_floats(ctypes.byref(p))
            if floats < 0:
                _lib.check(floats, "crit_b200.attend")
            _even_floats[key] = floats
        space = _workspace(device, floats, workspace)
        p.workspace, p.workspace_floats = _ptr(space), space.numel()
    if shards is not None:
        if lse is None:
            raise ValueError("a sharded context's merge writes lse too: pass lse")
        with torch.cuda.device(device):
            if launch in ("both", "decode", "push"):
                _run("crit_b200_decode", "crit_b200.attend", device, p)
            if launch in ("both", "merge"):
                shards.attend(p, out, lse)
            elif launch == "push":             # decode and fold + push, no wait: a measurement's
                shards.attend(p, out, lse, wait=False)
        return out
    _run({"both": "crit_b200_attend", "decode": "crit_b200_decode", "merge": "crit_b200_merge"}[launch], "crit_b200.attend", device, p)
    return out


def merge_shards(outs, lses, dtype=None):
    """Partials of the same queries over disjoint keys (outs [parts][tokens][heads][dim], lses [parts][tokens][heads]
    FP32, -inf for a part with no key) -> (out [tokens][heads][dim], lse): the parts weighted by exp(lse - max); a
    token no part saw gets zeros and -inf.  Reference: inference/partitioned-attention/plugin.py:52-64."""
    if not torch.is_tensor(outs):
        outs = torch.stack(list(outs))
    if not torch.is_tensor(lses):
        lses = torch.stack(list(lses))
    _cuda(outs, "outs")
    outs, lses = outs.contiguous(), lses.float().contiguous()
    if outs.dtype not in _DTYPES:
        outs = outs.float()
    parts, dim = outs.shape[0], outs.shape[-1]
    n = lses[0].numel()
    dtype = dtype or torch.float32
    out = torch.empty(outs.shape[1:], dtype=dtype, device=outs.device)
    lse = torch.empty(lses.shape[1:], dtype=torch.float32, device=outs.device)
    p = _lib.MergeShardsParams()
    p.outs, p.lses, p.out, p.lse = _ptr(outs), _ptr(lses), _ptr(out), _ptr(lse)
    p.n, p.parts, p.dim, p.in_dtype, p.out_dtype = n, parts, dim, _DTYPES[outs.dtype], _DTYPES[dtype]
    _run("crit_b200_merge_shards", "crit_b200.merge_shards", outs.device, p)
    return out, lse


def prefill_serves(head_dim, value_dim, q_dtype, kind, page):
    """Whether prefill() reads a cache of this geometry (else prompt rows go through attend in pieces)."""
    widths = (64, 128, 256) if kind in ("bf16", "fp16", "int4") else (64, 128)        # 256-wide heads: 16-bit pages (m16n8k16 tiles)
    return head_dim == value_dim and head_dim in widths and page % TILE == 0 and kind in KINDS and \
        q_dtype in (torch.bfloat16, torch.float16)


# -- prompt chunks ------------------------------------------------------------------------------------------------------
def _expansion(device, size, given, steady):
    """`size` bytes for a prompt launch's own use (16-byte aligned): `given`, or memory of the launch's stream that goes back to
    torch's allocator when the call returns.  steady: calls of this size repeat; else a prompt grows chunk by chunk, and sizes of
    powers of two are few, so that the allocator's blocks are found again."""
    if given is not None:
        if given.dtype != torch.float32 or 4 * given.numel() < size or not given.is_contiguous() or given.device != device:
            raise ValueError(f"prefill's workspace holds {given.numel()} floats; this launch needs {-(-size // 4)} contiguous FP32 ones on q's device")
        return given
    if not steady and not torch.cuda.is_current_stream_capturing():
        try:
            return torch.empty(1 << max(size - 1, 15).bit_length(), dtype=torch.uint8, device=device)
        except torch.OutOfMemoryError:
            pass
    return torch.empty(max(size, 16), dtype=torch.uint8, device=device)


def _expanded(q, key_pages, value_pages, key_scales, value_scales, table, position, ahead, starts, tokens, taken, width, page, workspace):
    """4-bit pages as 16-bit ones of q's type in memory of the launch's own, one launch: (that memory, the addresses of the keys,
    the values, the table that reads them, the positions and the starts, the slots of the pages).  taken: the pages of each
    sequence, one sequence's after another's, where the host knows; None: positions on the device, room for every page that the
    tables (of `width`) may name, or for the pool's where those are fewer."""
    hkv, d = key_pages.shape[-2], q.shape[-1]
    place = q.get_device()
    if value_scales is None or _check4(key_pages, key_scales, "keys") != (hkv, d) or _check4(value_pages, value_scales, "values") != (hkv, d) or \
            key_pages.numel() != value_pages.numel() or key_pages.get_device() != place or value_pages.get_device() != place or table.get_device() != place:
        raise ValueError(f"int4 pages hold keys and values of q's width, [...][kv_heads][{d // 2}] with their scales, on q's device")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q is bf16 or fp16")
    several = table.dim() == 2
    sequences, slots = table.shape[0] if several else 1, key_pages.numel() * 2 // (hkv * d)
    keep_ids = taken is None and slots // page < sequences * width
    pages = sum(taken) if taken is not None else slots // page if keep_ids else sequences * width
    bases = [0, *itertools.accumulate(taken)][:sequences] if several and taken is not None else []
    numbers, ints = _packed(ahead, (starts or []) + bases)
    side = pages * page * hkv * d * 2                                  # bytes of the keys, or the values
    read = taken is None                                               # (positions that the device reads)
    held = _expansion(q.device, 2 * side + 8 * len(numbers) + 8 * read * sequences + 4 * sequences * width, workspace, read)
    keys = held.data_ptr()
    sent = keys + 2 * side                                             # the lists; the positions read, brought within the tables; the table
    found = sent + 8 * len(numbers)
    if numbers:
        _send(numbers, sent, q.device)
    starts_at, bases_at = sent + 8 * ints if starts else 0, sent + 8 * ints + 4 * len(starts or ()) if bases else 0
    said, at = (position.data_ptr(), found) if read else (sent, sent) if ahead else (0, 0)
    tables_at = found + 8 * read * sequences
    e = _lib.block(_lib.ExpandParams, key_pages.data_ptr(), value_pages.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), table.data_ptr(),
                   said, starts_at, bases_at, keys, keys + side, tables_at, found if read else 0, _ptr(_status_word(q.device)), 0 if said else int(position),
                   slots, table.stride(0) if several else 0, sequences, width, tokens, hkv, d, page, _DTYPES[q.dtype], keep_ids)
    _run("crit_b200_expand", "crit_b200.prefill", q.device, e)
    return held, keys, keys + side, tables_at, at, starts_at, pages * page


def _pages_of(positions, ends, tokens, width, page):
    """The pages of tables of `width` that the sequences of a prompt launch over 4-bit pages take, or None: positions on the
    device.  What lies outside the tables is refused here."""
    longest = tokens if positions is None else max(ends, default=0)
    if longest > width * page:
        raise ValueError(f"a chunk's positions go up to {longest}; its page table holds {width * page}")
    if positions is None:
        return None
    if min(positions, default=0) < 0:
        raise ValueError("positions are not negative")
    return [-(-end // page) for end in ends]


def _packed(positions, ints):
    """Lists of positions (int64; None: none) and of int32 numbers as int64 ones: (them, where the int32 ones begin)."""
    numbers, odd = list(positions or ()), list(ints or ())
    if len(odd) % 2:
        odd.append(0)
    return numbers + [a | b << 32 for a, b in zip(odd[::2], odd[1::2])], len(numbers)


def _send(numbers, to, device):
    """Numbers to the device as a small kernel's parameters, which wait for nothing and which a capture keeps; a copy would leave
    a captured graph with the address of memory that is gone."""
    _run("crit_b200_put", "crit_b200.prefill", device, to, struct.pack(f"{len(numbers)}q", *numbers), len(numbers))


def prefill(q, key_pages, value_pages, kind, table, position, page, *, key_scales=None, value_scales=None,
            multipliers=(1.0, 1.0), scale=None, out=None, lse=None, int8_qk=False, fresh=None, flash=False,
            sinks=None, sliding=0, splits=None, workspace=None, derive=None, engine=None, starts=None):
    """A prompt chunk of one sequence: q [T][heads][dim] at positions position.. (their keys and values written),
    table [pages] int32 (or int64) -> out [T][heads][dim] in q's dtype (and lse [T][heads] FP32 when given), causal.  position: an
    int, or a one-element int64 device tensor read on the device.  Several sequences' chunks in ONE launch: table
    [S][pages], position a list of S ints or an int64 device tensor [S], q the sequences' tokens one after another
    (equal counts, or `starts`: S + 1 ints, sequence s's tokens being rows starts[s]..starts[s+1]).  engine: None
    (tcgen05.mma tiles with TMEM accumulators for 16-bit pages of 128-wide heads, m16n8k16 tiles otherwise), "mma.sync"
    or "tcgen05" (refused where not served); "tcgen05:single" / "tcgen05:pair" also name the block shape (128 query rows
    two blocks an SM / 256 rows over one ring of key and value tiles, which "tcgen05" picks by the launch's size).  The
    softmax's weights are rounded to q's type for the second product, their sum is not.
    "int4" pages are first made 16-bit ones of q's type (exact: no second rounding) in memory of the launch's own: the sequences'
    positions * kv_heads * dim * 4 bytes (with positions on the device those that the tables or the pool hold, whichever are
    fewer) and a few, of the current stream and given back when the call returns (a capture keeps its own), or `workspace` (FP32,
    read and written until the launch is through: not for two launches at once).
    Reference: paged_kv_attention/__init__.py:1245-1332."""
    _refuse(int8_qk=int8_qk, fresh=fresh, sinks=sinks, sliding=sliding, derive=derive)
    k_kind = _check_kind(kind, key_scales)
    _cuda(q, "q")
    T, hq, d = q.shape
    hkv = key_pages.shape[-2]
    if value_pages.shape[-1] * (2 if k_kind == 5 else 1) != d:
        raise ValueError("prompt chunks read keys and values of one width")
    if not key_pages.is_contiguous() or not value_pages.is_contiguous():
        raise ValueError("pages are contiguous [slots][kv_heads][dim] storage")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != q.get_device():
        raise ValueError(f"out is [{T}][{hq}][{d}] in q's dtype, on its device")
    if table.dtype not in (torch.int32, torch.int64) or table.dim() not in (1, 2):
        raise ValueError("table is the sequence's page ids, int32 (read in place) or int64 (converted)")
    if table.dtype != torch.int32 or not table.is_contiguous():
        table = table.to(torch.int32).contiguous()       # (the reference's pool hands its tables over as int64 slices)
    if q.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError("q and out have contiguous last dimensions")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (T, hq) or not lse.is_contiguous() or lse.get_device() != q.get_device()):
        raise ValueError(f"lse is contiguous FP32 [{T}][{hq}] on q's device")
    positions_at = starts_at = sequences = table_stride = 0
    if k_kind == 5 and torch.is_tensor(position) and position.get_device() != q.get_device():
        raise ValueError("positions read on the device are on q's device")
    ahead = held = None                                # (held: kept until every launch is made)
    if table.dim() == 2:             # several sequences, one launch
        S = table.shape[0]
        if not torch.is_tensor(position):
            if len(position) != S:
                raise ValueError("one position a sequence")
            ahead = [int(x) for x in position]
        elif position.dtype != torch.int64 or position.numel() != S or not position.is_cuda or not position.is_contiguous():
            raise ValueError("the sequences' positions are an int64 tensor [S] on the device")
        if starts is None:
            if T % S:
                raise ValueError("sequences of unequal token counts give `starts`")
            most = T // S
            counts = [most] * S
        else:
            starts = [int(x) for x in starts]
            if len(starts) != S + 1 or starts[0] != 0 or starts[-1] != T or any(b < a for a, b in zip(starts, starts[1:])):
                raise ValueError("starts: S + 1 rising row numbers from 0 to the number of tokens")
            counts = [b - a for a, b in zip(starts, starts[1:])]
            most = max(counts)
        if k_kind == 5:
            taken = _pages_of(ahead, None if ahead is None else [a + n for a, n in zip(ahead, counts)], most, table.shape[1], int(page))
        else:
            positions_at = position.data_ptr() if ahead is None else 0
            numbers, ints = _packed(ahead, starts)
            if numbers:
                held = torch.empty(len(numbers), dtype=torch.int64, device=q.device)
                at = held.data_ptr()
                _send(numbers, at, q.device)
                positions_at, starts_at = positions_at or at, at + 8 * ints if starts else 0
        sequences, table_stride, T = S, table.stride(0), most
        if ahead is not None:
            position = 0
    elif starts is not None:
        raise ValueError("starts goes with a table of several sequences")
    if not sequences and torch.is_tensor(position) and (position.dtype != torch.int64 or position.numel() != 1 or not position.is_cuda):
        raise ValueError("a position read on the device is a one-element int64 tensor there")
    page, q_code = int(page), _DTYPES[q.dtype]
    if k_kind == 5:
        if not sequences:
            taken = _pages_of(*((None, None) if torch.is_tensor(position) else ([int(position)], [int(position) + T])), T, table.shape[0], page)
        width = max(taken, default=0) if taken is not None else table.shape[-1]
        held, keys_at, values_at, table_at, at, starts_at, slots = _expanded(q, key_pages, value_pages, key_scales, value_scales, table, position, ahead, starts, T,
                                                                             taken, width, page, workspace)
        key_scales = value_scales = None
        table_stride, k_kind, page_dtype = width if sequences else 0, 0, q_code
        if sequences:
            positions_at = at
    else:
        keys_at, values_at, table_at, slots = key_pages.data_ptr(), value_pages.data_ptr(), table.data_ptr(), key_pages.numel() // (hkv * d)
        page_dtype = _page_dtype(kind, key_pages)
    device = q.device
    position_at = 0
    if sequences:
        position = 0
    elif torch.is_tensor(position):
        position_at, position = at if kind == "int4" else position.data_ptr(), 0
    q_token, q_head, _ = q.stride()
    out_token, out_head, _ = out.stride()
    p = _lib.block(_lib.PrefillParams, q.data_ptr(), out.data_ptr(), _ptr(lse), keys_at, values_at, _ptr(key_scales), _ptr(value_scales), table_at, position_at,
                   _ptr(_status_word(device)), int(position), slots, q_token, q_head, out_token, out_head, T, hq, hkv, d, d, page, k_kind, page_dtype, q_code,
                   _PREFILL_ENGINES[engine], float(scale if scale is not None else d ** -0.5), float(multipliers[0]), float(multipliers[1]),
                   starts_at, positions_at, sequences, table_stride)
    _run("crit_b200_prefill", "crit_b200.prefill", device, p)
    return out
