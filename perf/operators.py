"""Operators of a 4-bit paged KV cache, measured: writing and reading back "int4" pages, decode / verify windows and prompt
chunks over them, and the per-head norm + rotary step in front of the cache (alone, and fused with the write).

A case is a dict of plain values.  prepare() makes its inputs on the GPU from a seed; run() makes one pass: in plain torch
operations in 32 bits (own False) or through crit_b200's entry points (own True); exact() gives the same outputs from the
definitions in 64 bits.

The 4-bit page format ("int4"): a row of one kv head is `dim` codes of 4 bits, element 2 i in the low half of byte i and
element 2 i + 1 in the high half, and one byte of scale for each group of 32 elements (scales [...][kv_heads][dim / 32]).
The byte is an unsigned float of 5 exponent and 3 mantissa bits, the top byte of an FP16 number shifted left by one: 61,440 at
most, steps of 2^-17 below 2^-14.  scale = max |x| / 7 rounded to such a number, code = 8 + round(x / scale) within 1..15 (8
where the scale is 0), and the value a code stands for is (code - 8) * scale: no more than 8 significant bits, so 16-bit
types hold it as it is.
"""
import math
import random

import torch

own = False

GROUP = 32
EPS = 1e-6


# -- the cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the keys and values of one decode step of 64 sequences, quantised into their pages and read back
        dict(name="write decode step of 64", op="write", tokens=64, kv_heads=8, dim=128, page=16, dtype="bf16", scattered=True),
        # a prompt chunk of four sequences going into the cache
        dict(name="write prompt 4 x 2,048", op="write", tokens=8192, kv_heads=8, dim=128, page=16, dtype="bf16", scattered=False),
        # the decode step of a full batch: the repository's FP8 decode geometry over 4-bit pages
        dict(name="attend 64 x 4,096", op="attend", rows=64, columns=1, q_heads=64, kv_heads=8, dim=128, page=16, shortest=4096,
             longest=4096, middle=4096, dtype="bf16", lengths=1),
        # one user, a short conversation: latency
        dict(name="attend 1 x 777", op="attend", rows=1, columns=1, q_heads=32, kv_heads=8, dim=128, page=16, shortest=777,
             longest=777, middle=777, dtype="bf16", lengths=1),
        # one very long context of 256-wide heads
        dict(name="attend 1 x 200,000", op="attend", rows=1, columns=1, q_heads=24, kv_heads=4, dim=256, page=64,
             shortest=200000, longest=200000, middle=200000, dtype="bf16", lengths=1),
        # speculative verify windows of 6 drafts over contexts of very different lengths
        dict(name="attend verify 32 x 6 ragged", op="attend", rows=32, columns=6, q_heads=40, kv_heads=8, dim=128, page=16,
             shortest=512, longest=16384, middle=4096, dtype="fp16", lengths=5),
        # a prompt chunk behind a long prefix
        dict(name="prefill 2,048 at 32,768", op="prefill", sequences=1, tokens=2048, even=True, q_heads=32, kv_heads=8, dim=128,
             page=16, prefix=32768, dtype="bf16", lengths=1),
        # short prompts of different lengths in one launch
        dict(name="prefill ragged 420", op="prefill", sequences=3, tokens=420, even=False, q_heads=32, kv_heads=8, dim=128, page=16,
             prefix=700, dtype="bf16", lengths=3),
        # the queries and keys of a decode step: norm of each head and rotation
        dict(name="norm_rope decode step of 64", op="norm_rope", tokens=64, q_heads=64, kv_heads=8, dim=128, rotary=128, axes=1,
             norm=True, interleaved=False, far=65536, dtype="bf16"),
        # a prompt with images: positions of three axes (time, height, width)
        dict(name="norm_rope prompt 8,192, 3 axes", op="norm_rope", tokens=8192, q_heads=32, kv_heads=8, dim=128, rotary=128, axes=3,
             norm=True, interleaved=False, far=200000, dtype="bf16"),
        # a decode step's norm and rotation with the keys and values quantised into their pages in the same pass
        dict(name="norm_rope_write step of 64", op="norm_rope_write", tokens=64, q_heads=64, kv_heads=8, dim=128, rotary=128, axes=1,
             norm=True, interleaved=False, far=65536, page=16, dtype="bf16", scattered=True),
        # the same for a prompt chunk of four sequences
        dict(name="norm_rope_write prompt 8,192", op="norm_rope_write", tokens=8192, q_heads=32, kv_heads=8, dim=128, rotary=128,
             axes=1, norm=True, interleaved=False, far=200000, page=16, dtype="bf16", scattered=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "prefill", "norm_rope", "norm_rope_write"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 4, 5, 6, 8])
    page = rng.choice([16, 32, 64])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "write":
        return dict(op=op, tokens=_log(rng, 1, 8192), kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, scattered=rng.random() < 0.5)
    if op == "attend":
        rows, columns = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 6])
        # positions in all: at most the long context's 4 heads of 256, and at most 16,384 a row where there are many rows
        most = max(64, min(200000 * 1024 // (kv_heads * dim * rows), 200000 if rows == 1 else 16384))
        longest = _log(rng, 33, most)
        shortest = rng.choice([longest, max(1, longest // 20)])
        return dict(op=op, rows=rows, columns=columns, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                    shortest=shortest, longest=longest, middle=max(shortest, longest // 3), dtype=dtype, lengths=rng.randrange(1 << 20))
    if op == "prefill":
        sequences = rng.choice([1, 1, 2, 3])
        tokens = _log(rng, 17 * sequences, 2048)
        prefix = rng.choice([0, _log(rng, 16, 32768 // sequences)])
        # heads x dim x tokens x positions: at most a quarter of the listed prompt's
        while kv_heads * group * dim * tokens * (prefix + tokens) > 32 * 128 * 2048 * 34816 // 4:
            prefix, tokens = prefix // 2, max(17 * sequences, tokens * 3 // 4)
        return dict(op=op, sequences=sequences, tokens=tokens, even=sequences == 1, q_heads=kv_heads * group, kv_heads=kv_heads,
                    dim=dim, page=page, prefix=prefix, dtype=dtype, lengths=rng.randrange(1 << 20))
    case = dict(op=op, tokens=_log(rng, 1, 8192 * 32 // max(32, kv_heads * group)), q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                rotary=rng.choice([dim, dim, dim // 2]), axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.8,
                interleaved=rng.random() < 0.3, far=rng.choice([4096, 65536, 1000000]), dtype=dtype)
    if op == "norm_rope_write":
        case.update(page=page, scattered=rng.random() < 0.5)
    return case


def _contexts(case):
    """The attention rows' context lengths (positions before and with column 0), the same for every seed."""
    r = random.Random(case["lengths"])
    if case["shortest"] == case["longest"]:
        return [case["longest"]] * case["rows"]
    return [min(case["longest"], max(case["shortest"], int(round(r.lognormvariate(math.log(case["middle"]), 1.0))))) for _ in range(case["rows"])]


def _chunks(case):
    """The prompt sequences' (tokens, position of the first one)."""
    n, total = case["sequences"], case["tokens"]
    if case["even"]:
        return [(total // n, case["prefix"])] * n
    r = random.Random(case["lengths"])
    weights = [r.uniform(0.3, 1.0) for _ in range(n)]
    counts = [max(1, int(total * w / sum(weights))) for w in weights]
    counts[-1] = total - sum(counts[:-1])
    return [(c, int(case["prefix"] * r.random())) for c in counts]


# -- what a pass cannot do without ---------------------------------------------------------------------------------------
def _row_bytes(case):
    """Bytes of one row of one kv head in 4-bit pages: the codes, and a byte of scale a group."""
    return case["dim"] // 2 + case["dim"] // GROUP


def work(case):
    op, dim = case["op"], case["dim"]
    if op == "write":
        n = case["tokens"] * case["kv_heads"] * 2
        # read 16 bits, write 4-bit rows; read those back into 16 bits
        return {"bytes": n * (2 * dim + 2 * _row_bytes(case) + 2 * dim) + 16 * case["tokens"], "flops": n * dim * 6}
    if op == "attend":
        lengths = _contexts(case)
        kv = sum(n - 1 + case["columns"] for n in lengths) * case["kv_heads"] * 2 * _row_bytes(case)
        q = case["rows"] * case["columns"] * case["q_heads"]
        pairs = sum(sum(n + c for c in range(case["columns"])) for n in lengths) * case["q_heads"]
        return {"bytes": kv + q * (4 * dim + 4), "flops": 4 * dim * pairs}
    if op == "prefill":
        chunks = _chunks(case)
        kv = sum(c + p for c, p in chunks) * case["kv_heads"] * 2 * _row_bytes(case)
        q = sum(c for c, _ in chunks) * case["q_heads"]
        pairs = sum(c * p + c * (c + 1) // 2 for c, p in chunks) * case["q_heads"]
        return {"bytes": kv + q * (4 * dim + 4), "flops": 4 * dim * pairs}
    heads = case["q_heads"] + case["kv_heads"]
    rotated = case["tokens"] * heads * dim * 4 + case["tokens"] * case["axes"] * 8 + case["rotary"] * 2 + 4 * dim
    if op == "norm_rope_write":
        rows = case["tokens"] * case["kv_heads"]
        # queries in and out, keys and values in, 4-bit rows written, read back into 16 bits
        rotated = case["tokens"] * case["q_heads"] * dim * 4 + 2 * rows * (2 * dim + 2 * _row_bytes(case) + 2 * dim) + 24 * case["tokens"]
    return {"bytes": rotated, "flops": case["tokens"] * heads * dim * 8}


# -- inputs --------------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _keys(shape, g, dtype):
    """Keys as a model's projections give them: some channels sit away from zero."""
    bias = torch.randn(shape[-2:], generator=g, device="cuda") * 1.5
    return (torch.randn(shape, generator=g, device="cuda") + bias).to(dtype)


def _scale(x):
    """The bytes of the scales nearest to x (FP32, 0 or above), half to even."""
    bits = x.view(torch.int32)
    normal = ((bits + 0x7FFFF + ((bits >> 20) & 1)) >> 20) - (112 << 3)
    byte = torch.where(x < 2.0 ** -14, (x * 2.0 ** 17).round().to(torch.int32), normal)
    return byte.clamp(max=247).to(torch.uint8)


def _scale_value(byte):
    return (byte.to(torch.int16) << 7).view(torch.float16).float()


def _quantised(x):
    """(codes packed two a byte, a byte of scale a group) of rows [...][dim]."""
    grouped = x.float().unflatten(-1, (-1, GROUP))
    # (the divisor is a tensor: a scalar one would be multiplied by its reciprocal)
    byte = _scale(grouped.abs().amax(-1) / torch.full((), 7.0, device=x.device))
    scale = _scale_value(byte)
    codes = (grouped / torch.where(scale > 0, scale, 1.0)[..., None]).round().clamp(-7, 7) * (scale > 0)[..., None]
    codes = (codes + 8).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), byte


def _values(codes, scales):
    """The FP32 values that rows of packed codes [...][dim / 2] with scales [...][dim / 32] stand for."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP)) - 8
    return (n * _scale_value(scales)[..., None]).flatten(-2)


def _cache(case, lengths, g):
    """Pages of the sequences' keys and values over shuffled page tables (the last page is nobody's)."""
    page, hkv, dim = case["page"], case["kv_heads"], case["dim"]
    width = max(-(-n // page) for n in lengths)
    pages = width * len(lengths) + 1
    state = {"tables": torch.randperm(pages - 1, generator=g, device="cuda")[:width * len(lengths)].view(len(lengths), width).to(torch.int32)}
    for name in ("k", "v"):
        codes = torch.empty(pages, page, hkv, dim // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(pages, page, hkv, dim // GROUP, dtype=torch.uint8, device="cuda")
        bias = torch.randn((hkv, dim), generator=g, device="cuda") * (1.5 if name == "k" else 0.0)
        step = max(1, (1 << 26) // (page * hkv * dim))
        for a in range(0, pages, step):
            b = min(pages, a + step)
            codes[a:b], scales[a:b] = _quantised(torch.randn((b - a, page, hkv, dim), generator=g, device="cuda") + bias)
        state[name], state[name + "s"] = codes, scales
    return state


def _empty_pages(case, g):
    page, hkv, dim = case["page"], case["kv_heads"], case["dim"]
    pages = -(-case["tokens"] // page) * (2 if case["scattered"] else 1) + 1
    state = {}
    for name in ("k", "v"):
        state[name] = torch.zeros(pages, page, hkv, dim // 2, dtype=torch.uint8, device="cuda")
        state[name + "s"] = torch.zeros(pages, page, hkv, dim // GROUP, dtype=torch.uint8, device="cuda")
    if case["scattered"]:                      # a decode step: every token in a page of its own sequence
        state["slots"] = torch.randperm((pages - 1) * page, generator=g, device="cuda")[:case["tokens"]]
    else:                                      # a prompt chunk: whole pages, in shuffled order
        order = torch.randperm(pages - 1, generator=g, device="cuda")
        state["slots"] = (order[:, None] * page + torch.arange(page, device="cuda")).flatten()[:case["tokens"]].contiguous()
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dim, dtype = case["op"], case["dim"], _dtype(case)
    state = {"case": case}
    if op == "write":
        state.update(_empty_pages(case, g))
        state["keys"] = _keys((case["tokens"], case["kv_heads"], dim), g, dtype)
        state["values"] = torch.randn((case["tokens"], case["kv_heads"], dim), generator=g, device="cuda").to(dtype)
    elif op == "attend":
        lengths, columns = _contexts(case), case["columns"]
        state.update(_cache(case, [n - 1 + columns for n in lengths], g))
        tokens = case["rows"] * columns
        state["q"] = torch.randn((tokens, case["q_heads"], dim), generator=g, device="cuda").to(dtype)
        state["rows"] = torch.arange(case["rows"], dtype=torch.int32, device="cuda")
        state["starts"] = state["rows"] * columns
        state["firsts"] = torch.tensor([n - 1 for n in lengths], dtype=torch.int64, device="cuda")
        state["lse"] = torch.empty((tokens, case["q_heads"]), dtype=torch.float32, device="cuda")
    elif op == "prefill":
        chunks = _chunks(case)
        state.update(_cache(case, [c + p for c, p in chunks], g))
        tokens = sum(c for c, _ in chunks)
        state["q"] = torch.randn((tokens, case["q_heads"], dim), generator=g, device="cuda").to(dtype)
        state["firsts"] = torch.tensor([p for _, p in chunks], dtype=torch.int64, device="cuda")
        state["lse"] = torch.empty((tokens, case["q_heads"]), dtype=torch.float32, device="cuda")
        ends = [sum(c for c, _ in chunks[:i]) for i in range(len(chunks) + 1)]
        state["starts"] = ends                                     # (row numbers, as the entry point takes them)
    else:
        tokens = case["tokens"]
        state["q"] = torch.randn((tokens, case["q_heads"], dim), generator=g, device="cuda").to(dtype)
        state["keys"] = _keys((tokens, case["kv_heads"], dim), g, dtype)
        for name in ("q_weight", "key_weight"):
            state[name] = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype) if case["norm"] else None
        half = case["rotary"] // 2
        state["frequencies"] = (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
        shape = (tokens,) if case["axes"] == 1 else (case["axes"], tokens)
        state["positions"] = torch.randint(0, case["far"], shape, generator=g, device="cuda")
        state["axes"] = None
        if case["axes"] > 1:                   # a quarter of the pairs turn with time, the rest with height and width
            first = half // 4
            second = first + (half - first) // 2
            pair = torch.arange(half, device="cuda")
            state["axes"] = ((pair >= first).int() + (pair >= second).int()).to(torch.int32)
        if op == "norm_rope_write":
            state.update(_empty_pages(case, g))
            state["values"] = (4 * torch.randn((tokens, case["kv_heads"], dim), generator=g, device="cuda")).to(dtype)
    if "slots" in state:                       # the rows read back: the keys, then the values
        state["back"] = torch.empty((2, case["tokens"], case["kv_heads"], dim), dtype=dtype, device="cuda")
    return state


# -- one pass ------------------------------------------------------------------------------------------------------------
def _store(s, name, rows):
    """Rows into their slots' codes and scales, and the values they stand for there."""
    codes, scales = _quantised(rows)
    s[name].flatten(0, 1)[s["slots"]] = codes
    s[name + "s"].flatten(0, 1)[s["slots"]] = scales
    return _values(s[name].flatten(0, 1)[s["slots"]], s[name + "s"].flatten(0, 1)[s["slots"]])


def _read(s, name):
    """The tables' rows of a cache tensor: [sequences][positions][kv_heads][dim] in FP32."""
    tables = s["tables"].long()
    return _values(s[name][tables].flatten(1, 2), s[name + "s"][tables].flatten(1, 2))


def _attention(q, k, v, firsts, valid):
    """q [sequences][columns][q_heads][dim] at positions firsts + column over k, v [sequences][positions][kv_heads][dim]:
    (out, lse) of the valid columns, one after another."""
    n, columns, heads, dim = q.shape
    hkv, length = k.shape[2], k.shape[1]
    q = q.reshape(n, columns, hkv, heads // hkv, dim).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * dim ** -0.5
    seen = torch.arange(length, device=q.device) <= firsts[:, None, None] + torch.arange(columns, device=q.device)[:, None]
    s = s.unflatten(2, (-1, columns)).masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3)).unflatten(2, (-1, columns)) / total
    lse = (top + total.log())[..., 0]
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[valid], lse.permute(0, 3, 1, 2).flatten(2, 3)[valid]


def _padded(s):
    """A prompt launch's tokens as [sequences][most tokens]: their row numbers, and which of them there are."""
    starts = torch.tensor(s["starts"], device="cuda")
    counts = starts[1:] - starts[:-1]
    most = max(b - a for a, b in zip(s["starts"], s["starts"][1:]))
    column = torch.arange(most, device="cuda")
    valid = column < counts[:, None]
    return torch.where(valid, starts[:-1, None] + column, 0), valid


def _rotated(x, weight, s, case):
    """Rows [tokens][heads][dim]: each head divided by its root mean square and weighted, then its pairs turned."""
    x = x.float()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.float()
    half = case["rotary"] // 2
    positions = s["positions"].double()
    at = positions[:, None] if s["axes"] is None else positions[s["axes"].long()].T
    angle = at * s["frequencies"].double()
    c, d = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * d, b * c + a * d], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * d, b * c + a * d], -1)
    return torch.cat([turned, rest], -1)


def _plain(s):
    case = s["case"]
    op, dtype = case["op"], _dtype(case)
    if op == "write":
        return torch.stack([_store(s, "k", s["keys"]), _store(s, "v", s["values"])]).to(dtype)
    if op == "attend":
        q = s["q"].float().unflatten(0, (case["rows"], case["columns"]))
        valid = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
        out, lse = _attention(q, _read(s, "k"), _read(s, "v"), s["firsts"], valid)
        return [out.to(dtype), lse]
    if op == "prefill":
        rows, valid = _padded(s)
        out, lse = _attention(s["q"].float()[rows], _read(s, "k"), _read(s, "v"), s["firsts"], valid)
        return [out.to(dtype), lse]
    q, keys = _rotated(s["q"], s["q_weight"], s, case), _rotated(s["keys"], s["key_weight"], s, case)
    if op == "norm_rope":
        return [q.to(dtype), keys.to(dtype)]
    # (the keys go into the pages as they are in 32 bits: one next to the border between two codes may take either)
    return [q.to(dtype), torch.stack([_store(s, "k", keys), _store(s, "v", s["values"])]).to(dtype)]


def _kernels(s):
    import crit_b200 as pk
    case = s["case"]
    op, page = case["op"], case.get("page")
    if op == "write":
        pk.write(s["keys"], s["values"], s["slots"], s["k"], s["v"], "int4", s["ks"], s["vs"])
    if op == "attend":
        out = pk.attend(s["q"], s["k"], s["v"], "int4", s["tables"], s["rows"], s["starts"], s["firsts"], case["columns"], page,
                        key_scales=s["ks"], value_scales=s["vs"], lse=s["lse"])
        return [out, s["lse"]]
    if op == "prefill":
        out = pk.prefill(s["q"], s["k"], s["v"], "int4", s["tables"], s["firsts"], page, key_scales=s["ks"], value_scales=s["vs"],
                         lse=s["lse"], starts=None if case["even"] else s["starts"])
        return [out, s["lse"]]
    if op != "write":
        rotation = dict(q_weight=s["q_weight"], key_weight=s["key_weight"], eps=EPS, axes=s["axes"], interleaved=case["interleaved"])
    if op == "norm_rope":
        return list(pk.norm_rope(s["q"], s["keys"], s["positions"], s["frequencies"], **rotation))
    if op == "norm_rope_write":
        q = pk.norm_rope_write(s["q"], s["keys"], s["values"], s["positions"], s["frequencies"], s["slots"], s["k"], s["v"],
                               "int4", s["ks"], s["vs"], **rotation)
    pk.gather(s["k"], "int4", page, slots=s["slots"], scales=s["ks"], out=s["back"][0])
    pk.gather(s["v"], "int4", page, slots=s["slots"], scales=s["vs"], out=s["back"][1])
    return s["back"] if op == "write" else [q, s["back"]]


def run(state):
    return _kernels(state) if own else _plain(state)


# -- the same from the definitions, in 64 bits ---------------------------------------------------------------------------
def _exact_scales(device):
    """Every finite scale, by its byte: m * 2^-17 for the first 8, then (8 + m) * 2^(e - 18)."""
    return torch.tensor([(b % 8 + (8 if b >= 8 else 0)) * 2.0 ** (max(b // 8, 1) - 18) for b in range(248)], dtype=torch.float64, device=device)


def _exact_row_values(x):
    """What rows stand for once written: per group of 32 the nearest of 7 steps either side of zero."""
    out = torch.empty_like(x, dtype=torch.float64)
    every = _exact_scales(x.device)
    for at in range(0, x.shape[-1], GROUP):
        part = x[..., at:at + GROUP].double()
        wide = part.abs().max(-1, keepdim=True).values / torch.tensor(7.0, dtype=torch.float64, device=x.device)
        above = torch.searchsorted(every, wide).clamp(1, 247)            # every[above - 1] < wide <= every[above], within the ends
        up, down = every[above] - wide, wide - every[above - 1]
        byte = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1)
        step = every[byte]
        out[..., at:at + GROUP] = torch.where(step > 0, step * torch.round(part / step.clamp_min(2.0 ** -17)).clamp(-7.0, 7.0), 0.0)
    return out


def _exact_cached(s, name, sequence, head, length):
    page = s["case"]["page"]
    slots = torch.arange(length, device="cuda")
    slots = s["tables"][sequence].long()[slots // page] * page + slots % page
    codes = s[name].flatten(0, 1)[slots, head].long()
    scales = _exact_scales("cuda")[s[name + "s"].flatten(0, 1)[slots, head].long()]
    n = torch.empty(length, s["case"]["dim"], dtype=torch.float64, device="cuda")
    n[:, 0::2], n[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    return (n - 8.0) * scales.repeat_interleave(GROUP, 1)


def _exact_attention(s, spans):
    """spans: (sequence, first row of q, tokens, position of the first)."""
    case = s["case"]
    heads, hkv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    group = heads // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for sequence, first, count, position in spans:
        for h in range(hkv):
            k = _exact_cached(s, "k", sequence, h, position + count)
            v = _exact_cached(s, "v", sequence, h, position + count)
            later = torch.arange(position + count, device="cuda") > position + torch.arange(count, device="cuda")[:, None]
            for j in range(h * group, (h + 1) * group):
                x = s["q"][first:first + count, j].double() @ k.T / math.sqrt(dim)
                x[later] = -math.inf
                lse[first:first + count, j] = torch.logsumexp(x, -1)
                out[first:first + count, j] = torch.exp(x - lse[first:first + count, j, None]) @ v
    return [out, lse]


def _exact_rotated(x, weight, s, case):
    y = x.double()
    if weight is not None:
        y = y * torch.rsqrt(torch.mean(y * y, -1, keepdim=True) + EPS) * weight.double()
    out = y.clone()
    half = case["rotary"] // 2
    for i in range(half):
        at = s["positions"] if s["axes"] is None else s["positions"][int(s["axes"][i])]
        angle = at.double() * float(s["frequencies"][i])
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None] * torch.complex(y[..., a].contiguous(), y[..., b].contiguous())
        out[..., a], out[..., b] = turn.real, turn.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "write":
        return torch.stack([_exact_row_values(s["keys"]), _exact_row_values(s["values"])])
    if op == "attend":
        return _exact_attention(s, [(r, r * case["columns"], case["columns"], n - 1) for r, n in enumerate(_contexts(case))])
    if op == "prefill":
        return _exact_attention(s, [(i, s["starts"][i], c, p) for i, (c, p) in enumerate(_chunks(case))])
    q, keys = _exact_rotated(s["q"], s["q_weight"], s, case), _exact_rotated(s["keys"], s["key_weight"], s, case)
    if op == "norm_rope":
        return [q, keys]
    return [q, torch.stack([_exact_row_values(keys), _exact_row_values(s["values"])])]
