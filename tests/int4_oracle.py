"""The 4-bit page kind restated on the CPU in 64 bits (numpy), for the tests: the format, and attention over its pages."""
import math

import numpy as np
import torch

GROUP = 32
SCALES = np.array([(b % 8 + (8 if b >= 8 else 0)) * 2.0 ** (max(b // 8, 1) - 18) for b in range(248)])


def scale_byte(x):
    """The byte of the scale nearest to x >= 0, half to even."""
    above = np.clip(np.searchsorted(SCALES, x), 1, 247)
    up, down = SCALES[above] - x, x - SCALES[above - 1]
    return np.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1).astype(np.uint8)


def quantise4(x):
    """Rows [...][dim] of finite numbers -> (codes [...][dim], scale bytes [...][dim / 32])."""
    grouped = x.reshape(*x.shape[:-1], -1, GROUP)
    byte = scale_byte(np.float32(np.abs(grouped).max(-1)) / np.float32(7))       # (the quotient as FP32 has it)
    s = SCALES[byte][..., None]
    codes = np.where(s > 0, np.clip(np.rint(grouped / np.where(s > 0, s, 1)), -7, 7), 0) + 8
    return codes.astype(np.uint8).reshape(x.shape), byte


def values4(codes, byte):
    return ((codes.astype(np.float64) - 8).reshape(*codes.shape[:-1], -1, GROUP) * SCALES[byte][..., None]).reshape(codes.shape)


class Cache4:
    """One layer's int4 pages on the GPU; filled(): sequences over shuffled pages, written through the product."""

    def __init__(self, heads, dim, page, pages):
        self.heads, self.dim, self.page = heads, dim, page
        self.k, self.v = (torch.zeros(pages, page, heads, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.ks, self.vs = (torch.zeros(pages, page, heads, dim // GROUP, dtype=torch.uint8, device="cuda") for _ in range(2))

    @classmethod
    def filled(cls, heads, dim, page, lengths, seed, poison=False, scale=1.0, spare=0):
        """poison: what is not written holds 0xff bytes (NaN scales)."""
        g = torch.Generator().manual_seed(seed)
        width = max(-(-(n + spare) // page) for n in lengths)
        cache = cls(heads, dim, page, width * len(lengths) + 1)
        if poison:
            for x in (cache.k, cache.v, cache.ks, cache.vs):
                x.fill_(0xFF)
        cache.tables = torch.randperm(width * len(lengths), generator=g).view(len(lengths), width).to(torch.int32).cuda()
        bias = torch.randn(heads, dim, generator=g)
        for s, n in enumerate(lengths):
            keys, values = torch.randn(n, heads, dim, generator=g) + bias, torch.randn(n, heads, dim, generator=g)
            cache.write(s, 0, (keys * scale).bfloat16().cuda(), (values * scale).bfloat16().cuda())
        return cache

    def slots(self, s, positions):
        positions = positions.to(self.tables.device)
        return self.tables[s][positions // self.page].long() * self.page + positions % self.page

    def write(self, s, start, keys, values):
        import crit_b200 as pk
        slots = self.slots(s, torch.arange(start, start + keys.shape[0]))
        pk.write(keys, values, slots, self.k, self.v, "int4", self.ks, self.vs)

    def rows(self, which, s, count):
        """The sequence's first `count` rows as stored, [count][heads][dim] float64 (NaN where the scale is)."""
        slots = self.slots(s, torch.arange(count))
        packed = getattr(self, which).flatten(0, 1)[slots].cpu().numpy()
        byte = getattr(self, which + "s").flatten(0, 1)[slots].cpu().numpy()
        codes = np.stack([packed & 15, packed >> 4], -1).reshape(count, self.heads, self.dim)
        found = values4(codes, np.minimum(byte, 247))
        return np.where(np.repeat(byte > 247, GROUP, -1), np.nan, found)


def attention4(cache, q, row, first, column, count, token, scale=None, parents=None, sliding=0, sinks=None, blocks=None,
               block_size=None, context=False):
    """Token `token` (column `column` of a row of `count` at position first..) over the cache, in 64 bits: (out
    [q_heads][dim], lse [q_heads], room [q_heads][dim]: the weighted sum of |values|)."""
    heads, dim = q.shape
    length = first if context else first + count
    pos = np.arange(length)
    own = first + column
    if context:
        see = pos < first
    elif parents is not None:
        see, at, base = pos < first, column, token - column
        while at >= 0:
            see = see | (pos == first + at)
            at = int(parents[base + at])
    else:
        see = pos <= own
    if sliding:
        see &= pos > own - sliding
    if blocks is not None:
        see &= np.isin(pos // block_size, blocks[token].cpu().numpy()) & (pos <= own)
    out, lse, room = np.zeros((heads, dim)), np.full(heads, -np.inf), np.zeros((heads, dim))
    if length:
        k, v = cache.rows("k", row, length), cache.rows("v", row, length)
    for h in range(heads):
        kv = h // (heads // cache.heads)
        s = np.array([])
        if length and see.any():
            s = (k[see, kv] @ q[h].double().cpu().numpy()) * (scale if scale is not None else dim ** -0.5)
        every = np.append(s, float(sinks[h])) if sinks is not None else s
        if not len(every):
            continue
        top = every.max()
        total = np.exp(every - top).sum()
        lse[h] = top + math.log(total)
        if len(s):
            w = np.exp(s - top) / total
            out[h], room[h] = w @ v[see, kv], w @ np.abs(v[see, kv])
    return out, lse, room


def bounds4(want, room, positions, dtype):
    """What the kernel's roundings can add up to: half a step of the output's type; a weight rounded to FP16 and the product
    with its scale rounded again, 2 * 2^-11 of the weighted sum of |values|; scores whose 128 products are summed in FP32,
    136 * 2^-24 of a sum of |q k| that stays below 30 here, in the weight and in the total, 4.9e-4 (the two together below 2^-9);
    and FP16's smallest step where weights are tiny, 2^-25 times a code of 7 against a total of 1/4 or more, 2^-20 a position."""
    return torch.finfo(dtype).eps / 2 * np.abs(want) + 2.0 ** -9 * room + positions * 2.0 ** -20 * (np.abs(room).max() + 1e-30) + 1e-30
