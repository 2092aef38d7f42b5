"""numpy restatement of the 4-bit paged cache (test infrastructure only): its layout, its write, and
attention over it in 64 bits. The reference has no such cache; the definitions are those of
include/turingserve_hip.h.

A unit is one block of one KV head, a row of bytes: 16 rows of 4-bit codes, then 16 rows of (step, low) in
fp16 for each group of min(32, D) channels; a code stands for fp16(low + code * step).
"""

from __future__ import annotations

import numpy as np

from oracle import int8_cache as O8

BLOCK = 16
F32, F16 = np.float32, np.float16
rotate = O8.rotate


def groups(D: int) -> int:
    return max(1, D // 32)


def unit_bytes(D: int) -> int:
    return BLOCK * D // 2 + BLOCK * groups(D) * 4


def code_place(row: int, d: int, D: int, values: bool) -> tuple[int, int]:
    """(byte, shift) of a code in its unit."""
    octet, c = d // 8, d % 8
    nibble = c // 2 + 4 * (c % 2)
    word = octet * BLOCK + row if values else row * (D // 8) + octet
    return 4 * word + nibble // 2, 4 * (nibble % 2)


def number_places(row: int, group: int, D: int, values: bool) -> tuple[int, int]:
    """Byte offsets of a row's step and low of a group in their unit."""
    at = BLOCK * D // 2
    if values:
        at += (group * 4 + row // 4) * 16 + 2 * (row % 4)
        return at, at + 8
    at += (row * groups(D) + group) * 4
    return at, at + 2


def _places(D: int, values: bool):
    """Index arrays of a unit: codes' bytes and shifts [16, D], steps' and lows' first bytes [16, G]."""
    code = np.array([[code_place(r, d, D, values) for d in range(D)] for r in range(BLOCK)])
    num = np.array([[number_places(r, g, D, values) for g in range(groups(D))] for r in range(BLOCK)])
    return code[..., 0], code[..., 1], num[..., 0], num[..., 1]


def unpack(cache, D: int, values: bool):
    """cache [..., bytes] -> codes [..., 16, D] uint8, steps and lows [..., 16, G] fp16."""
    at, shift, step, low = _places(D, values)
    half = lambda p: np.ascontiguousarray(np.stack([cache[..., p], cache[..., p + 1]], -1)).view(F16)[..., 0]
    return (cache[..., at] >> shift.astype(np.uint8)) & np.uint8(15), half(step), half(low)


def pack(codes, steps, lows, values: bool):
    """The inverse: [..., bytes]."""
    D = codes.shape[-1]
    at, shift, step, low = _places(D, values)
    out = np.zeros((*codes.shape[:-2], unit_bytes(D)), np.uint8)
    for r in range(BLOCK):
        for d in range(D):
            out[..., at[r, d]] |= codes[..., r, d].astype(np.uint8) << np.uint8(shift[r, d])
        for g in range(groups(D)):
            for p, x in ((step, steps), (low, lows)):
                out[..., p[r, g]:p[r, g] + 2] = np.ascontiguousarray(x[..., r, g, None].astype(F16)).view(np.uint8)
    return out


def toward_zero(x):
    """fp32 numbers >= 0 to fp16, rounded towards zero."""
    h = x.astype(F16)
    return np.where(h.astype(F32) > x, np.nextafter(h, F16(0)), h).astype(F16)


def quantise(x):
    """Rows x [..., D] (fp32 values) -> codes [..., D], steps and lows [..., G]."""
    D = x.shape[-1]
    x = x.astype(F32).reshape(*x.shape[:-1], groups(D), D // groups(D))
    lows = x.min(-1).astype(F16) + F16(0)                      # (-0 as 0)
    wide = lows.astype(F32)
    steps = toward_zero(np.maximum(x.max(-1) - wide, F32(0)) / F32(15))
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.clip(np.rint((x - wide[..., None]) / steps.astype(F32)[..., None]), 0, 15)
    codes = np.where(steps[..., None] > 0, codes, 0).astype(np.uint8)
    return codes.reshape(*codes.shape[:-2], D), steps, lows


def held(x):
    """What the cache holds for rows x [..., D], fp16."""
    return values_of(*quantise(x))


def values_of(codes, steps, lows):
    """What codes [..., D] stand for, [..., D] fp16 (64 bits hold the product and the sum exactly)."""
    G = steps.shape[-1]
    x = codes.reshape(*codes.shape[:-1], G, codes.shape[-1] // G).astype(np.float64)
    x = x * steps.astype(np.float64)[..., None] + lows.astype(np.float64)[..., None]
    return x.reshape(codes.shape).astype(F16)


def write(k, v, k_cache, v_cache, slots) -> None:
    """Rows k, v [T, KVH, D] (fp32 values) into the caches [NB, KVH, bytes] at `slots`, in place. A
    token whose K or V row of a head is not finite in fp16 is NaN in that head, K and V."""
    D = k.shape[-1]
    k, v = k.astype(F32), v.astype(F32)
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(k) <= 65504).all(-1) & (np.abs(v) <= 65504).all(-1))
    for x, cache, is_v in ((k, k_cache, False), (v, v_cache, True)):
        codes, steps, lows = quantise(np.where(bad[..., None], F32(0), x))
        lows[bad] = np.nan
        at, shift, step, low = _places(D, is_v)
        for t, slot in enumerate(np.asarray(slots)[:len(k)].tolist()):
            if not 0 <= slot < BLOCK * len(cache):
                continue
            unit, r = cache[slot // BLOCK], slot % BLOCK                     # [KVH, bytes]
            for d in range(D):
                b, s = at[r, d], shift[r, d]
                unit[:, b] = (unit[:, b] & np.uint8(255 - (15 << s))) | codes[t, :, d] << np.uint8(s)
            for g in range(groups(D)):
                for p, n in ((step, steps), (low, lows)):
                    unit[:, p[r, g]:p[r, g] + 2] = np.ascontiguousarray(n[t, :, g, None]).view(np.uint8)


def values(cache, table_row, length: int, D: int, is_v: bool):
    """The first `length` tokens of a sequence as float64 [length, KVH, D]."""
    blocks = np.asarray(table_row[:-(-length // BLOCK)], dtype=np.int64)
    x = values_of(*unpack(cache[blocks], D, is_v)).astype(np.float64)
    return x.transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], D)[:length]


def paged_attention(q, k_cache, v_cache, tables, seq_lens, starts, scale: float):
    """q [T, H, D] -> (out, bound) float64 [T, H * D]; rows outside every sequence are NaN in both, rows
    that see a token of NaN in `out`. `bound` is how far fp16 results may be off, as for the 8-bit
    cache (oracle.int8_cache.paged_attention) with V scales of 1: K and V enter the products as the fp16
    numbers that they stand for, a weight is rounded to fp16 against a reference that the row's
    largest weight is never below (2^-11 of it, or 2^-25 of the largest, times the value)."""
    T, H, D = q.shape
    out, bound = np.full((T, H * D), np.nan), np.full((T, H * D), np.nan)
    tables = np.asarray(tables)
    g = H // k_cache.shape[1]
    for b, length in enumerate(np.asarray(seq_lens).tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        n = max(0, min(length, BLOCK * tables.shape[1]))
        k, v = values(k_cache, tables[b], n, D, False), values(v_cache, tables[b], n, D, True)
        nan = np.isnan(k).any(-1)                                            # [tokens, KVH]
        k, v = np.where(np.isnan(k), 0.0, k), np.where(np.isnan(v), 0.0, v)
        seen = np.clip(np.arange(lo, hi) - lo + length - (hi - lo) + 1, 0, n)
        o, lim = O8.attention(q[lo:hi].astype(np.float64), k, v, np.ones(k.shape[:2]), seen, scale)
        hit = np.concatenate([np.zeros((1, k.shape[1]), bool), np.maximum.accumulate(nan, 0)])[seen]
        o[np.repeat(hit, g, axis=1)] = np.nan
        out[lo:hi], bound[lo:hi] = o.reshape(-1, H * D), lim.reshape(-1, H * D)
    return out, bound
