"""numpy restatement of the 8-bit paged cache (test infrastructure only): its write, and attention
over it in 64 bits. The reference has no such cache; the definitions are those of
include/turingserve_hip.h.

codes [NB, KVH, 16, D] int8, scales [NB, KVH] fp32, a code standing for code * scale. A step is
described by its sequences' (block table row, seq_len) and query_start_loc.
"""

from __future__ import annotations

import numpy as np

BLOCK = 16
F32 = np.float32


def write_block(rows, codes, scales, at: int) -> None:
    """rows [KVH, n, D] (fp32 values) into rows at .. at + n - 1 of one block's codes [KVH, 16, D]
    and scales [KVH], in place."""
    rows = rows.astype(F32)
    n = rows.shape[1]
    for h in range(rows.shape[0]):
        was = scales[h] if at > 0 else F32(0)
        top = np.abs(rows[h]).max()
        if not np.isfinite(top) or np.isnan(was):
            scales[h] = np.nan
            codes[h, at:at + n] = 0
            continue
        now = max(was, top / F32(127))
        if now > was:
            codes[h, :at] = np.rint(codes[h, :at].astype(F32) * (was / now))
        codes[h, at:at + n] = np.clip(np.rint(rows[h] / now), -127, 127) if now > 0 else 0
        scales[h] = now


def write(x, codes, scales, tables, seq_lens, starts) -> None:
    """The step's rows x [T, KVH, D] into codes / scales, in place."""
    tables = np.asarray(tables)
    for b, length in enumerate(np.asarray(seq_lens).tolist()):
        n = int(starts[b + 1] - starts[b])
        first = length - n                           # position of the sequence's first new row
        pos = max(first, 0)
        while pos < length:
            j = pos // BLOCK
            end = min(length, BLOCK * (j + 1))
            if j < tables.shape[1] and 0 <= tables[b, j] < codes.shape[0]:
                t = int(starts[b]) + pos - first
                blk = tables[b, j]
                write_block(np.moveaxis(x[t:t + end - pos], 0, 1), codes[blk], scales[blk],
                            pos - BLOCK * j)
            pos = end


def rotate(x, cos, sin):
    """Rotate-half RoPE of x [T, heads, D] by cos / sin [T, D / 2], in float64."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], axis=-1)


def values(codes, scales, table_row, length: int):
    """The first `length` tokens of a sequence as float64 [length, KVH, D]."""
    blocks = np.asarray(table_row[:-(-length // BLOCK)], dtype=np.int64)
    v = codes[blocks].astype(np.float64) * scales[blocks].astype(np.float64)[:, :, None, None]
    return v.transpose(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])[:length]


def attention(q, k, v, seen, scale: float):
    """q [n, H, D], k / v [tokens, KVH, D] in float64; row i sees the first seen[i] tokens (none:
    zeros). Returns (out [n, H, D], weight [n, H, D] = sum_j w_j |v_j|, reach [n, H] = the largest
    sum_d |q_d k_jd| * scale among the tokens seen)."""
    n, H, D = q.shape
    g = H // k.shape[1]
    out, weight, reach = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros((n, H))
    for h in range(H):
        kk, vv = k[:, h // g], v[:, h // g]
        s, r = q[:, h] @ kk.T * scale, np.abs(q[:, h]) @ np.abs(kk).T * scale
        for i in range(n):
            m = int(seen[i])
            if m <= 0:
                continue
            w = np.exp(s[i, :m] - s[i, :m].max())
            w /= w.sum()
            out[i, h], weight[i, h] = w @ vv[:m], w @ np.abs(vv[:m])
            reach[i, h] = r[i, :m].max()
    return out, weight, reach


def paged_attention(q, codes, scales, tables, seq_lens, starts, scale: float):
    """q [T, H, D] -> (out, bound) float64 [T, H * D] over (k, v) pairs codes / scales; rows outside
    every sequence are NaN in both. `bound` is how far fp16 results may be off:

    * the score of a token is a dot product of D terms in fp32, times two fp32 factors: off by at
      most (D + 4) 2^-24 reach; the exponent's argument and the exponential add 4 * 2^-24 * reach
      and 2^-22, the ratio of a block's V scale to the largest, which may pass through a base-2
      logarithm of at most 30, another 2^-19; call the sum e. Weights are then off by a factor within 1 +- 2 e (numerator and
      sum);
    * a weight is rounded to fp16 relative to a running reference that the row's largest weight is
      never below: 2^-11 of it, or 2^-25 (half a subnormal step) of the largest V value;
    * P.V adds up in fp32: tokens * 2^-24 of the sum of magnitudes, times 2;
    * the result is rounded to fp16: 2^-11 of it, or 2^-25."""
    T, H, D = q.shape
    out = np.full((T, H * D), np.nan)
    bound = np.full((T, H * D), np.nan)
    tables = np.asarray(tables)
    for b, length in enumerate(np.asarray(seq_lens).tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        held = max(0, min(length, BLOCK * tables.shape[1]))
        k, v = (values(c, s, tables[b], held) for c, s in zip(codes, scales))
        seen = np.clip(np.arange(lo, hi) - lo + length - (hi - lo) + 1, 0, held)
        o, w, r = attention(q[lo:hi].astype(np.float64), k, v, seen, scale)
        e = (D + 8) * 2.0 ** -24 * r[:, :, None] + 2.0 ** -22 + 2.0 ** -19
        top = np.abs(v).max() if held else 0.0
        lim = ((2.0 ** -11 + 2 * e + held * 2.0 ** -23) * w + held * 2.0 ** -25 * top
               + 2.0 ** -11 * np.abs(o) + 2.0 ** -25)
        out[lo:hi], bound[lo:hi] = o.reshape(-1, H * D), lim.reshape(-1, H * D)
    return out, bound
