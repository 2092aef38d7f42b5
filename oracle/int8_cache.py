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


def attention(q, k, v, vs, seen, scale: float):
    """q [n, H, D], k / v [tokens, KVH, D] and the tokens' V scales vs [tokens, KVH] in float64; row i
    sees the first seen[i] tokens (none: zeros). Returns (out [n, H, D], bound [n, H, D]), the bound
    as in paged_attention."""
    n, H, D = q.shape
    g, u = H // k.shape[1], 2.0 ** -24
    out, bound = np.zeros((n, H, D)), np.zeros((n, H, D))
    hidden = np.arange(k.shape[0])[None, :] >= seen[:, None]
    some = seen > 0
    for h in range(H if some.any() else 0):
        kk, vv, sv = k[:, h // g], v[:, h // g], np.maximum(vs[:, h // g], 2.0 ** -40)
        s = np.where(hidden, -np.inf, q[:, h] @ kk.T * scale)[some]
        reach = np.where(hidden, 0.0, np.abs(q[:, h]) @ np.abs(kk).T * scale)[some].max(1)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        o, size, m = w @ vv, w @ np.abs(vv), seen[some][:, None]
        # the scores
        e = 2 * ((D + 8) * u * reach + 2.0 ** -22 + 2.0 ** -17)
        spread = size.copy()
        for i in np.flatnonzero(e > 2.0 ** -6):
            spread[i] = np.minimum(size[i], w[i] @ np.abs(vv - o[i]))
        off = np.expm1(np.minimum(e, 60.0))[:, None] * spread
        # the rounding of P to fp16, and the sums
        off += (2.0 ** -11 + (m / 32 + 16) * u + 8 * u * np.sqrt(m + 256)) * (size + off)
        top = np.minimum((w * sv).max(1) * np.exp(np.minimum(e, 60.0)), np.where(hidden[some], 0.0, sv).max(1))
        codes = np.cumsum(np.abs(vv) / sv[:, None], 0)[seen[some] - 1]
        off += 2.0 ** -25 * top[:, None] * codes
        out[some, h], bound[some, h] = o, off
    return out, bound + 2.0 ** -11 * (np.abs(out) + bound) + 2.0 ** -25 + 2.0 ** -32


def paged_attention(q, codes, scales, tables, seq_lens, starts, scale: float):
    """q [T, H, D] -> (out, bound) float64 [T, H * D] over (k, v) pairs codes / scales; rows outside
    every sequence are NaN in both. `bound` is how far fp16 results may be off. Every term is of the
    row and KV head alone and of the tokens that the row sees:

    * a token's exponent is a dot product of D terms in fp32, times two fp32 factors: off by at most
      (D + 4) 2^-24 reach, reach the largest sum_d |q_d k_jd| * scale; the argument and the exponential
      add 4 * 2^-24 * reach and 2^-22. V's scale may pass through a base-2 logarithm of at most 40 in
      magnitude: one unit in its last place, 2^-23 of it, and three roundings of 2^-24 of it, 40 * 5 *
      2^-24 ln 2 < 2^-17. Call the sum e. A weight, divided by the sum of all, is then off by a factor
      within e^(+-2 e), the result by at most e^(2 e) - 1 times the smaller of sum_j w_j |v_j| and, as
      the weights still add up to one, sum_j w_j |v_j - out| (looked at where 2 e is above 2^-6);
    * a weight times its V scale is rounded to fp16 against a running reference that the row's largest
      such product is never below: 2^-11 of it, or 2^-25 (half a subnormal step) of the largest
      product, times the code;
    * the row's sum is one of positive numbers over at least 32 chains: tokens / 32 + 16 roundings of
      2^-24; P.V adds up in fp32 with roundings that do not hang together: 8 sqrt(tokens + 256) 2^-24
      of the sum of magnitudes (256 for the wavefronts' and splits' parts; eight deviations);
    * the result is rounded to fp16: 2^-11 of it, or 2^-25; a V scale below 2^-40 may count as 2^-40,
      127 * 2^-40 < 2^-32."""
    T, H, D = q.shape
    out = np.full((T, H * D), np.nan)
    bound = np.full((T, H * D), np.nan)
    tables = np.asarray(tables)
    for b, length in enumerate(np.asarray(seq_lens).tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        held = max(0, min(length, BLOCK * tables.shape[1]))
        k, v = (values(c, s, tables[b], held) for c, s in zip(codes, scales))
        vs = np.repeat(scales[1][tables[b][:-(-held // BLOCK)]].astype(np.float64), BLOCK, 0)[:held]
        seen = np.clip(np.arange(lo, hi) - lo + length - (hi - lo) + 1, 0, held)
        o, lim = attention(q[lo:hi].astype(np.float64), k, v, vs, seen, scale)
        out[lo:hi], bound[lo:hi] = o.reshape(-1, H * D), lim.reshape(-1, H * D)
    return out, bound
