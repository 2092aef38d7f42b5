"""Batches over an 8-bit paged cache for the tests: seeded inputs on the host, and their tensors."""

from __future__ import annotations

import numpy as np
import torch

from oracle import int8_cache as O
from turingserve_amd.metadata import AttentionMetadata

BLOCK = 16
HEADS = [(4, 2, 16), (6, 2, 32), (14, 2, 64), (12, 2, 128), (8, 8, 64), (34, 2, 64), (4, 1, 256)]


class Case:
    """items: (cached, new) tokens of each sequence, decode rows first. The cache is filled with
    seeded codes and scales everywhere, also where no sequence has tokens yet."""

    def __init__(self, heads, items, num_decode=0, seed=0, spare=3, k_size=1.0, tail_rows=0):
        self.H, self.KVH, self.D = heads
        self.items, self.num_decode = items, num_decode
        rng = np.random.default_rng(seed)
        need = [-(-(c + n) // BLOCK) for c, n in items]
        self.NB = sum(need) + 1 + spare
        ids = rng.permutation(self.NB - 1)[:sum(need)] + 1
        self.tables = np.zeros((len(items), max(1, max(need))), np.int32)
        at = 0
        for b, w in enumerate(need):
            self.tables[b, :w] = ids[at:at + w]
            at += w
        self.lens = np.array([c + n for c, n in items], np.int32)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in items])]).astype(np.int32)
        self.T = int(self.starts[-1]) + tail_rows
        self.pos = np.concatenate([np.arange(c, c + n) for c, n in items]
                                  + [np.zeros(tail_rows, np.int64)]).astype(np.int64)
        self.qkv = rng.standard_normal((self.T, (self.H + 2 * self.KVH) * self.D)).astype(np.float16)
        shape = (2, self.NB, self.KVH)
        self.codes = rng.integers(-127, 128, (*shape, BLOCK, self.D)).astype(np.int8)
        self.scales = np.exp(rng.normal(-4.0, 0.7, shape)).astype(np.float32)
        self.scales[0] *= k_size
        self.scale = self.D ** -0.5

    def split(self):
        x = self.qkv.reshape(self.T, self.H + 2 * self.KVH, self.D)
        return x[:, :self.H], x[:, self.H:self.H + self.KVH], x[:, self.H + self.KVH:]

    def on(self, device):
        """(qkv, q, k, v views, (k_cache, v_cache, k_scale, v_scale), meta) as tensors."""
        t = lambda a: torch.from_numpy(a).to(device)
        qkv = t(self.qkv)
        x = qkv.view(self.T, self.H + 2 * self.KVH, self.D)
        codes, scales = t(self.codes.copy()), t(self.scales.copy())
        return (qkv, x[:, :self.H], x[:, self.H:self.H + self.KVH], x[:, self.H + self.KVH:],
                (codes[0], codes[1], scales[0], scales[1]), self.meta(device))

    def meta(self, device, **changes):
        t = lambda a: torch.from_numpy(a).to(device)
        n = np.diff(self.starts)
        f = dict(query_start_loc=t(self.starts), seq_lens=t(self.lens), block_tables=t(self.tables),
                 slot_mapping=torch.full((self.T,), -1, dtype=torch.int64, device=device),
                 num_decode=self.num_decode, max_query_len=int(n.max()), max_seq_len=int(self.lens.max()),
                 max_prefill_seq_len=int(self.lens[self.num_decode:].max(initial=0)))
        return AttentionMetadata(**{**f, **changes})


def roll_back(ops, device):
    """Five drafted rows in a block that holds ten, of which two are accepted, then a row behind those,
    in both namespaces' write: the rejected rows' scale stays in the block, NaN if one of them was not
    finite; a caller who puts the block's codes and scales back and writes the accepted rows again has
    what was never drafted."""
    c = Case((4, 2, 32), [(10, 5)], seed=39)
    blk = int(c.tables[0, 0])
    for big in (40.0, np.inf):
        c.qkv[4, c.H * c.D] = big                        # K of head 0, the last rejected row
        _, _, k, v, cache, _ = c.on(device)

        def write(rows, length, cache=cache):
            at = torch.tensor(rows, device=device)
            ops.kv_write_int8(k[at], v[at], *cache, c.meta(
                device, seq_lens=torch.tensor([length], dtype=torch.int32, device=device),
                query_start_loc=torch.tensor([0, len(rows)], dtype=torch.int32, device=device)))

        was = [t[blk].clone() for t in cache]
        never = tuple(t.clone() for t in cache)
        write([0, 1], 12, never)
        write([2], 13, never)

        write([0, 1, 2, 3, 4], 15)
        drafted = [t[blk].clone() for t in cache]
        write([2], 13)
        k_scale = float(cache[2][blk, 0])
        if np.isfinite(big):
            assert k_scale == float(drafted[2][0]) == float(np.float32(big) / np.float32(127)) > float(never[2][blk, 0])
        else:
            assert np.isnan(k_scale) and np.isfinite(float(never[2][blk, 0]))
        assert torch.equal(cache[0][blk, 1, :13], drafted[0][1, :13])        # (rows that were there)

        for t, x in zip(cache, was):
            t[blk] = x
        write([0, 1], 12)
        write([2], 13)
        assert all(torch.equal(a[blk][:, :13] if a.dim() == 4 else a[blk], b[blk][:, :13] if b.dim() == 4 else b[blk])
                   for a, b in zip(cache, never))


def near_the_rows(ops, device, heads):
    """Prompts written in one piece, then attention: as near to attention over the rows themselves as half
    a code allows. A K value is off by half its block's scale (and 2^-16 of it: the scale's and the quotient's
    rounding), a score by at most d = scale * sum |q| * that, a weight by a factor within e^(+-2 d), a V value by
    half its scale; the kernels' own error over the codes comes on top."""
    c = Case(heads, [(0, 70), (0, 33)], seed=42)
    _, q, k, v, cache, meta = c.on(device)
    ops.kv_write_int8(k, v, *cache, meta)
    out = ops.paged_attention_int8(q, *cache, meta, c.scale).double().cpu().numpy()
    codes, scales = (torch.stack(t).cpu().numpy() for t in (cache[:2], cache[2:]))
    _, lim = O.paged_attention(c.split()[0], codes, scales, c.tables, c.lens, c.starts, c.scale)
    qn, kn, vn = (x.astype(np.float64) for x in c.split())
    half = 0.5 + 2.0 ** -16
    g = c.H // c.KVH
    for b, (_, n) in enumerate(c.items):
        lo = int(c.starts[b])
        step = np.repeat(scales[:, c.tables[b, :-(-n // BLOCK)]].astype(np.float64), BLOCK, 1)[:, :n] * half
        for h in range(c.H):
            for i in range(n):
                x, kk, vv = qn[lo + i, h], kn[lo:lo + i + 1, h // g], vn[lo:lo + i + 1, h // g]
                s = kk @ x * c.scale
                w = np.exp(s - s.max())
                w /= w.sum()
                d = c.scale * np.abs(x).sum() * step[0, :i + 1, h // g].max()
                off = np.expm1(2 * d) * (w @ np.abs(vv)) + step[1, :i + 1, h // g].max()
                at = slice(h * c.D, (h + 1) * c.D)
                assert (np.abs(out[lo + i, at] - w @ vv) <= off + lim[lo + i, at]).all()
