"""Batches over a 4-bit paged cache for the tests: seeded inputs on the host, and their tensors."""

from __future__ import annotations

import numpy as np
import torch

from oracle import int4_cache as O
from turingserve_amd.metadata import AttentionMetadata

BLOCK = 16
HEADS = [(4, 2, 16), (6, 2, 32), (14, 2, 64), (12, 2, 128), (8, 8, 64), (34, 2, 64), (4, 1, 256)]


class Case:
    """items: (cached, new) tokens of each sequence, decode rows first. The cache is filled with
    seeded codes and numbers everywhere, also where no sequence has tokens yet: codes, steps, lows [2 (K,
    V), NB, KVH, 16, ...], whose bytes are `cache`."""

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
        self.slots = np.concatenate([self.tables[b, np.arange(c, c + n) // BLOCK].astype(np.int64) * BLOCK
                                     + np.arange(c, c + n) % BLOCK for b, (c, n) in enumerate(items)]
                                    + [np.full(tail_rows, -1, np.int64)])
        self.qkv = rng.standard_normal((self.T, (self.H + 2 * self.KVH) * self.D)).astype(np.float16)
        shape = (2, self.NB, self.KVH, BLOCK)
        self.codes = rng.integers(0, 16, (*shape, self.D)).astype(np.uint8)
        steps = np.exp(rng.normal(-1.6, 0.5, (*shape, O.groups(self.D))))
        lows = steps * (-7.5 + rng.normal(0, 2, steps.shape))
        steps[0] *= k_size
        lows[0] *= k_size
        self.steps, self.lows = steps.astype(np.float16), lows.astype(np.float16)
        self.scale = self.D ** -0.5

    @property
    def cache(self):
        """[2, NB, KVH, bytes]."""
        return np.stack([O.pack(self.codes[j], self.steps[j], self.lows[j], bool(j)) for j in range(2)])

    def split(self):
        x = self.qkv.reshape(self.T, self.H + 2 * self.KVH, self.D)
        return x[:, :self.H], x[:, self.H:self.H + self.KVH], x[:, self.H + self.KVH:]

    def on(self, device):
        """(qkv, q, k, v views, cache [1, 2, NB, KVH, bytes], meta) as tensors."""
        t = lambda a: torch.from_numpy(a).to(device)
        qkv = t(self.qkv)
        x = qkv.view(self.T, self.H + 2 * self.KVH, self.D)
        return (qkv, x[:, :self.H], x[:, self.H:self.H + self.KVH], x[:, self.H + self.KVH:],
                t(self.cache)[None], self.meta(device))

    def meta(self, device, **changes):
        t = lambda a: torch.from_numpy(a).to(device)
        n = np.diff(self.starts)
        f = dict(query_start_loc=t(self.starts), seq_lens=t(self.lens), block_tables=t(self.tables),
                 slot_mapping=t(self.slots), num_decode=self.num_decode, max_query_len=int(n.max()),
                 max_seq_len=int(self.lens.max()),
                 max_prefill_seq_len=int(self.lens[self.num_decode:].max(initial=0)))
        return AttentionMetadata(**{**f, **changes})


def near_the_rows(ops, device, heads):
    """Prompts written in one piece, then attention: as near to attention over the rows themselves as the
    codes allow. With s the largest step of a side, a value is off by at most e = s (1/2 + 15 / 2^10 + 2^-16)
    (half a code; where the step was rounded towards zero, by less than 2^-10 of itself, 15 of them at the
    group's end, or 2^-24 where it is subnormal; the quotient's rounding), and by the roundings of its
    group's low (2^-11 of it, twice the largest value's 2^-11 with the result's own). A score is then off by
    d = scale sum|q| e_k at most, a weight by a factor within e^(+-2 d), a V value by e_v; the kernels'
    own error over the codes comes on top."""
    c = Case(heads, [(0, 70), (0, 33)], seed=42)
    _, q, k, v, cache, meta = c.on(device)
    ops.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    out = ops.paged_attention_int4(q, cache[0, 0], cache[0, 1], meta, c.scale).double().cpu().numpy()
    mine = cache[0].cpu().numpy()
    _, lim = O.paged_attention(c.split()[0], mine[0], mine[1], c.tables, c.lens, c.starts, c.scale)
    qn, kn, vn = (x.astype(np.float64) for x in c.split())
    g = c.H // c.KVH
    off = [O.unpack(mine[j], c.D, bool(j))[1][c.tables].astype(np.float64).max()
           * (0.5 + 15 / 2 ** 10 + 2.0 ** -16) + 2.0 ** -10 * np.abs(x).max() + 15 * 2.0 ** -24
           for j, x in enumerate((kn, vn))]
    for b, (_, n) in enumerate(c.items):
        lo = int(c.starts[b])
        for h in range(c.H):
            for i in range(n):
                x, kk, vv = qn[lo + i, h], kn[lo:lo + i + 1, h // g], vn[lo:lo + i + 1, h // g]
                s = kk @ x * c.scale
                w = np.exp(s - s.max())
                w /= w.sum()
                d = c.scale * np.abs(x).sum() * off[0]
                bar = np.expm1(2 * d) * (w @ np.abs(vv)) + off[1]
                at = slice(h * c.D, (h + 1) * c.D)
                assert (np.abs(out[lo + i, at] - w @ vv) <= bar + lim[lo + i, at]).all()


TINY = ["below half a step of fp16", "subnormal", "zeros", "negative zeros"]


def tiny_rows(heads, kind):
    """A case whose rows of qkv are next to nothing: one channel of 2^-24 in the second half of k, whose
    rotation is the least number of its group and rounds to -0; multiples of 2^-24; zeros of both signs; of one."""
    c = Case(heads, [(5, 1), (31, 1), (0, 40)], num_decode=2, seed=72)
    rng = np.random.default_rng(73)
    if kind == TINY[0]:
        c.qkv[:] = 0
        x = c.qkv.reshape(c.T, -1, c.D)
        x[:, :, c.D // 2:] = (rng.random(x[:, :, c.D // 2:].shape) < 0.1) * np.float16(2.0 ** -24)
    elif kind == TINY[1]:
        c.qkv[:] = rng.integers(-40, 41, c.qkv.shape) * 2.0 ** -24
    elif kind == TINY[2]:
        c.qkv[:] = np.where(rng.random(c.qkv.shape) < 0.5, np.float16(0), np.float16(-0.0))
    else:
        c.qkv[:] = np.float16(-0.0)
    return c


def coherent_rows(heads):
    """A case whose K decides its results: k_j = a_j u (1 + noise), v_j = a_j t (1 + noise) with u, t rows
    of signs of a KV head and a_j between -1 and 1, q = +-(0.7 .. 1) r u with scale D r = 3. A score is about
    +-3 a_j where a code moves it by a fifteenth, and a row's result +-0.6 t."""
    c = Case(heads, [(0, 70), (0, 33)], seed=74)
    rng = np.random.default_rng(75)
    x = c.qkv.reshape(c.T, c.H + 2 * c.KVH, c.D)
    signs = lambda: rng.choice([-1.0, 1.0], (c.KVH, c.D))
    u, t, a = signs(), signs(), rng.uniform(-1, 1, (c.T, c.KVH, 1))
    noise = lambda: 1 + 0.05 * rng.standard_normal((c.T, c.KVH, c.D))
    g = c.H // c.KVH
    size = rng.uniform(0.7, 1.0, (c.T, c.H, 1)) * rng.choice([-1, 1], (c.T, c.H, 1)) * 3 / (c.scale * c.D)
    x[:, :c.H] = size * np.repeat(u, g, 0)
    x[:, c.H:c.H + c.KVH] = a * u * noise()
    x[:, c.H + c.KVH:] = a * t * noise()
    return c


def over_the_cache(ops, device, c, scale=None):
    """(attention over the cache that the case's rows were written to, the cache)."""
    _, q, k, v, cache, meta = c.on(device)
    ops.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    out = ops.paged_attention_int4(q, cache[0, 0], cache[0, 1], meta, c.scale if scale is None else scale)
    return out.double().cpu().numpy(), cache[0].cpu().numpy()


def over_the_rows(c, cache):
    """(attention over the rows themselves in 64 bits, how far attention over their codes may be off).
    A number x of a group whose span is 15 steps is off by e <= (1/2 + 2^-16) of one (15 * 2^-24 at least, by
    which the end of a group of a subnormal step may be off) and 2^-11 |x| + 2^-25 (lows are exact: the rows
    are fp16 numbers), a score by d_j = scale sum_i |q_i| e_ji, a weight, divided by the sum of all, by a factor within e^(+-(d_j + d)), d the largest d_j that the row
    sees; as the weights add up to one, the result by sum_j w_j (e^(d_j + d) - 1) |v_j - out|, and by V's own
    error at most. The operator's error over the codes (oracle.int4_cache) comes on top."""
    _, lim = O.paged_attention(c.split()[0], cache[0], cache[1], c.tables, c.lens, c.starts, c.scale)
    qn, kn, vn = (x.astype(np.float64) for x in c.split())

    def error(x):
        by = x.reshape(*x.shape[:2], O.groups(c.D), -1)
        half = np.maximum((by.max(-1) - by.min(-1)) / 15 * (0.5 + 2.0 ** -16), 15 * 2.0 ** -24)
        return np.repeat(half, c.D // O.groups(c.D), -1) + 2.0 ** -11 * np.abs(x) + 2.0 ** -25

    ek, ev = error(kn), error(vn)
    g = c.H // c.KVH
    ref, bar = np.zeros((2, c.T, c.H, c.D))
    for b, (_, n) in enumerate(c.items):
        lo = int(c.starts[b])
        for h in range(c.H):
            for i in range(n):
                at = slice(lo, lo + i + 1)
                x, kk, vv = qn[lo + i, h], kn[at, h // g], vn[at, h // g]
                s = kk @ x * c.scale
                w = np.exp(s - s.max())
                w /= w.sum()
                d = ek[at, h // g] @ np.abs(x) * c.scale
                ref[lo + i, h] = w @ vv
                off = (w * np.expm1(d + d.max())) @ np.abs(vv - ref[lo + i, h])
                bar[lo + i, h] = off + ev[at, h // g].max(0)
    return ref.reshape(c.T, -1), bar.reshape(c.T, -1) + lim


def outside(c, out, ref, bar):
    """The (row, head)s with any result outside the bar."""
    return (~(np.abs(out - ref) <= bar)).reshape(c.T, c.H, c.D).any(-1)
