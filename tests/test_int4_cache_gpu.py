"""The 4-bit paged cache on the GPU against the 64-bit oracle (oracle/int4_cache.py): its write must give
the oracle's bytes, its read the numbers that they stand for, attention stay inside the oracle's error
bound."""

from __future__ import annotations

import dataclasses
import math

import numpy as np
import pytest
import torch

from oracle import int4_cache as O
from tests.int4_cases import (HEADS, TINY, Case, coherent_rows, near_the_rows, outside, over_the_cache,
                              over_the_rows, tiny_rows)
from turingserve_amd import get_ops
from turingserve_amd import hip_ops as H
from turingserve_amd.quant import Int4KVCache
from turingserve_amd.qwen2 import rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def oracle_write(c, k=None, v=None, slots=None):
    """The cache's bytes after the write of the case's (or the given) rows."""
    cache = c.cache
    _, kn, vn = c.split()
    O.write(kn if k is None else k, vn if v is None else v, *cache, c.slots if slots is None else slots)
    return cache


def assert_cache(cache, want, what=""):
    got = cache[0].cpu().numpy()
    assert np.array_equal(got, want), f"{what}: {int((got != want).sum())} bytes differ"


def attend(q, cache, meta, scale):
    return H.paged_attention_int4(q, cache[0, 0], cache[0, 1], meta, scale)


def assert_rows(out, c, what="", rows=slice(None), **kw):
    """out against the oracle's bound, over the rows that belong to sequences."""
    cache = kw["cache"] if "cache" in kw else c.cache
    q = kw.get("q", c.split()[0])
    ref, bound = O.paged_attention(q, *cache, c.tables, kw.get("lens", c.lens), c.starts, c.scale)
    got = out.double().cpu().numpy()
    got, ref, bound = got[rows], ref[rows], bound[rows]
    real = ~np.isnan(bound) & ~np.isnan(ref)
    assert np.isnan(got[~np.isnan(bound) & np.isnan(ref)]).all(), f"{what}: rows that see NaN"
    err = np.abs(got - ref)
    worst = np.nanmax(np.where(real, err / bound, 0.0)) if real.any() else 0.0
    assert (err[real] <= bound[real]).all(), f"{what}: {worst:.3g} of the bound"
    return worst


# ------------------------------------------------------------------------------------- write and read
ITEMS = [(5, 1), (15, 1), (16, 1), (0, 1), (0, 16), (3, 40), (31, 17), (0, 300), (1, 2), (30, 18)]


@pytest.mark.parametrize("heads", HEADS)
def test_write_matches_the_oracle(heads):
    c = Case(heads, ITEMS, num_decode=4, seed=1, tail_rows=3)
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    want = oracle_write(c)
    assert_cache(cache, want, f"write {heads}")
    H.kv_write_int4(k.contiguous(), v.contiguous(), cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert_cache(cache, want, f"write again {heads}")


@pytest.mark.parametrize("heads", HEADS)
def test_rope_write_matches_the_oracle(heads):
    h, kvh, d = heads
    c = Case(heads, ITEMS, num_decode=4, seed=2, tail_rows=3)
    qkv, _, _, _, cache, meta = c.on(DEV)
    before = qkv.clone()
    cos, sin = rope_tables(d, 1e6, 512, DEV)
    q = H.rope_kv_write_int4(qkv, torch.from_numpy(c.pos).to(DEV), cos, sin, h, kvh, d, cache[0, 0],
                             cache[0, 1], meta.slot_mapping)
    assert torch.equal(qkv, before)
    qn, kn, _ = c.split()
    cn, sn = cos.cpu().numpy()[c.pos], sin.cpu().numpy()[c.pos]
    assert_cache(cache, oracle_write(c, k=O.rotate(kn, cn, sn)), f"rope write {heads}")
    # q: a product and a fused product-sum in fp32 (2^-24 of each product's size, once each), then
    # fp16 (2^-11, or half a subnormal step)
    want = O.rotate(qn, cn, sn)
    half = d // 2
    size = np.abs(qn.astype(np.float64))
    size = size + np.concatenate([size[..., half:], size[..., :half]], -1)
    lim = 2.0 ** -11 * np.abs(want) + 2.0 ** -23 * size + 2.0 ** -25
    assert (np.abs(q.double().cpu().numpy() - want) <= lim).all()


@pytest.mark.parametrize("heads", HEADS)
def test_read_matches_the_oracle(heads):
    """Several layers, blocks in any order, twice the same one, ids outside the cache (block 0)."""
    parts = [Case(heads, [(0, 90)], seed=s) for s in (50, 51, 52)]
    both = np.stack([p.cache for p in parts])
    cache = torch.from_numpy(both).to(DEV)
    ids = [3, 1, 3, 0, -1, parts[0].NB, 2 ** 31 - 1, 5]
    real = [3, 1, 3, 0, 0, 0, 0, 5]
    for dtype in (torch.int32, torch.int64):
        got = H.kv_read_int4(cache, torch.tensor(ids, dtype=dtype, device=DEV)).cpu().numpy()
        for i in range(3):
            for j in range(2):
                want = O.values_of(*O.unpack(both[i, j], heads[2], bool(j)))[real]
                assert np.array_equal(got[i, j], want), (i, j)
    far = torch.tensor([2 ** 32 + 1, -2 ** 32 + 2, 2 ** 62], device=DEV)
    got = H.kv_read_int4(cache[1:2], far).cpu().numpy()
    assert np.array_equal(got[0, 0], O.values_of(*O.unpack(both[1, 0], heads[2], False))[[0, 0, 0]])
    for dtype in (torch.uint8, torch.int8, torch.int16):
        got = H.kv_read_int4(cache[:1], torch.tensor([3, 1, 100], dtype=dtype, device=DEV)).cpu().numpy()
        assert np.array_equal(got[0, 1], O.values_of(*O.unpack(both[0, 1], heads[2], True))[[3, 1, 0]])
    wide = torch.tensor(ids, dtype=torch.int32, device=DEV).repeat_interleave(2)[::2]
    assert np.array_equal(H.kv_read_int4(cache, wide).cpu().numpy()[2, 1], O.values_of(
        *O.unpack(both[2, 1], heads[2], True))[real])
    assert H.kv_read_int4(cache, wide[:0]).shape == (3, 2, 0, heads[1], 16, heads[2])
    with pytest.raises(ValueError, match="contiguous"):
        H.kv_read_int4(cache[:, :, ::2], wide)
    with pytest.raises(ValueError, match="GPU"):
        H.kv_read_int4(cache, wide.cpu())


def test_read_back_is_what_attention_uses():
    """The fp16 operators over the blocks read back, tables renumbered, against attention over the 4-bit
    cache: the same numbers go in, so both stay within the bound around the same result."""
    c = Case((12, 2, 128), [(700, 1), (90, 1), (300, 200)], num_decode=2, seed=53)
    _, q, _, _, cache, meta = c.on(DEV)
    ids = torch.from_numpy(np.unique(c.tables)).to(DEV)
    kc, vc = H.kv_read_int4(cache, ids)[0]
    place = torch.zeros(c.NB, dtype=torch.int32, device=DEV)
    place[ids.long()] = torch.arange(len(ids), dtype=torch.int32, device=DEV)
    there = dataclasses.replace(meta, block_tables=place[meta.block_tables.long()])
    assert_rows(H.paged_attention(q, kc, vc, there, c.scale), c, "fp16")
    assert_rows(attend(q, cache, meta, c.scale), c, "4 bits")


@pytest.mark.parametrize("size", [0.0, 6e-8, 1e-6, 1e-4, 60000.0, 65504.0])
def test_write_of_rows_of_any_size(size):
    """Zero rows, subnormal ones (spans below 15 subnormal steps have a step of 0), the largest."""
    c = Case((2, 2, 64), [(7, 1), (0, 1), (9, 30)], num_decode=2, seed=3)
    c.qkv[:] = np.clip(c.qkv.astype(np.float32), -1, 1) * np.float32(size)
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert_cache(cache, oracle_write(c), f"rows of {size}")
    got = H.kv_read_int4(cache, meta.block_tables[2, :3])
    assert torch.isfinite(got).all()
    c.qkv[:] = np.sign(c.qkv) * np.float16(size)                         # two values, zeros of both signs
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert_cache(cache, oracle_write(c), f"rows of +-{size}")


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_rows_that_are_not_finite(bad):
    """K and V of such a token and head are NaN, nothing else is; a row written over it is forgotten."""
    c = Case((2, 2, 64), [(7, 1), (20, 1), (9, 40)], num_decode=2, seed=4)
    good = c.qkv.copy()
    c.qkv[0, 2 * 64 + 5] = bad                       # K of head 0, the first sequence's row
    c.qkv[9, 5 * 64 + 7] = bad                       # V of head 1, inside the chunk
    _, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    want = oracle_write(c)
    assert_cache(cache, want)
    lost = np.isnan(np.stack([O.values_of(*O.unpack(want[j], 64, bool(j))) for j in range(2)]))
    assert lost.sum() == 4 * 64
    for t, h in ((0, 0), (9, 1)):
        assert lost[:, c.slots[t] // 16, h, c.slots[t] % 16].all()
    assert_rows(attend(q, cache, meta, c.scale), c, cache=want)
    c.qkv[:] = good
    _, _, k, v, _, _ = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert_cache(cache, oracle_write(c))


def test_rotation_past_the_largest_number_is_not_finite():
    """A rotated k above 65504 is no fp16 number: its token is NaN in that head."""
    c = Case((1, 1, 64), [(0, 3)], seed=54)
    c.qkv[:, :] = 0.25
    c.qkv[1, 64], c.qkv[1, 96] = 60000.0, 60000.0
    qkv, q, _, _, cache, meta = c.on(DEV)
    cos, sin = rope_tables(64, 1e6, 8, DEV)
    H.rope_kv_write_int4(qkv, torch.tensor([0, 1, 2], device=DEV), cos, sin, 1, 1, 64, cache[0, 0], cache[0, 1],
                         meta.slot_mapping)
    _, kn, _ = c.split()
    turned = O.rotate(kn, cos.cpu().numpy()[:3], sin.cpu().numpy()[:3])
    assert np.abs(turned[1]).max() > 65504
    want = oracle_write(c, k=turned)
    assert_cache(cache, want)
    out = attend(q, cache, meta, c.scale)
    assert torch.isfinite(out[0]).all() and out[1:].isnan().all()


def test_write_skips_padding_and_foreign_slots():
    c = Case((4, 2, 32), [(7, 1), (0, 1), (3, 1), (9, 40), (0, 25)], num_decode=3, seed=5)
    c.slots[[1, 5, 9, 20, 30]] = [-1, 16 * c.NB, 2 ** 40, -2 ** 40, -17]
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert_cache(cache, oracle_write(c))


def test_write_layouts_and_refusals():
    """int32 slots, a longer slot mapping, strided ones, separate k / v tensors; what is refused."""
    c = Case((4, 2, 64), [(7, 1), (3, 1), (9, 100), (0, 25)], num_decode=2, seed=7)
    _, _, k, v, start, meta = c.on(DEV)
    want = oracle_write(c)
    s = meta.slot_mapping
    for slots in (s.int(), torch.cat([s, s.new_full((9,), 3)]), s.repeat_interleave(2)[::2]):
        cache = start.clone()
        H.kv_write_int4(k.contiguous(), v, cache[0, 0], cache[0, 1], slots)
        assert_cache(cache, want)
    layer = start[0, 0], start[0, 1]
    with pytest.raises(ValueError, match="unit stride"):
        H.kv_write_int4(k.transpose(0, 2).contiguous().transpose(0, 2), v, *layer, s)
    with pytest.raises(ValueError, match="fp16"):
        H.kv_write_int4(k.float(), v.float(), *layer, s)
    odd = torch.empty(k.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(k.shape)
    with pytest.raises(ValueError, match="aligned"):
        H.kv_write_int4(odd, v, *layer, s)
    with pytest.raises(ValueError, match="shorter"):
        H.kv_write_int4(k, v, *layer, s[:-1])
    with pytest.raises(ValueError, match="same GPU"):
        H.kv_write_int4(k, v, *layer, s.cpu())
    with pytest.raises(ValueError, match="mismatch"):
        H.kv_write_int4(k[:, :1], v[:, :1], *layer, s)


def test_strides_of_axes_of_one_element_do_not_matter():
    """One row, or one KV head, cut out of rows of an odd width."""
    c = Case((1, 1, 64), [(4, 1)], num_decode=1, seed=40)
    qkv, q, k, v, cache, meta = c.on(DEV)
    slots = meta.slot_mapping
    start = cache.clone()
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], slots)
    want = attend(q, cache, meta, c.scale)
    cos, sin = rope_tables(64, 1e6, 8, DEV)
    pos = torch.from_numpy(c.pos).to(DEV)
    turned = start.clone()
    rotated = H.rope_kv_write_int4(qkv, pos, cos, sin, 1, 1, 64, turned[0, 0], turned[0, 1], slots)

    def odd(x):                                      # x [1, ...] at the start of a row of 4097 elements
        wide = torch.zeros(2, 4097, dtype=x.dtype, device=DEV)
        wide[0, :x.numel()] = x.flatten()
        return wide[:1, :x.numel()].as_strided(x.shape, (4097,) * (x.dim() - 1) + (1,))

    mine = start.clone()
    H.kv_write_int4(odd(k), odd(v), mine[0, 0], mine[0, 1], slots)
    assert torch.equal(mine, cache)
    assert torch.equal(attend(odd(q), mine, meta, c.scale), want)
    mine = start.clone()
    wide = torch.zeros(1, 193, dtype=torch.float16, device=DEV)
    wide[:, :192] = qkv
    got = H.rope_kv_write_int4(wide, pos, cos, sin, 1, 1, 64, mine[0, 0], mine[0, 1], slots)
    assert torch.equal(got, rotated) and torch.equal(mine, turned)


def test_rope_write_clamps_positions_and_takes_one_row():
    c = Case((2, 1, 16), [(4, 1)], num_decode=1, seed=8)
    qkv, _, _, _, cache, meta = c.on(DEV)
    cos, sin = rope_tables(16, 1e6, 8, DEV)
    last = cache.clone()
    a = H.rope_kv_write_int4(qkv, torch.tensor([10 ** 9], device=DEV), cos, sin, 2, 1, 16, cache[0, 0],
                             cache[0, 1], meta.slot_mapping)
    b = H.rope_kv_write_int4(qkv, torch.tensor([7], device=DEV), cos, sin, 2, 1, 16, last[0, 0], last[0, 1],
                             meta.slot_mapping)
    assert torch.equal(a, b) and torch.equal(cache, last)


@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_the_cache_is_near_that_over_the_rows(heads):
    near_the_rows(H, DEV, heads)


def test_appends_row_by_row_in_a_replayed_graph():
    """Forty single-row steps through one captured write, each checked."""
    c = Case((4, 2, 64), [(0, 40), (13, 40)], seed=9)
    _, kn, vn = c.split()
    _, _, k, v, cache, meta = c.on(DEV)
    kk, vv = k[:2].contiguous(), v[:2].contiguous()
    slots = torch.full((2,), -1, dtype=torch.int64, device=DEV)
    H.kv_write_int4(kk, vv, cache[0, 0], cache[0, 1], slots)     # writes nothing
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        H.kv_write_int4(kk, vv, cache[0, 0], cache[0, 1], slots)
    want = c.cache
    for i in range(40):
        rows = [i, 40 + i]
        kk.copy_(k[rows])
        vv.copy_(v[rows])
        slots.copy_(torch.from_numpy(c.slots[rows]))
        graph.replay()
        O.write(kn[rows], vn[rows], *want, c.slots[rows])
        assert_cache(cache, want, f"step {i}")


def test_past_two_to_the_31_bytes():
    """Blocks far into a large cache (offsets above 2^31), and its first ones left alone."""
    unit = O.unit_bytes(128)
    nb = (1 << 31) // (2 * unit) + 50
    c = Case((2, 2, 128), [(20, 1), (0, 33)], num_decode=1, seed=10)
    up = nb - c.NB
    high = c.tables + up
    high[c.tables == 0] = 0
    data = torch.zeros(1, 2, nb, 2, unit, dtype=torch.uint8, device=DEV)
    data[:, :, up:] = torch.from_numpy(c.cache).to(DEV)
    _, q, k, v, _, meta = c.on(DEV)
    meta = dataclasses.replace(meta, block_tables=torch.from_numpy(high).to(DEV),
                               slot_mapping=meta.slot_mapping + 16 * up)
    H.kv_write_int4(k, v, data[0, 0], data[0, 1], meta.slot_mapping)
    want = oracle_write(c)
    assert_cache(data[:, :, up:], want)
    assert not data[:, :, :up].any()
    for bound in (33, 30000):                        # tiles of 16 rows, the prompt kernel
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(attend(q, data, m, c.scale), c, f"{bound}", cache=want)
    got = H.kv_read_int4(data, torch.from_numpy(high[0]).to(DEV)).cpu().numpy()
    for j in range(2):
        assert np.array_equal(got[0, j, :2], O.values_of(*O.unpack(want[j], 128, bool(j)))[c.tables[0, :2]])


# ------------------------------------------------------------------------------------- decode
DECODE_LENS = [1, 2, 15, 16, 17, 31, 33, 128, 255, 256, 257, 500, 513, 1000, 1025, 4096]


@pytest.mark.parametrize("heads", HEADS)
def test_decode_matches_the_oracle(heads):
    c = Case(heads, [(n - 1, 1) for n in DECODE_LENS], num_decode=len(DECODE_LENS), seed=11)
    _, q, _, _, cache, meta = c.on(DEV)
    want = c.cache
    assert_rows(attend(q, cache, meta, c.scale), c, f"decode {heads}", cache=want)
    # the host's bound on the lengths decides the splits only
    for bound in (0, 1, 300, 40000):
        m = dataclasses.replace(meta, max_seq_len=bound)
        assert_rows(attend(q, cache, m, c.scale), c, f"decode {heads} bound {bound}", cache=want)


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64), (1, 1, 16)])
def test_decode_of_a_long_sequence(heads):
    """More blocks than the splits of 16 hold, and more than a split looks up at once."""
    c = Case(heads, [(69999, 1), (16384, 1)], num_decode=2, seed=12)
    _, q, _, _, cache, meta = c.on(DEV)
    want = c.cache
    assert_rows(attend(q, cache, meta, c.scale), c, f"long {heads}", cache=want)
    short = dataclasses.replace(meta, max_seq_len=64)         # one split of 4375 blocks
    assert_rows(attend(q, cache, short, c.scale), c, f"long, unsplit {heads}", cache=want)


@pytest.mark.parametrize("rows,bound", [(1, 1), (2, 2), (2, 200)])   # a decode row, a short chunk, the prompt kernel
def test_the_longest_table(rows, bound):
    """2^26 blocks, the longest table that is taken (its entries repeat): K of zeros, V of 64 in all blocks
    but the last 64th, -64 there. Every sum of these is exact, and their mean is 62 (for the row before the
    last one, too, once it is rounded)."""
    nb = 1 << 26
    data = torch.zeros(1, 2, 3, 1, O.unit_bytes(16), dtype=torch.uint8, device=DEV)
    zeros, wide = torch.zeros(48, 1, 16, device=DEV).half(), torch.zeros(48, 1, 16, device=DEV).half()
    wide[16:32], wide[32:] = 64, -64
    H.kv_write_int4(zeros, wide, data[0, 0], data[0, 1], torch.arange(48, device=DEV))
    table = torch.ones(1, nb, dtype=torch.int32, device=DEV)
    table[0, nb - nb // 64:] = 2
    c = Case((1, 1, 16), [(0, rows)])
    _, q, _, _, _, _ = c.on(DEV)
    meta = c.meta(DEV, seq_lens=torch.tensor([16 * nb], dtype=torch.int32, device=DEV), block_tables=table,
                  num_decode=int(rows == 1), max_query_len=bound, max_seq_len=16 * nb,
                  max_prefill_seq_len=16 * nb)
    out = attend(q, data, meta, c.scale)
    assert out.eq(62).all(), out


def test_decode_rows_do_not_depend_on_the_batch():
    c = Case((12, 2, 128), [(n - 1, 1) for n in DECODE_LENS * 5], num_decode=5 * len(DECODE_LENS), seed=13)
    _, q, _, _, cache, meta = c.on(DEV)
    whole = attend(q, cache, meta, c.scale)
    for i in (3, 30, 79):
        one = dataclasses.replace(meta, seq_lens=meta.seq_lens[i:i + 1], num_decode=1,
                                  block_tables=meta.block_tables[i:i + 1],
                                  query_start_loc=meta.query_start_loc[:2])
        assert torch.equal(attend(q[i:i + 1], cache, one, c.scale)[0], whole[i])


@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 1, 256), (14, 2, 64), (4, 2, 16)])
def test_one_decode_row_over_tables_of_any_width(heads):
    """One sequence's splits start up to 15 blocks before a multiple of 16, or anywhere (past 1024 blocks):
    lengths at those edges, over tables that end with the sequence or before it, among foreign ids."""
    for n in (0, 1, 16, 17, 256, 257, 271, 273, 289, 545, 1009, 4081, 16384, 16385, 16700):
        c = Case(heads, [(max(n - 1, 0), 1)], num_decode=1, seed=n)
        c.lens[:] = n
        _, q, _, _, cache, meta = c.on(DEV)
        want = c.cache
        assert_rows(attend(q, cache, meta, c.scale), c, f"{n} tokens", cache=want)
        if n > 32:
            c.tables = np.ascontiguousarray(c.tables[:, :n // 16 - 1])
            bad = torch.from_numpy(c.tables).to(DEV)
            bad[0, 1], bad[0, -1] = c.NB + 7, -1
            c.tables[0, 1] = c.tables[0, -1] = 0
            m = dataclasses.replace(meta, block_tables=bad)
            assert_rows(attend(q, cache, m, c.scale), c, f"{n} tokens, fewer blocks", cache=want)


def test_decode_of_more_rows_than_a_lookup_holds():
    """300 sequences, some empty: rows without tokens are zeros."""
    lens = [(7 * i) % 40 for i in range(300)]
    c = Case((4, 2, 16), [(max(n - 1, 0), 1) for n in lens], num_decode=300, seed=14)
    c.lens[:] = lens
    _, q, _, _, cache, meta = c.on(DEV)
    out = attend(q, cache, meta, c.scale)
    assert_rows(out, c)
    assert not out[torch.tensor(lens, device=DEV) == 0].any()


@pytest.mark.parametrize("heads,far", [((8, 8, 64), 1400), ((28, 4, 128), 2800), ((4, 1, 256), 5000)])
def test_more_splits_than_workgroups(heads, far):
    """60 sequences, some without tokens, whose splits are more than the chip holds at once: decode rows alone,
    the same bits as one by one, then half of them as short chunks."""
    lens = [(far // 15 * i + 7 * i) % far for i in range(60)]
    c = Case(heads, [(max(n - 1, 0), 1) for n in lens], num_decode=60, seed=54)
    c.lens[:] = lens
    assert sum(max(1, -(-n // 256)) for n in lens) * c.KVH > (512 if c.D > 128 else 1024)
    _, q, _, _, cache, meta = c.on(DEV)
    out = attend(q, cache, meta, c.scale)
    assert_rows(out, c, "decode rows")
    for i in (1, 31, 59):
        one = dataclasses.replace(meta, seq_lens=meta.seq_lens[i:i + 1], num_decode=1,
                                  block_tables=meta.block_tables[i:i + 1],
                                  query_start_loc=meta.query_start_loc[:2])
        assert torch.equal(attend(q[i:i + 1], cache, one, c.scale)[0], out[i])
    c = Case(heads, [(max(n - 1, 0), 1 + i % 5 * (i > 29)) for i, n in enumerate(lens)], num_decode=30, seed=55)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(attend(q, cache, meta, c.scale), c, "beside chunks")


@pytest.mark.parametrize("k_size", [0.0, 1e-4, 30.0, 3000.0])
def test_decode_of_flat_and_steep_scores(k_size):
    c = Case((12, 2, 128), [(n - 1, 1) for n in (1, 40, 700, 2000)], num_decode=4, seed=15, k_size=k_size)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(attend(q, cache, meta, c.scale), c, f"k of {k_size}")


def test_more_heads_than_a_chunk_may_have_rows():
    """300 query heads of one KV head: 19 tiles of 16 rows for one token."""
    c = Case((300, 1, 16), [(4000, 1), (20, 1), (900, 3)], num_decode=2, seed=35)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(attend(q, cache, meta, c.scale), c)


@pytest.mark.parametrize("heads", [(4, 2, 16), (14, 2, 64)])
def test_one_long_prompt_among_many_short_ones(heads):
    c = Case(heads, [(5, 1)] * 3 + [(0, 3)] * 70 + [(40, 700)] + [(2, 9)] * 60, num_decode=3, seed=33)
    _, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    want = oracle_write(c)
    assert_cache(cache, want)
    for bounds in (dict(), dict(max_query_len=9, max_prefill_seq_len=60), dict(max_prefill_seq_len=30000)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(attend(q, cache, m, c.scale), c, f"{bounds}", cache=want)


def test_decode_graph_replayed_over_growing_sequences():
    """A captured step of two layers (writes, attention) with max_seq_len of the longest that it may meet,
    replayed while the lengths grow, with eager calls between the replays."""
    c = Case((12, 2, 128), [(0, 600), (0, 600), (0, 600)], seed=24)
    _, kn, vn = c.split()
    _, q, k, v, cache, meta = c.on(DEV)
    cache = torch.cat([cache, cache.flip(2)]).contiguous()
    qq, kk, vv = (x[:3].contiguous() for x in (q, k, v))
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    slots = torch.full((3,), -1, dtype=torch.int64, device=DEV)
    step = c.meta(DEV, seq_lens=lens, num_decode=3, max_query_len=1, max_seq_len=600, slot_mapping=slots,
                  query_start_loc=torch.arange(4, dtype=torch.int32, device=DEV))

    def once():
        outs = []
        for i in range(2):
            H.kv_write_int4(kk, vv, cache[i, 0], cache[i, 1], slots)
            outs.append(H.paged_attention_int4(qq, cache[i, 0], cache[i, 1], step, c.scale))
        return torch.stack(outs)

    assert not once().any()                           # lengths 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    want = c.cache
    for now in ([1, 17, 255], [2, 18, 256], [3, 0, 257], [4, 19, 258], [511, 20, 0], [512, 21, 600]):
        rows = [max(n - 1, 0) + 600 * b for b, n in enumerate(now)]
        mine = np.where(np.array(now) > 0, c.slots[rows], -1)
        qq.copy_(q[rows]), kk.copy_(k[rows]), vv.copy_(v[rows])
        lens.copy_(torch.tensor(now)), slots.copy_(torch.from_numpy(mine))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, once()), now
        O.write(kn[rows], vn[rows], *want, mine)
        assert_cache(cache[:1], want, str(now))
        ref, bound = O.paged_attention(c.split()[0][rows], *want, c.tables, now, [0, 1, 2, 3], c.scale)
        assert (np.abs(got[0].double().cpu().numpy() - ref) <= bound).all(), str(now)


# ------------------------------------------------------------------------------------- several rows
PREFILL = [(0, 1), (0, 15), (15, 16), (37, 16), (1000, 17), (0, 300), (16, 530), (63, 65), (4000, 5)]


@pytest.mark.parametrize("heads", HEADS)
def test_prefill_matches_the_oracle(heads):
    c = Case(heads, PREFILL, seed=17)
    _, q, _, _, cache, meta = c.on(DEV)
    want = c.cache
    assert_rows(attend(q, cache, meta, c.scale), c, f"prefill {heads}", cache=want)
    # host bounds below the batch's own, and far above it
    for bounds in (dict(max_query_len=1), dict(max_query_len=40, max_prefill_seq_len=100, max_seq_len=100),
                   dict(max_query_len=2000, max_prefill_seq_len=30000, max_seq_len=30000),
                   dict(max_query_len=0, max_prefill_seq_len=0, max_seq_len=0)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(attend(q, cache, m, c.scale), c, f"prefill {heads} {bounds}", cache=want)


VERIFY = [(0, 5), (1, 5), (12, 3), (300, 5), (2047, 4), (9, 1), (255, 2), (5000, 5), (4094, 5)]


@pytest.mark.parametrize("heads", HEADS)
def test_a_few_rows_per_sequence(heads):
    """The rows of a speculative step: up to five a sequence, beside decode rows."""
    c = Case(heads, [(100, 1), (0, 1)] + VERIFY, num_decode=2, seed=30)
    c.lens[3] = 3                                    # five rows, three positions
    _, q, _, _, cache, meta = c.on(DEV)
    want = c.cache
    out = attend(q, cache, meta, c.scale)
    assert_rows(out, c, f"verify {heads}", cache=want)
    assert not out[int(c.starts[3]):int(c.starts[3]) + 2].any()
    for bounds in (dict(max_query_len=2), dict(max_seq_len=100, max_prefill_seq_len=0),
                   dict(max_query_len=200), dict(num_decode=0)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(attend(q, cache, m, c.scale), c, f"verify {heads} {bounds}", cache=want)


@pytest.mark.parametrize("heads", HEADS)
def test_short_chunks_beside_long_prefixes(heads):
    """Up to 21 rows a sequence: several tiles of 16 rows whose splits are merged, with as many
    partials in the workspace as one tile has."""
    items = [(4200, 16), (300, 21), (2047, 9), (20000, 12), (0, 21), (100, 1), (33, 20)]
    c = Case(heads, [(1500, 1)] + items, num_decode=1, seed=32)
    _, q, _, _, cache, meta = c.on(DEV)
    want = c.cache
    assert_rows(attend(q, cache, meta, c.scale), c, f"short chunks {heads}", cache=want)
    # host bounds below the batch's own leave fewer partials: fewer splits
    for bounds in (dict(max_query_len=3), dict(max_query_len=8, max_seq_len=900, max_prefill_seq_len=900),
                   dict(max_query_len=1, max_seq_len=20100, max_prefill_seq_len=20100)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(attend(q, cache, m, c.scale), c, f"short chunks {heads} {bounds}", cache=want)


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64)])
def test_prefill_over_a_long_prefix(heads):
    """More blocks than are looked up at once, and split along the keys."""
    c = Case(heads, [(9000, 70), (3, 200), (30000, 3)], seed=18)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(attend(q, cache, meta, c.scale), c, f"long prefix {heads}")


@pytest.mark.parametrize("heads", HEADS)
def test_mixed_batch(heads):
    """Decode rows beside chunks, a padding row, a sequence without positions, rows behind the last
    sequence, which keep what stood there; the step's write before the attention."""
    items = [(40, 1), (0, 1), (777, 1), (0, 20), (100, 130), (5, 3)]
    c = Case(heads, items, num_decode=3, seed=19, tail_rows=2)
    c.lens[1] = 0
    c.slots[1] = -1
    c.lens[5] = 2                                    # three rows, two positions
    _, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    want = oracle_write(c)
    assert_cache(cache, want)
    for bound in (777, 30000):                       # tiles of 16 rows, the prompt kernel
        out = attend(q, cache, dataclasses.replace(meta, max_prefill_seq_len=bound), c.scale)
        assert_rows(out, c, f"mixed {heads} {bound}", cache=want)
        assert not out[1].any() and not out[int(c.starts[5])].any()


def test_rows_behind_the_last_sequence_are_not_written():
    from turingserve_amd import _native as N

    c = Case((4, 2, 64), [(40, 1), (100, 130)], num_decode=1, seed=55, tail_rows=3)
    _, q, _, _, cache, meta = c.on(DEV)
    out = torch.full((c.T, 256), 7.0, dtype=torch.float16, device=DEV)
    for bound in (230, 30000):
        size = N.lib().ts_paged_attention_int4_workspace_bytes(2, 1, 130, 230, bound, 4, 2, 64, 256)
        ws = torch.empty(size + 256, dtype=torch.uint8, device=DEV)
        N.check(N.lib().ts_paged_attention_int4(
            q.data_ptr(), q.stride(0), 64, out.data_ptr(), 256, c.T, cache[0, 0].data_ptr(),
            cache[0, 1].data_ptr(), c.NB, meta.block_tables.data_ptr(), c.tables.shape[1], c.tables.shape[1],
            meta.seq_lens.data_ptr(), meta.query_start_loc.data_ptr(), 2, 1, 130, 230, bound, 4, 2, 64, c.scale,
            ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream), "attention")
        assert_rows(out, c)
        assert out[-3:].eq(7).all()


def test_sequences_without_rows():
    """Sequences of no new rows between the others, and a step of rows that belong to none."""
    c = Case((14, 2, 64), [(100, 1), (40, 0), (0, 0), (5, 20), (300, 0), (70, 60)], num_decode=1, seed=37)
    _, q, _, _, cache, meta = c.on(DEV)
    want = c.cache
    for bound in (300, 30000):
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(attend(q, cache, m, c.scale), c, f"{bound}", cache=want)
    none = dataclasses.replace(meta, seq_lens=meta.seq_lens[:0], block_tables=meta.block_tables[:0],
                               query_start_loc=meta.query_start_loc[:1], num_decode=0)
    assert attend(q, cache, none, c.scale).shape == (c.T, c.H * c.D)


def test_table_shorter_than_the_sequence():
    c = Case((14, 2, 64), [(299, 1), (50, 200)], num_decode=1, seed=20)
    c.tables = np.ascontiguousarray(c.tables[:, :8])          # 128 tokens of 300 and 250
    _, q, _, _, cache, meta = c.on(DEV)
    for bound in (300, 30000):
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(attend(q, cache, m, c.scale), c, f"{bound}")


def test_foreign_block_ids_read_block_zero():
    c = Case((14, 2, 64), [(99, 1), (50, 60)], num_decode=1, seed=21)
    _, q, _, _, cache, meta = c.on(DEV)
    bad = meta.block_tables.clone()
    bad[0, 2], bad[1, 3] = c.NB + 100, -5
    c.tables[0, 2] = c.tables[1, 3] = 0
    for bound in (100, 30000):
        m = dataclasses.replace(meta, block_tables=bad, max_prefill_seq_len=bound)
        assert_rows(attend(q, cache, m, c.scale), c, f"{bound}")


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("bound", [501, 30000])      # tiles of 16 rows, the prompt kernel
def test_tokens_that_are_not_finite(heads, side, bound):
    """Rows that see such a token are NaN, rows before it (and other sequences and heads) are within the
    bound; blocks past a sequence's end, and rows past its last one, have no say."""
    c = Case(heads, [(100, 1), (500, 1), (5, 150), (0, 40)], num_decode=2, seed=22)
    cache = c.cache
    g, kvh, d = c.H // c.KVH, c.KVH, c.D
    k, v = np.zeros((2, 3, kvh, d), np.float32)
    (k, v)[side][:2, 0, 1] = [np.inf, np.nan]
    # position 322 of the second sequence, 80 of the third; the row behind the first one's last
    k[2], v[2] = np.nan, np.inf
    O.write(k, v, *cache, [c.tables[1, 20] * 16 + 2, c.tables[2, 5] * 16, c.tables[0, 6] * 16 + 101 % 16])
    unused = sorted(set(range(c.NB)) - set(c.tables.ravel().tolist()))
    nan = np.full((16 * len(unused), kvh, d), np.nan, np.float32)
    O.write(nan, nan, *cache, np.concatenate([np.arange(16) + 16 * u for u in unused]))
    _, q, _, _, _, meta = c.on(DEV)
    meta = dataclasses.replace(meta, max_prefill_seq_len=bound)
    out = attend(q, torch.from_numpy(cache).to(DEV)[None], meta, c.scale)
    hit = np.zeros((c.T, c.H), bool)
    hit[1, :g] = True
    lo = int(c.starts[2])
    hit[lo + 75:lo + 150, :g] = True                 # rows at positions 80 and later
    got = out.cpu().numpy().reshape(c.T, c.H, c.D)
    assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()
    assert_rows(out, c, cache=cache)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("bound", [90, 30000])      # tiles of 16 rows, the prompt kernel
def test_hidden_tokens_have_no_say(heads, bound):
    """Whatever stands in the tokens that a row does not see, its bits are the same, and rows that see
    small values ahead of hidden ones of the largest are as exact as alone."""
    c = Case(heads, [(0, 90), (0, 90)], seed=38)
    _, q, _, _, cache, meta = c.on(DEV)
    meta = dataclasses.replace(meta, max_prefill_seq_len=bound)
    out = attend(q, cache, meta, c.scale)
    assert_rows(out, c)
    big = torch.empty(2, 67, c.KVH, c.D, device=DEV).uniform_(-60000, 60000).half()
    other = cache.clone()
    for b in range(2):                               # tokens 23 and later of both
        slots = torch.from_numpy(c.slots[int(c.starts[b]) + 23:int(c.starts[b + 1])]).to(DEV)
        H.kv_write_int4(big[0], big[1], other[0, 0], other[0, 1], slots)
    again = attend(q, other, meta, c.scale)
    for lo in c.starts[:2].tolist():
        assert torch.equal(out[lo:lo + 23], again[lo:lo + 23])
        assert not torch.equal(out[lo + 23:lo + 90], again[lo + 23:lo + 90])


def test_attention_refuses():
    c = Case((4, 2, 64), [(7, 1), (9, 20)], num_decode=1, seed=23)
    _, q, _, _, cache, meta = c.on(DEV)
    with pytest.raises(ValueError, match="fp16"):
        attend(q.float(), cache, meta, c.scale)
    with pytest.raises(ValueError, match="unit stride"):
        attend(q.transpose(0, 2).contiguous().transpose(0, 2), cache, meta, c.scale)
    with pytest.raises(ValueError, match="scale"):
        attend(q, cache, meta, -1.0)
    with pytest.raises(ValueError, match="same GPU"):
        attend(q, cache, dataclasses.replace(meta, seq_lens=meta.seq_lens.cpu()), 1.0)
    odd = torch.empty(q.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(q.shape)
    with pytest.raises(ValueError, match="misaligned"):
        attend(odd, cache, meta, c.scale)
    for change in (dict(num_decode=3), dict(num_decode=-1), dict(query_start_loc=meta.query_start_loc[:2]),
                   dict(block_tables=meta.block_tables[:1])):
        with pytest.raises(ValueError, match="metadata of 2"):
            attend(q, cache, dataclasses.replace(meta, **change), c.scale)
    assert attend(q[:0], cache, meta, c.scale).shape == (0, 256)


def test_chunk_graphs_of_one_pool():
    """Two captured mixed steps (one for each of the attention's kernels) whose workspaces share a
    memory pool, replayed in turn with other inputs each time and eager calls in between."""
    c = Case((14, 2, 64), [(900, 1), (300, 40), (0, 500), (17, 1)], num_decode=1, seed=36)
    _, q, k, v, cache, meta = c.on(DEV)
    start = cache.clone()
    qq, kk, vv = q.clone(), k.clone(), v.clone()
    metas = [dataclasses.replace(meta, max_prefill_seq_len=b) for b in (500, 30000)]

    def step(m):
        H.kv_write_int4(kk, vv, cache[0, 0], cache[0, 1], m.slot_mapping)
        return attend(qq, cache, m, c.scale)

    for m in metas:
        step(m)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m in metas:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            outs.append(step(m))
    for turn in range(3):
        for g, out, m in zip(graphs, outs, metas):
            qq.copy_(q.roll(turn, 0)), kk.copy_(k.roll(turn, 0)), vv.copy_(v.roll(-turn, 0))
            cache.copy_(start)
            g.replay()
            got, after = out.clone(), cache.clone()
            cache.copy_(start)
            assert torch.equal(step(m), got) and torch.equal(after, cache), turn
        _, kn, vn = c.split()
        want = oracle_write(c, np.roll(kn, turn, 0), np.roll(vn, -turn, 0))
        assert_cache(cache, want)
        assert_rows(got, c, f"{turn}", cache=want, q=np.roll(c.split()[0], turn, 0))


def test_two_streams_at_once():
    """The same calls on two streams, workspaces of their own each."""
    c = Case((12, 2, 128), [(3000, 1), (1000, 1), (500, 90)], num_decode=2, seed=25)
    _, q, _, _, cache, meta = c.on(DEV)
    want = attend(q, cache, meta, c.scale)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(attend(q, cache, meta, c.scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------------------------- together
def test_model_step_matches_the_reference_twins():
    """A chunked prompt beside decode rows through the whole model, 4-bit cache: hip against the
    reference namespace. Both round activations to fp16 at other places, and a rounded k can land on the
    neighbouring code, a step of a fifteenth of its group's span rather than one of 255ths of the
    block's: as many of them as the 8-bit cache's, each 17 times as large, so the bar is 17 times the
    part of its 2e-2 that codes have (fp16's own bar is 1e-2): 0.18."""
    from turingserve_amd.metadata import BatchItem, InputBuilder, SeqState
    from turingserve_amd.qwen2 import Qwen2Config, Qwen2Model, random_weights

    cfg = Qwen2Config(256, 512, 2, 4, 2, 500, max_position_embeddings=512)
    w = random_weights(cfg, DEV, seed=26, draw_on="cpu", init_std=0.06)
    g = torch.Generator().manual_seed(27)
    seqs = [SeqState(torch.randint(0, 500, (200,), generator=g).tolist(), list(range(1 + 13 * i, 14 + 13 * i)))
            for i in range(3)]
    logits = {}
    for name in ("hip", "reference"):
        model = Qwen2Model(cfg, w, get_ops(name), 512)
        kv = model.new_kv_cache(40, "int4")
        assert isinstance(kv, Int4KVCache)
        builder = InputBuilder(256, 8, 13, DEV)
        got = []
        for items in ([BatchItem(seqs[0], 0, seqs[0].token_ids[:50]), BatchItem(seqs[1], 0, seqs[1].token_ids[:33])],
                      [BatchItem(seqs[0], 50, seqs[0].token_ids[50:51]), BatchItem(seqs[1], 33, seqs[1].token_ids[33:34]),
                       BatchItem(seqs[2], 0, seqs[2].token_ids[:70])],
                      [BatchItem(s, n, s.token_ids[n:n + 1]) for s, n in zip(seqs, (51, 34, 70))]):
            inp = builder.build(items)
            got.append(model.compute_logits(model.forward(inp.input_ids, inp.positions, inp.meta, kv),
                                            inp.sample_indices))
        logits[name] = torch.cat(got)
    a, b = logits["hip"], logits["reference"]
    assert torch.isfinite(a).all()
    assert float((a - b).norm() / b.norm()) < 0.18


def test_engine_tokens_with_graphs_equal_eager():
    from turingserve_amd.engine import GreedyEngine
    from turingserve_amd.qwen2 import TINY_G2, Qwen2Model, random_weights

    model = Qwen2Model(TINY_G2, random_weights(TINY_G2, DEV, seed=28), get_ops("hip"), 1024)
    g = torch.Generator().manual_seed(29)
    prompts = [torch.randint(0, TINY_G2.vocab_size, (n,), generator=g).tolist() for n in (100, 3, 47, 300)]
    outs = []
    for sizes, dev_meta in (((), False), ((1, 2, 4), False), ((4,), True)):
        eng = GreedyEngine(model, 128, max_num_batched_tokens=128, graph_sizes=sizes,
                           device_metadata=dev_meta, kv_cache_dtype="int4")
        outs.append(eng.generate(prompts, 24))
        assert bool(sizes) == (eng.graph_steps > 0) and eng.mixed_steps > 0
    assert outs[0] == outs[1] == outs[2]


def _small(case):
    """A case of perf/more_operators.py with the same structure and fewer, shorter sequences."""
    most = dict(layers=2, decodes=5, ctx_lo=200, ctx_hi=700, chunks=3, q_lo=90, q_hi=150, prefix_lo=100, prefix_hi=333)
    return {k: min(v, most[k]) if k in most else v for k, v in case.items()}


def _case_names():
    from perf import more_operators
    return [c["name"] for c in more_operators.listed()]


@pytest.mark.parametrize("name", _case_names())
def test_cases_as_a_program_calls_them(name, monkeypatch):
    """The measured cases' calls (the split map of a decode step, its graph, layers with caches of their own,
    the read-back) at small sizes, twice over the same state, against their results in 64 bits. Written
    values are equal. A rotated q: a product and a fused product-sum in fp32, then fp16. Attention, with V
    the largest value: a score is a sum of D products in fp32, off by e = (D + 8) 2^-24 scale |q| |k| and the
    exponential's 2^-22, a weight by a factor within e^(+-2 e); a weight is rounded to fp16, by 2^-11 of it or
    2^-25 of the largest; sums over n tokens as in oracle.int8_cache.paged_attention; the result rounds once."""
    from perf import more_operators as cases

    case = _small(next(c for c in cases.listed() if c["name"] == name))
    monkeypatch.setattr(cases, "own", True)
    state = cases.prepare(case, 7)
    want = cases.exact(case, 7)
    h, d = case["heads"], case["head_dim"]
    assert ("graph" in state) == (case["chunks"] == 0 and case["kind"] != "read")
    for _ in range(2):
        out = cases.run(state)
        torch.cuda.synchronize()
        if case["kind"] == "read":
            assert torch.equal(out.double(), want)
            continue
        if case["kind"] == "write":
            assert torch.equal(out["cache"].double(), want["cache"])
            assert len(out["q"]) == len(want["q"]) == (case["layers"] if case["rope"] else 0)
            for i, (a, b) in enumerate(zip(out["q"], want["q"])):
                x = state["q"][i].double().abs()
                size = x + torch.cat([x[..., d // 2:], x[..., :d // 2]], -1)
                assert ((a.double() - b).abs() <= 2.0 ** -11 * b.abs() + 2.0 ** -23 * size + 2.0 ** -25).all()
            continue
        n, u = state["batch"]["max_seq_len"], 2.0 ** -24
        held = H.kv_read_int4(state["cache"].data, torch.arange(state["batch"]["blocks"], device=DEV)).double()
        assert len(out) == len(want) == case["layers"]
        for i, (a, b) in enumerate(zip(out, want)):
            v = float(held[i, 1].abs().max())
            reach = float(state["q"][i].double().norm(dim=-1).max() * held[i, 0].norm(dim=-1).max()) * state["scale"]
            e = (d + 8) * u * reach + 2.0 ** -22
            off = (math.expm1(2 * e) + 2.0 ** -11 + n * 2.0 ** -25 + (n / 32 + 16) * u
                   + 8 * u * math.sqrt(n + 256)) * v
            assert a.shape == b.shape == (state["q"].shape[1], h * d)
            assert ((a.double() - b).abs() <= off + 2.0 ** -11 * (b.abs() + off) + 2.0 ** -25).all()


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("kind", TINY)
def test_rope_write_of_tiny_rows(heads, kind):
    """Byte for byte, rotated and as they are: a least number that is or rounds to -0 is 0, and so is the step of
    a group of such."""
    h, kvh, d = heads
    c = tiny_rows(heads, kind)
    qkv, _, _, _, cache, meta = c.on(DEV)
    cos, sin = rope_tables(d, 1e6, 64, DEV)
    H.rope_kv_write_int4(qkv, torch.from_numpy(c.pos).to(DEV), cos, sin, h, kvh, d, cache[0, 0], cache[0, 1],
                         meta.slot_mapping)
    _, kn, _ = c.split()
    turned = O.rotate(kn, cos.cpu().numpy()[c.pos], sin.cpu().numpy()[c.pos])
    assert_cache(cache, oracle_write(c, k=turned), f"{heads} {kind}")
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert_cache(cache, oracle_write(c), f"{heads} {kind} as they are")


@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_the_cache_is_that_over_coherent_rows(heads):
    c = coherent_rows(heads)
    out, cache = over_the_cache(H, DEV, c)
    ref, bar = over_the_rows(c, cache)
    assert not outside(c, out, ref, bar).any()


def test_model_over_the_cache_is_the_fp16_model_over_what_it_holds():
    """Each step through the model with a 4-bit cache, then through the same model over that cache read back
    as fp16, its own new rows going to blocks behind it that no table names: both attend the same numbers, and
    differ by fp16's roundings alone (bar 1e-2, a fifth at most of what the 4 bits themselves move the
    logits by). Of every layer, the rows held are those that the fp16 model wrote, within half a step (and the
    1e-2 of the activations)."""
    from turingserve_amd.metadata import BatchItem, InputBuilder, SeqState
    from turingserve_amd.qwen2 import Qwen2Config, Qwen2Model, random_weights

    layers, blocks = 3, 40
    cfg = Qwen2Config(256, 512, layers, 4, 2, 500, max_position_embeddings=512)
    model = Qwen2Model(cfg, random_weights(cfg, DEV, seed=26, draw_on="cpu", init_std=0.06), get_ops("hip"), 512)
    g = torch.Generator().manual_seed(27)
    seqs = [SeqState(torch.randint(0, 500, (200,), generator=g).tolist(), list(range(1 + 13 * i, 14 + 13 * i)))
            for i in range(3)]
    kv, plain, builder = model.new_kv_cache(blocks, "int4"), model.new_kv_cache(blocks), InputBuilder(256, 8, 13, DEV)
    pure_decode = model.pure_decode
    mine, moved = [], []
    for items in ([BatchItem(seqs[0], 0, seqs[0].token_ids[:50]), BatchItem(seqs[1], 0, seqs[1].token_ids[:33])],
                  [BatchItem(seqs[0], 50, seqs[0].token_ids[50:51]), BatchItem(seqs[1], 33, seqs[1].token_ids[33:34]),
                   BatchItem(seqs[2], 0, seqs[2].token_ids[:70])],
                  [BatchItem(s, n, s.token_ids[n:n + 1]) for s, n in zip(seqs, (51, 34, 70))]):
        inp = builder.build(items)
        T, slots = inp.input_ids.shape[0], inp.meta.slot_mapping
        logits = lambda cache, meta: model.compute_logits(model.forward(inp.input_ids, inp.positions, meta, cache),
                                                          inp.sample_indices)
        model.pure_decode = pure_decode
        got = logits(kv, inp.meta)
        mine.append(got), moved.append(logits(plain, inp.meta))
        held = H.kv_read_int4(kv.data, torch.arange(blocks, device=DEV))
        both = torch.cat([held, torch.zeros_like(held)[:, :, :-(-T // 16)]], dim=2)
        model.pure_decode = lambda *_: False             # (attention reads its rows from the cache)
        behind = torch.arange(T, device=DEV)
        want = logits(both, dataclasses.replace(inp.meta, slot_mapping=16 * blocks + behind))
        assert torch.equal(both[:, :, :blocks], held)
        assert float((got - want).norm() / want.norm()) < 1e-2
        wrote = both[:, :, blocks + behind // 16, :, behind % 16].double()                # [T, L, 2, KVH, D]
        there = held[:, :, slots // 16, :, slots % 16].double()
        rms = lambda x: x.square().mean((0, 3, 4)).sqrt()                                 # [L, 2]
        for j in range(2):
            steps = torch.from_numpy(O.unpack(kv.data[:, j].cpu().numpy(), cfg.head_dim, bool(j))[1].astype(np.float64))
            step = rms(steps.to(DEV)[:, None, slots // 16, :, slots % 16].expand(-1, -1, 2, -1, -1))[:, j]
            assert (rms(there - wrote)[:, j] <= 0.5 * step + 1e-2 * rms(wrote)[:, j]).all()
            assert (0.5 * step < 0.25 * rms(wrote)[:, j]).all()
    mine, moved = torch.cat(mine), torch.cat(moved)
    assert float((mine - moved).norm() / moved.norm()) > 5e-2


@pytest.mark.parametrize("heads", HEADS)
def test_results_of_the_largest_values_are_finite(heads):
    """V of 65504 in one half of the heads and -65504 in the other: a result is a mean of these, which no
    rounding of a weight may take past the largest number. Every 32nd token has a score of 0, the others one
    of log2(1/2 + 1.2 * 2^-12) in base 2: their weight is rounded up to 1/2 + 2^-11 for the product, not in the
    sum, and the mean comes out 2^-11 too large. One piece, merged splits, the prompt kernel, cut tiles."""
    c = Case(heads, [(n - 1, 1) for n in DECODE_LENS] + [(0, 90), (300, 40)], num_decode=len(DECODE_LENS), seed=76)
    _, q, _, _, cache, meta = c.on(DEV)
    n = 16 * c.NB
    place = np.zeros(n, np.int64)                        # a slot's position
    for b, length in enumerate(c.lens):
        at = np.arange(length)
        place[c.tables[b, at // 16].astype(np.int64) * 16 + at % 16] = at
    k, v = torch.zeros(2, n, c.KVH, c.D, device=DEV).half()
    k[torch.from_numpy(place % 32 > 0).to(DEV), :, 0] = -1
    v[:, :c.KVH // 2], v[:, c.KVH // 2:] = 65504, -65504
    H.kv_write_int4(k, v, cache[0, 0], cache[0, 1], torch.arange(n, device=DEV))
    held = cache[0].cpu().numpy()
    c.qkv[:] = 0
    c.split()[0][..., 0] = 1
    q = c.on(DEV)[1]
    c.scale = -math.log(0.5 + 1.2 * 2.0 ** -12)
    for bounds in (dict(), dict(max_seq_len=64), dict(max_prefill_seq_len=30000)):
        out = attend(q, cache, dataclasses.replace(meta, **bounds), c.scale)
        assert torch.isfinite(out).all(), bounds
        assert_rows(out, c, f"{bounds}", cache=held)
