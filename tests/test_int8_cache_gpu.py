"""The 8-bit paged cache on the GPU against the 64-bit oracle (oracle/int8_cache.py): its write must
give the oracle's codes and scales bit for bit, attention stay inside the oracle's error bound."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from oracle import int8_cache as O
from tests.int8_cases import HEADS, Case, near_the_rows, roll_back
from turingserve_amd import get_ops
from turingserve_amd import hip_ops as H
from turingserve_amd.qwen2 import rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def oracle_write(c, k=None, v=None):
    """(codes, scales) after the write of the case's (or the given) rows."""
    codes, scales = c.codes.copy(), c.scales.copy()
    _, kn, vn = c.split()
    for j, x in enumerate((kn if k is None else k, vn if v is None else v)):
        O.write(x, codes[j], scales[j], c.tables, c.lens, c.starts)
    return codes, scales


def assert_cache(cache, want, what=""):
    codes, scales = torch.stack(cache[:2]).cpu().numpy(), torch.stack(cache[2:]).cpu().numpy()
    assert np.array_equal(scales, want[1], equal_nan=True), f"{what}: scales"
    assert np.array_equal(codes, want[0]), f"{what}: {int((codes != want[0]).sum())} codes differ"


def assert_rows(out, c, what="", rows=slice(None), **kw):
    """out against the oracle's bound, over the rows that belong to sequences."""
    codes, scales = kw.get("cache", (c.codes, c.scales))
    q = kw.get("q", c.split()[0])
    ref, bound = O.paged_attention(q, codes, scales, c.tables, kw.get("lens", c.lens), c.starts, c.scale)
    got = out.double().cpu().numpy()
    got, ref, bound = got[rows], ref[rows], bound[rows]
    real = ~np.isnan(bound)
    err = np.abs(got - ref)
    worst = np.nanmax(np.where(real, err / bound, 0.0)) if real.any() else 0.0
    assert (err[real] <= bound[real]).all(), f"{what}: {worst:.3g} of the bound"
    return worst


# ------------------------------------------------------------------------------------- the write
ITEMS = [(5, 1), (15, 1), (16, 1), (0, 1), (0, 16), (3, 40), (31, 17), (0, 300), (1, 2), (30, 18)]


@pytest.mark.parametrize("heads", HEADS)
def test_write_matches_the_oracle(heads):
    c = Case(heads, ITEMS, num_decode=4, seed=1, tail_rows=3)
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    assert_cache(cache, oracle_write(c), f"write {heads}")
    # once more: rows already there keep their codes, the scales stay
    H.kv_write_int8(k, v, *cache, meta)
    assert_cache(cache, oracle_write(c), f"write again {heads}")


@pytest.mark.parametrize("heads", HEADS)
def test_rope_write_matches_the_oracle(heads):
    h, kvh, d = heads
    c = Case(heads, ITEMS, num_decode=4, seed=2, tail_rows=3)
    qkv, _, _, _, cache, meta = c.on(DEV)
    before = qkv.clone()
    cos, sin = rope_tables(d, 1e6, 512, DEV)
    q = H.rope_kv_write_int8(qkv, torch.from_numpy(c.pos).to(DEV), cos, sin, h, kvh, d, *cache, meta)
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


@pytest.mark.parametrize("size", [0.0, 6e-8, 1e-4, 60000.0])
def test_write_of_rows_of_any_size(size):
    """Zero rows (scale 0 unless rows stand there), subnormal ones, the largest."""
    c = Case((2, 2, 64), [(7, 1), (0, 1), (9, 30)], num_decode=2, seed=3)
    c.qkv[:] = (np.sign(c.qkv.astype(np.float32)) * size).astype(np.float16)
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    assert_cache(cache, oracle_write(c), f"rows of {size}")


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_rows_that_are_not_finite_poison_their_block_only(bad):
    c = Case((2, 2, 64), [(7, 1), (20, 1), (9, 40)], num_decode=2, seed=4)
    c.qkv[0, 2 * 64 + 5] = bad                       # K of head 0, the first sequence's row
    c.qkv[9, 5 * 64 + 7] = bad                       # V of head 1, inside the chunk
    _, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    want = oracle_write(c)
    assert np.isnan(want[1]).sum() == 2
    assert_cache(cache, want)
    # a block that starts anew forgets it
    again = Case((2, 2, 64), [(7, 1), (20, 1), (9, 40)], num_decode=2, seed=4)
    again.scales[:] = np.nan
    _, _, k, v, cache, _ = again.on(DEV)
    meta = again.meta(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    assert_cache(cache, oracle_write(again))


def test_write_skips_padding_foreign_and_missing_blocks():
    c = Case((4, 2, 32), [(7, 1), (0, 1), (3, 1), (9, 40), (0, 25)], num_decode=3, seed=5)
    c.lens[1] = 0                                    # a graph's padding row
    c.tables[3, 1] = c.NB + 7                        # out of the cache
    c.tables[4, 0] = -1
    c.tables = np.ascontiguousarray(c.tables[:, :3])  # the chunk's last block is not in the table
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    assert_cache(cache, oracle_write(c))


def test_write_with_fewer_positions_than_rows():
    """seq_len below the number of rows: rows at negative positions are skipped."""
    c = Case((4, 2, 32), [(0, 40), (0, 9)], seed=6)
    c.lens[:] = [25, 0]
    _, _, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    assert_cache(cache, oracle_write(c))


def test_write_host_bounds_and_layouts():
    """A bound below the real rows changes nothing; int64 metadata, a table slice with a wider
    stride and separate k / v tensors are taken."""
    c = Case((4, 2, 64), [(7, 1), (3, 1), (9, 100), (0, 25)], num_decode=2, seed=7)
    _, _, k, v, cache, meta = c.on(DEV)
    wide = torch.zeros(6, c.tables.shape[1] + 5, dtype=torch.int32, device=DEV)
    wide[:4, :c.tables.shape[1]] = meta.block_tables
    for change in (dict(max_query_len=1), dict(num_decode=0), dict(max_query_len=0),
                   dict(seq_lens=meta.seq_lens.long(), query_start_loc=meta.query_start_loc.long(),
                        block_tables=meta.block_tables.long()),
                   dict(block_tables=wide[:4, :c.tables.shape[1]])):
        _, _, _, _, cache, _ = c.on(DEV)
        H.kv_write_int8(k.contiguous(), v.contiguous(), *cache, dataclasses.replace(meta, **change))
        assert_cache(cache, oracle_write(c), str(list(change)))
    with pytest.raises(ValueError, match="unit stride"):
        H.kv_write_int8(k.transpose(0, 2).contiguous().transpose(0, 2), v, *cache, meta)
    odd = torch.empty(k.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(k.shape)
    with pytest.raises(ValueError, match="aligned"):
        H.kv_write_int8(odd, v, *cache, meta)


def test_strides_of_axes_of_one_element_do_not_matter():
    """One row, or one KV head, cut out of rows of an odd width."""
    c = Case((1, 1, 64), [(4, 1)], num_decode=1, seed=40)
    qkv, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    want = H.paged_attention_int8(q, *cache, meta, c.scale)
    cos, sin = rope_tables(64, 1e6, 8, DEV)
    pos = torch.from_numpy(c.pos).to(DEV)
    _, _, _, _, turned, _ = c.on(DEV)
    rotated = H.rope_kv_write_int8(qkv, pos, cos, sin, 1, 1, 64, *turned, meta)

    def odd(x):                                      # x [1, ...] at the start of a row of 4097 elements
        wide = torch.zeros(2, 4097, dtype=x.dtype, device=DEV)
        wide[0, :x.numel()] = x.flatten()
        return wide[:1, :x.numel()].as_strided(x.shape, (4097,) * (x.dim() - 1) + (1,))

    _, _, _, _, mine, _ = c.on(DEV)
    H.kv_write_int8(odd(k), odd(v), *mine, meta)
    assert_cache(mine, oracle_write(c))
    assert torch.equal(H.paged_attention_int8(odd(q), *mine, meta, c.scale), want)
    _, _, _, _, mine, _ = c.on(DEV)
    wide = torch.zeros(1, 193, dtype=torch.float16, device=DEV)
    wide[:, :192] = qkv
    assert torch.equal(H.rope_kv_write_int8(wide, pos, cos, sin, 1, 1, 64, *mine, meta), rotated)
    assert all(torch.equal(a, b) for a, b in zip(mine, turned))


def test_rope_write_clamps_positions_and_takes_one_row():
    c = Case((2, 1, 16), [(4, 1)], num_decode=1, seed=8)
    qkv, _, _, _, cache, meta = c.on(DEV)
    cos, sin = rope_tables(16, 1e6, 8, DEV)
    far = torch.tensor([10 ** 9], device=DEV)
    a = H.rope_kv_write_int8(qkv, far, cos, sin, 2, 1, 16, *cache, meta)
    _, _, _, _, last, _ = c.on(DEV)
    b = H.rope_kv_write_int8(qkv, torch.tensor([7], device=DEV), cos, sin, 2, 1, 16, *last, meta)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(cache, last))


@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_the_cache_is_near_that_over_the_rows(heads):
    near_the_rows(H, DEV, heads)


def test_rows_that_are_taken_back_keep_their_say():
    roll_back(H, DEV)


def test_appends_row_by_row_in_a_replayed_graph():
    """Forty single-row steps through one captured write, each checked."""
    c = Case((4, 2, 64), [(0, 40), (13, 40)], seed=9)
    _, kn, vn = c.split()
    _, _, k, v, cache, meta = c.on(DEV)
    kk, vv = k[:2].contiguous(), v[:2].contiguous()
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    step = c.meta(DEV, seq_lens=lens, num_decode=2, max_query_len=1,
                  query_start_loc=torch.arange(3, dtype=torch.int32, device=DEV))
    H.kv_write_int8(kk, vv, *cache, step)             # lengths 0: writes nothing
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        H.kv_write_int8(kk, vv, *cache, step)
    codes, scales = c.codes.copy(), c.scales.copy()
    for i in range(40):
        rows = [i, 40 + i]
        kk.copy_(k[rows])
        vv.copy_(v[rows])
        lens.copy_(torch.tensor([i + 1, 14 + i]))
        graph.replay()
        for j, x in enumerate((kn, vn)):
            O.write(x[rows], codes[j], scales[j], c.tables, [i + 1, 14 + i], [0, 1, 2])
        assert_cache(cache, (codes, scales), f"step {i}")


def test_write_past_two_to_the_31_bytes():
    """Blocks far into a large cache (offsets above 2^31), and its first ones left alone."""
    nb = (1 << 31) // (2 * 16 * 128) + 50
    c = Case((2, 2, 128), [(20, 1), (0, 33)], num_decode=1, seed=10)
    high = c.tables + nb - c.NB
    high[c.tables == 0] = 0
    kc, vc = (torch.zeros(nb, 2, 16, 128, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(nb, 2, device=DEV) for _ in range(2))
    lo = nb - c.NB
    for j, (x, s) in enumerate(((kc, ks), (vc, vs))):
        x[lo:] = torch.from_numpy(c.codes[j]).to(DEV)
        s[lo:] = torch.from_numpy(c.scales[j]).to(DEV)
    _, q, k, v, _, meta = c.on(DEV)
    meta = dataclasses.replace(meta, block_tables=torch.from_numpy(high).to(DEV))
    H.kv_write_int8(k, v, kc, vc, ks, vs, meta)
    want = oracle_write(c)
    assert_cache((kc[lo:], vc[lo:], ks[lo:], vs[lo:]), want)
    assert not kc[:lo].any() and not vc[:lo].any() and not ks[:lo].any()
    for bound in (33, 30000):                        # tiles of 16 rows, the prompt kernel
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(H.paged_attention_int8(q, kc, vc, ks, vs, m, c.scale), c, f"{bound}", cache=want)


# ------------------------------------------------------------------------------------- decode
DECODE_LENS = [1, 2, 15, 16, 17, 31, 33, 128, 255, 256, 257, 500, 513, 1000, 1025, 4096]


@pytest.mark.parametrize("heads", HEADS)
def test_decode_matches_the_oracle(heads):
    c = Case(heads, [(n - 1, 1) for n in DECODE_LENS], num_decode=len(DECODE_LENS), seed=11)
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    assert_rows(out, c, f"decode {heads}")
    # the host's bound on the lengths decides the splits only
    for bound in (0, 1, 300, 40000):
        m = dataclasses.replace(meta, max_seq_len=bound)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"decode {heads} bound {bound}")


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64), (1, 1, 16)])
def test_decode_of_a_long_sequence(heads):
    """More blocks than the splits of 16 hold, and more than a split looks up at once."""
    c = Case(heads, [(69999, 1), (16384, 1)], num_decode=2, seed=12)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(H.paged_attention_int8(q, *cache, meta, c.scale), c, f"long {heads}")
    short = dataclasses.replace(meta, max_seq_len=64)         # one split of 4375 blocks
    assert_rows(H.paged_attention_int8(q, *cache, short, c.scale), c, f"long, unsplit {heads}")


@pytest.mark.parametrize("rows,bound", [(1, 1), (2, 2), (2, 200)])   # a decode row, a short chunk, the prompt kernel
def test_the_longest_table(rows, bound):
    """2^26 blocks, the longest table that is taken (its entries repeat): K of zeros, V of 64 in all blocks
    but the last 64th, -64 there. Every sum of these is exact, and their mean is 62 (for the row before the
    last one, too, once it is rounded)."""
    nb = 1 << 26
    codes = torch.zeros(2, 3, 1, 16, 16, dtype=torch.int8, device=DEV)
    codes[1, 1], codes[1, 2] = 64, -64
    scales = torch.ones(2, 3, 1, device=DEV)
    table = torch.ones(1, nb, dtype=torch.int32, device=DEV)
    table[0, nb - nb // 64:] = 2
    c = Case((1, 1, 16), [(0, rows)])
    _, q, _, _, _, _ = c.on(DEV)
    meta = c.meta(DEV, seq_lens=torch.tensor([16 * nb], dtype=torch.int32, device=DEV), block_tables=table,
                  num_decode=int(rows == 1), max_query_len=bound, max_seq_len=16 * nb,
                  max_prefill_seq_len=16 * nb)
    out = H.paged_attention_int8(q, codes[0], codes[1], scales[0], scales[1], meta, c.scale)
    assert out.eq(62).all(), out


def test_decode_rows_do_not_depend_on_the_batch():
    c = Case((12, 2, 128), [(n - 1, 1) for n in DECODE_LENS * 5], num_decode=5 * len(DECODE_LENS), seed=13)
    _, q, _, _, cache, meta = c.on(DEV)
    whole = H.paged_attention_int8(q, *cache, meta, c.scale)
    for i in (3, 30, 79):
        one = dataclasses.replace(meta, seq_lens=meta.seq_lens[i:i + 1], num_decode=1,
                                  block_tables=meta.block_tables[i:i + 1],
                                  query_start_loc=meta.query_start_loc[:2])
        assert torch.equal(H.paged_attention_int8(q[i:i + 1], *cache, one, c.scale)[0], whole[i])


def test_decode_of_more_rows_than_a_lookup_holds():
    """300 sequences, some empty: rows without tokens are zeros."""
    lens = [(7 * i) % 40 for i in range(300)]
    c = Case((4, 2, 16), [(max(n - 1, 0), 1) for n in lens], num_decode=300, seed=14)
    c.lens[:] = lens
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    assert_rows(out, c)
    assert not out[torch.tensor(lens, device=DEV) == 0].any()


@pytest.mark.parametrize("k_size", [0.0, 1e-30, 300.0, 1e5])
def test_decode_of_flat_and_steep_scores(k_size):
    c = Case((12, 2, 128), [(n - 1, 1) for n in (1, 40, 700, 2000)], num_decode=4, seed=15, k_size=k_size)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(H.paged_attention_int8(q, *cache, meta, c.scale), c, f"k of {k_size}")


def test_scales_of_very_different_size():
    """V scales over sixty orders of two, zero among them: the small ones next to large ones count
    for nothing, alone they keep their precision."""
    c = Case((12, 2, 128), [(99, 1), (1999, 1), (15, 1), (0, 90)], num_decode=3, seed=16)
    rng = np.random.default_rng(0)
    c.scales[1] = np.exp2(rng.integers(-40, 10, c.scales[1].shape)).astype(np.float32)
    c.scales[1, c.tables[2, 0]] = 2.0 ** -20
    c.scales[1, c.tables[1, ::3]] = 0
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(H.paged_attention_int8(q, *cache, meta, c.scale), c)


@pytest.mark.parametrize("bound", [101, 30000])
def test_scales_too_small_for_fp16(bound):
    """V scales down to fp32's subnormal numbers: such blocks are zeros, beside others and alone."""
    c = Case((4, 2, 64), [(99, 1), (30, 1), (40, 60)], num_decode=2, seed=34)
    c.scales[1, c.tables[0, ::2]] = 1e-40
    c.scales[1, c.tables[1]] = 1e-42
    c.scales[1, c.tables[2, 1:3]] = 1e-36
    c.scales[0, c.tables[2, 3]] = 1e-41
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, dataclasses.replace(meta, max_prefill_seq_len=bound), c.scale)
    assert_rows(out, c, f"{bound}")
    assert not out[1].any()


@pytest.mark.parametrize("heads", [(4, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("bound", [101, 30000])
@pytest.mark.parametrize("big", [1e37, 3e38])
def test_scales_too_large_for_fp16(heads, bound, big):
    """V scales that are finite in fp32 only: codes of 0 stay 0, others are infinite, and blocks that a row
    does not see leave it as it is."""
    c = Case(heads, [(99, 1), (20, 1), (0, 60)], num_decode=2, seed=43)
    c.scales[1, c.tables[0]] = big                   # zeros only
    c.codes[1, c.tables[0]] = 0
    c.scales[1, c.tables[1, :2]] = big               # one sign a column
    c.codes[1, c.tables[1, :2]] = np.where(np.arange(c.D) % 2, 1, -1)
    c.scales[1, c.tables[2, 3]] = big                # tokens 48 .. 59
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, dataclasses.replace(meta, max_prefill_seq_len=bound), c.scale)
    assert not out[0].any()
    assert out[1].isinf().all() and (out[1].view(c.H, c.D) > 0).eq(torch.arange(c.D, device=DEV) % 2 == 1).all()
    assert_rows(out, c, rows=slice(2, 50))


def test_more_heads_than_a_chunk_may_have_rows():
    """160 query heads on one KV head: ten tiles a token."""
    c = Case((160, 1, 16), [(900, 1), (4, 1), (300, 3), (70, 1)], num_decode=2, seed=35)
    _, q, _, _, cache, meta = c.on(DEV)
    for bound in (303, 30000):
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"{bound}")


# ------------------------------------------------------------------------------------- prefill
@pytest.mark.parametrize("heads", [(4, 2, 16), (14, 2, 64)])
def test_one_long_prompt_among_many_short_ones(heads):
    """More sequences than a lookup holds at once, their blocks and tiles numbered across them: the
    write (also with the host's bound far below the long one), both kernels' attention."""
    items = [(9, 1), (700, 1)] + [(i % 37, 1 + i % 5) for i in range(75)] + [(40, 2500)] + \
        [(i % 50, 1 + i % 30) for i in range(90)]
    c = Case(heads, items, num_decode=2, seed=33)
    c.lens[10] = 0                                   # a chunk without positions
    _, q, k, v, cache, meta = c.on(DEV)
    want = oracle_write(c)
    for bound in (2500, 1, 90):
        mine = tuple(t.clone() for t in cache)
        H.kv_write_int8(k, v, *mine, dataclasses.replace(meta, max_query_len=bound))
        assert_cache(mine, want, f"{bound}")
    for bounds in (dict(), dict(max_query_len=8), dict(max_query_len=3, max_prefill_seq_len=60)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(H.paged_attention_int8(q, *mine, m, c.scale), c, f"{bounds}", cache=want)


PREFILL = [(0, 1), (0, 15), (15, 16), (37, 16), (1000, 17), (0, 300), (16, 530), (63, 65), (4000, 5)]


@pytest.mark.parametrize("heads", HEADS)
def test_prefill_matches_the_oracle(heads):
    c = Case(heads, PREFILL, seed=17)
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    assert_rows(out, c, f"prefill {heads}")
    # host bounds below the batch's own, and far above it
    for bounds in (dict(max_query_len=1), dict(max_query_len=40, max_prefill_seq_len=100, max_seq_len=100),
                   dict(max_query_len=2000, max_prefill_seq_len=30000, max_seq_len=30000),
                   dict(max_query_len=0, max_prefill_seq_len=0, max_seq_len=0)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"prefill {heads} {bounds}")


VERIFY = [(0, 5), (1, 5), (12, 3), (300, 5), (2047, 4), (9, 1), (255, 2), (5000, 5), (4094, 5)]


@pytest.mark.parametrize("heads", HEADS)
def test_a_few_rows_per_sequence(heads):
    """The rows of a speculative step: up to five a sequence, beside decode rows."""
    c = Case(heads, [(100, 1), (0, 1)] + VERIFY, num_decode=2, seed=30)
    c.lens[3] = 3                                    # five rows, three positions
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    assert_rows(out, c, f"verify {heads}")
    assert not out[int(c.starts[3]):int(c.starts[3]) + 2].any()
    for bounds in (dict(max_query_len=2), dict(max_seq_len=100, max_prefill_seq_len=0),
                   dict(max_query_len=200), dict(num_decode=0)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"verify {heads} {bounds}")


@pytest.mark.parametrize("heads", HEADS)
def test_short_chunks_beside_long_prefixes(heads):
    """Up to 21 rows a sequence: several tiles of 16 rows whose splits are merged, with as many
    partials in the workspace as one tile has."""
    items = [(4200, 16), (300, 21), (2047, 9), (20000, 12), (0, 21), (100, 1), (33, 20)]
    c = Case(heads, [(1500, 1)] + items, num_decode=1, seed=32)
    _, q, _, _, cache, meta = c.on(DEV)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    assert_rows(out, c, f"short chunks {heads}")
    # host bounds below the batch's own leave fewer partials: fewer splits
    for bounds in (dict(max_query_len=3), dict(max_query_len=8, max_seq_len=900, max_prefill_seq_len=900),
                   dict(max_query_len=1, max_seq_len=20100, max_prefill_seq_len=20100)):
        m = dataclasses.replace(meta, **bounds)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"short chunks {heads} {bounds}")


@pytest.mark.parametrize("side", [0, 1])
def test_a_few_rows_around_a_block_without_a_finite_scale(side):
    """Rows before the block are right, rows that see it NaN, also where later blocks are hidden."""
    c = Case((14, 2, 64), [(317, 40), (30, 36)], seed=31)
    c.scales[side, c.tables[0, 20], 1] = np.nan      # tokens 320 .. 335
    c.scales[side, c.tables[1, 3], 1] = np.nan       # tokens 48 .. 63
    _, q, _, _, cache, meta = c.on(DEV)
    clean = np.nan_to_num(c.scales, nan=0.0)
    hit = np.zeros((c.T, c.H), bool)
    hit[3:40, 7:] = True                             # positions 320 and later of the first
    hit[40 + 18:, 7:] = True                         # 48 and later of the second
    for bound in (40, 4):                            # the chunk kernel; tiles of 16 rows, unsplit
        out = H.paged_attention_int8(q, *cache, dataclasses.replace(meta, max_query_len=bound), c.scale)
        got = out.cpu().numpy().reshape(c.T, c.H, c.D)
        assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all(), bound
        ref, lim = O.paged_attention(c.split()[0], c.codes, clean, c.tables, c.lens, c.starts, c.scale)
        ok = ~np.repeat(hit, c.D, axis=1).reshape(c.T, -1)
        assert (np.abs(out.double().cpu().numpy() - ref) <= lim)[ok].all(), bound


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64)])
def test_prefill_over_a_long_prefix(heads):
    """More blocks than are looked up at once, and split along the keys."""
    c = Case(heads, [(9000, 70), (3, 200), (30000, 3)], seed=18)
    _, q, _, _, cache, meta = c.on(DEV)
    assert_rows(H.paged_attention_int8(q, *cache, meta, c.scale), c, f"long prefix {heads}")


@pytest.mark.parametrize("heads", HEADS)
def test_mixed_batch(heads):
    """Decode rows beside chunks, a padding row, a sequence without positions, rows behind the last
    sequence; the step's write before the attention."""
    items = [(40, 1), (0, 1), (777, 1), (0, 20), (100, 130), (5, 3)]
    c = Case(heads, items, num_decode=3, seed=19, tail_rows=2)
    c.lens[1] = 0
    c.lens[5] = 2                                    # three rows, two positions
    _, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    want = oracle_write(c)
    assert_cache(cache, want)
    for bound in (777, 30000):                       # tiles of 16 rows, the prompt kernel
        out = H.paged_attention_int8(q, *cache, dataclasses.replace(meta, max_prefill_seq_len=bound), c.scale)
        assert_rows(out, c, f"mixed {heads} {bound}", cache=want)
        assert not out[1].any() and not out[int(c.starts[5])].any()


def test_sequences_without_rows():
    """Sequences of no new rows between the others, and a step of rows that belong to none."""
    c = Case((14, 2, 64), [(100, 1), (40, 0), (0, 0), (5, 20), (300, 0), (70, 60)], num_decode=1, seed=37)
    qkv, q, k, v, cache, meta = c.on(DEV)
    H.kv_write_int8(k, v, *cache, meta)
    want = oracle_write(c)
    assert_cache(cache, want)
    for bound in (300, 30000):
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"{bound}", cache=want)
    none = dataclasses.replace(meta, seq_lens=meta.seq_lens[:0], block_tables=meta.block_tables[:0],
                               query_start_loc=meta.query_start_loc[:1], num_decode=0)
    cos, sin = rope_tables(c.D, 1e6, 512, DEV)
    pos = torch.from_numpy(c.pos).to(DEV)
    H.kv_write_int8(k, v, *cache, none)
    rotated = H.rope_kv_write_int8(qkv, pos, cos, sin, c.H, c.KVH, c.D, *cache, none)
    assert_cache(cache, want)
    assert torch.equal(rotated, H.rope_kv_write_int8(qkv, pos, cos, sin, c.H, c.KVH, c.D,
                                                     *(t.clone() for t in cache), meta))
    assert H.paged_attention_int8(q, *cache, none, c.scale).shape == (c.T, c.H * c.D)


def test_table_shorter_than_the_sequence():
    c = Case((14, 2, 64), [(299, 1), (50, 200)], num_decode=1, seed=20)
    c.tables = np.ascontiguousarray(c.tables[:, :8])          # 128 tokens of 300 and 250
    _, q, _, _, cache, meta = c.on(DEV)
    for bound in (300, 30000):
        m = dataclasses.replace(meta, max_prefill_seq_len=bound)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"{bound}")


def test_foreign_block_ids_read_block_zero():
    c = Case((14, 2, 64), [(99, 1), (50, 60)], num_decode=1, seed=21)
    _, q, _, _, cache, meta = c.on(DEV)
    bad = meta.block_tables.clone()
    bad[0, 2], bad[1, 3] = c.NB + 100, -5
    c.tables[0, 2] = c.tables[1, 3] = 0
    for bound in (100, 30000):
        m = dataclasses.replace(meta, block_tables=bad, max_prefill_seq_len=bound)
        assert_rows(H.paged_attention_int8(q, *cache, m, c.scale), c, f"{bound}")


@pytest.mark.parametrize("heads", [(12, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("bound", [501, 30000])      # tiles of 16 rows, the prompt kernel
def test_blocks_without_a_finite_scale(heads, side, bad, bound):
    """Rows that see a token of such a block are NaN, rows before it (and other sequences) are not;
    blocks past a sequence's end have no say."""
    c = Case(heads, [(100, 1), (500, 1), (5, 150), (0, 40)], num_decode=2, seed=22)
    c.scales[side, c.tables[1, 20], 0] = bad         # tokens 320 .. 335 of the second sequence
    c.scales[side, c.tables[2, 5], 0] = bad          # tokens 80 .. 95 of the third
    unused = sorted(set(range(c.NB)) - set(c.tables.ravel().tolist()))
    c.scales[:, unused] = np.nan
    _, q, _, _, cache, meta = c.on(DEV)
    meta = dataclasses.replace(meta, max_prefill_seq_len=bound)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    clean = np.nan_to_num(c.scales, nan=0.0, posinf=0.0)
    got = out.cpu().numpy().reshape(c.T, c.H, c.D)
    g = c.H // c.KVH
    hit = np.zeros((c.T, c.H), bool)
    hit[1, :g] = True
    lo = int(c.starts[2])
    hit[lo + 75:lo + 150, :g] = True                 # rows at positions 80 and later
    assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()
    ref, bound = O.paged_attention(c.split()[0], c.codes, clean, c.tables, c.lens, c.starts, c.scale)
    ok = ~np.repeat(hit, c.D, axis=1).reshape(c.T, -1)
    assert (np.abs(out.double().cpu().numpy() - ref) <= bound)[ok].all()


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("bound", [90, 30000])      # tiles of 16 rows, the prompt kernel
def test_hidden_blocks_have_no_say(heads, bound):
    """Rows that see only blocks with small V scales, ahead of blocks whose V scales are 2^20 and 2^25
    times theirs: as exact as if those blocks were not there, and the same bits whatever stands in
    them."""
    c = Case(heads, [(0, 90), (0, 90)], seed=38)
    c.scales[1, c.tables] = 2.0 ** 8
    c.scales[1, c.tables[0, 0]] = 2.0 ** -12
    c.scales[1, c.tables[1, 0]] = 2.0 ** -17
    _, q, _, _, cache, meta = c.on(DEV)
    meta = dataclasses.replace(meta, max_prefill_seq_len=bound)
    out = H.paged_attention_int8(q, *cache, meta, c.scale)
    for b, lo in enumerate(c.starts[:2].tolist()):
        alone = np.arange(lo, lo + 16)
        ref, lim = O.paged_attention(c.split()[0][alone], c.codes, c.scales, c.tables[b:b + 1], [16], [0, 16],
                                     c.scale)
        err = np.abs(out[lo:lo + 16].double().cpu().numpy() - ref)
        assert (err <= lim).all(), f"sequence {b}: {(err / lim).max():.3g} of the bound"
    assert_rows(out, c)
    # tokens 23 and later of both
    other = [t.clone() for t in cache]
    for b in range(2):
        for t in other[:2]:
            t[c.tables[b, 1], :, 7:] = t[c.tables[b, 1], :, 7:].flip(0, 1, 2)
            t[c.tables[b, 2:]] = t[c.tables[b, 2:]].flip(0, 1, 2, 3)
        for t in other[2:]:
            t[c.tables[b, 2:]] = torch.exp2(torch.randint(-30, 9, t[c.tables[b, 2:]].shape, device=DEV).float())
    again = H.paged_attention_int8(q, *other, meta, c.scale)
    for lo in c.starts[:2].tolist():
        assert torch.equal(out[lo:lo + 23], again[lo:lo + 23])
        assert not torch.equal(out[lo + 23:lo + 90], again[lo + 23:lo + 90])


def test_attention_refuses():
    c = Case((4, 2, 64), [(7, 1), (9, 20)], num_decode=1, seed=23)
    _, q, _, _, cache, meta = c.on(DEV)
    with pytest.raises(ValueError, match="fp16"):
        H.paged_attention_int8(q.float(), *cache, meta, c.scale)
    with pytest.raises(ValueError, match="unit stride"):
        H.paged_attention_int8(q.transpose(0, 2).contiguous().transpose(0, 2), *cache, meta, c.scale)
    with pytest.raises(ValueError, match="scale"):
        H.paged_attention_int8(q, *cache, meta, -1.0)
    with pytest.raises(ValueError, match="same GPU"):
        H.paged_attention_int8(q, *cache, dataclasses.replace(meta, seq_lens=meta.seq_lens.cpu()), 1.0)
    odd = torch.empty(q.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(q.shape)
    with pytest.raises(ValueError, match="misaligned"):
        H.paged_attention_int8(odd, *cache, meta, c.scale)
    assert H.paged_attention_int8(q[:0], *cache, meta, c.scale).shape == (0, 256)


def test_decode_graph_replayed_over_growing_sequences():
    """A captured step (write, then attention) with max_seq_len of the longest that it may meet,
    replayed while the lengths grow, with eager calls between the replays."""
    c = Case((12, 2, 128), [(0, 600), (0, 600), (0, 600)], seed=24)
    _, kn, vn = c.split()
    _, q, k, v, cache, meta = c.on(DEV)
    qq, kk, vv = (x[:3].contiguous() for x in (q, k, v))
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    step = c.meta(DEV, seq_lens=lens, num_decode=3, max_query_len=1, max_seq_len=600,
                  query_start_loc=torch.arange(4, dtype=torch.int32, device=DEV))

    def once():
        H.kv_write_int8(kk, vv, *cache, step)
        return H.paged_attention_int8(qq, *cache, step, c.scale)

    assert not once().any()                           # lengths 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    codes, scales = c.codes.copy(), c.scales.copy()
    for now in ([1, 17, 255], [2, 18, 256], [3, 0, 257], [4, 19, 258], [511, 20, 0], [512, 21, 600]):
        rows = [max(n - 1, 0) + 600 * b for b, n in enumerate(now)]
        qq.copy_(q[rows]), kk.copy_(k[rows]), vv.copy_(v[rows])
        lens.copy_(torch.tensor(now))
        graph.replay()
        eager = once()
        assert torch.equal(out, eager)
        for j, x in enumerate((kn, vn)):
            O.write(x[rows], codes[j], scales[j], c.tables, now, [0, 1, 2, 3])
        assert_cache(cache, (codes, scales), str(now))
        ref, bound = O.paged_attention(c.split()[0][rows], codes, scales, c.tables, now, [0, 1, 2, 3],
                                       c.scale)
        assert (np.abs(out.double().cpu().numpy() - ref) <= bound).all(), str(now)


def test_chunk_graphs_of_one_pool():
    """Two captured mixed steps (one for each of the attention's kernels) whose workspaces share a
    memory pool, replayed in turn with other inputs each time and eager calls in between."""
    c = Case((14, 2, 64), [(900, 1), (300, 40), (0, 500), (17, 1)], num_decode=1, seed=36)
    _, q, k, v, cache, meta = c.on(DEV)
    start = tuple(t.clone() for t in cache)
    qq, kk, vv = q.clone(), k.clone(), v.clone()
    metas = [dataclasses.replace(meta, max_prefill_seq_len=b) for b in (500, 30000)]

    def step(m):
        H.kv_write_int8(kk, vv, *cache, m)
        return H.paged_attention_int8(qq, *cache, m, c.scale)

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
            for t, s in zip(cache, start):
                t.copy_(s)
            g.replay()
            got, codes = out.clone(), tuple(t.clone() for t in cache)
            for t, s in zip(cache, start):
                t.copy_(s)
            assert torch.equal(step(m), got), turn
            assert all(torch.equal(a, b) for a, b in zip(codes, cache)), turn
        _, kn, vn = c.split()
        want = oracle_write(c, np.roll(kn, turn, 0), np.roll(vn, -turn, 0))
        assert_cache(cache, want)
        assert_rows(got, c, f"{turn}", cache=want, q=np.roll(c.split()[0], turn, 0))


def test_two_streams_at_once():
    """The same calls on two streams, workspaces of their own each."""
    c = Case((12, 2, 128), [(3000, 1), (1000, 1), (500, 90)], num_decode=2, seed=25)
    _, q, _, _, cache, meta = c.on(DEV)
    want = H.paged_attention_int8(q, *cache, meta, c.scale)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(H.paged_attention_int8(q, *cache, meta, c.scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------------------------- together
def test_model_step_matches_the_reference_twins():
    """A chunked prompt beside decode rows through the whole model, 8-bit cache: hip against the
    reference namespace. Both round activations to fp16 at other places, and a rounded k can land on
    the neighbouring code, so the bar is the fp16 model test's kind: logits close relative to their
    spread."""
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
        kv = model.new_kv_cache(40, "int8")
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
    assert float((a - b).norm() / b.norm()) < 2e-2


def test_engine_tokens_with_graphs_equal_eager():
    from turingserve_amd.engine import GreedyEngine
    from turingserve_amd.qwen2 import TINY_G2, Qwen2Model, random_weights

    model = Qwen2Model(TINY_G2, random_weights(TINY_G2, DEV, seed=28), get_ops("hip"), 1024)
    g = torch.Generator().manual_seed(29)
    prompts = [torch.randint(0, TINY_G2.vocab_size, (n,), generator=g).tolist() for n in (100, 3, 47, 300)]
    outs = []
    for sizes, dev_meta in (((), False), ((1, 2, 4), False), ((4,), True)):
        eng = GreedyEngine(model, 128, max_num_batched_tokens=128, graph_sizes=sizes,
                           device_metadata=dev_meta, kv_cache_dtype="int8")
        outs.append(eng.generate(prompts, 24))
        assert bool(sizes) == (eng.graph_steps > 0) and eng.mixed_steps > 0
    assert outs[0] == outs[1] == outs[2]
