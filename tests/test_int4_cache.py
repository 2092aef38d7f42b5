"""The 4-bit paged cache on the CPU: the oracle against brute force, the torch twins against the
oracle, and every refusal of the entry points."""

from __future__ import annotations

import ctypes
import dataclasses

import numpy as np
import pytest
import torch

from oracle import int4_cache as O
from tests.int4_cases import (HEADS, TINY, Case, coherent_rows, near_the_rows, outside, over_the_cache,
                              over_the_rows, tiny_rows)
from turingserve_amd import _native as N
from turingserve_amd import get_ops
from turingserve_amd import hip_ops as H
from turingserve_amd import reference_ops as R
from turingserve_amd.quant import Int4KVCache, int4_head_dim, int4_quantise, int4_unit_bytes, int4_views
from turingserve_amd.qwen2 import rope_tables

P = ctypes.c_void_p(256)                 # never dereferenced: the call fails validation first
odd = ctypes.c_void_p(264)


def test_group_by_hand():
    x = np.linspace(-1.0, 2.0, 16)[None]                 # steps of 0.2: low -1, fifteen of them up to 2
    codes, steps, lows = O.quantise(x)
    assert lows[0, 0] == -1 and float(steps[0, 0]) == float(np.float16(0.2)) < 0.2
    assert codes[0].tolist() == list(range(16))
    x = np.full((1, 16), 7.0)
    codes, steps, lows = O.quantise(x)
    assert lows[0, 0] == 7 and steps[0, 0] == 0 and not codes.any() and (O.held(x) == 7).all()
    # ties to even, and the upper end: 15 codes of 1
    x = np.array([[0.0, 0.5, 1.5, 2.5, 14.5, 15.0] + [0.0] * 10])
    assert O.quantise(x)[0][0, :6].tolist() == [0, 0, 2, 2, 14, 15]
    # the largest numbers: nothing leaves the range
    x = np.where(np.arange(16) % 2, 65504.0, -65504.0)[None]
    assert np.isfinite(O.held(x)).all() and np.abs(O.held(x) - x).max() < 2.0 ** -10 * 131008 + 32


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("size", [1e-7, 1e-3, 1.0, 300.0, 60000.0])
def test_values_are_within_half_a_step(D, size):
    """Off by half a step, by what the step was rounded down by (2^-10 of it, 2^-24 where it is subnormal;
    15 of them at the group's end), by low's rounding and by the value's own."""
    x = (np.random.default_rng(D).uniform(-1, 1, (50, D)) * size).astype(np.float16)
    _, steps, lows = O.quantise(x)
    wide = lambda n: np.repeat(n.astype(np.float64), D // O.groups(D), -1)
    lim = wide(steps) * (0.5 + 15 / 1024 + 2.0 ** -16) + 15 * 2.0 ** -24 + 2.0 ** -11 * np.abs(wide(lows)) \
        + 2.0 ** -11 * np.abs(x.astype(np.float64)) + 2.0 ** -24
    got = O.held(x).astype(np.float64)
    assert (np.abs(got - x) <= lim).all()
    assert (got <= np.repeat(x.reshape(50, O.groups(D), -1).max(-1), D // O.groups(D), -1)).all()


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("values", [False, True])
def test_layout(D, values):
    """Every nibble and every byte of the numbers has one place; the torch views see the same ones."""
    rng = np.random.default_rng(D)
    codes = rng.integers(0, 16, (3, 2, 16, D)).astype(np.uint8)
    steps, lows = (rng.standard_normal((3, 2, 16, O.groups(D))).astype(np.float16) for _ in range(2))
    cache = O.pack(codes, steps, lows, values)
    assert cache.shape[-1] == O.unit_bytes(D) == int4_unit_bytes(D) and int4_head_dim(cache.shape[-1]) == D
    places = {O.code_place(r, d, D, values) for r in range(16) for d in range(D)}
    places |= {(p + i, s) for r in range(16) for g in range(O.groups(D)) for p in O.number_places(r, g, D, values)
               for i in range(2) for s in (0, 4)}
    assert places == {(b, s) for b in range(O.unit_bytes(D)) for s in (0, 4)}
    back = O.unpack(cache, D, values)
    assert all(np.array_equal(a, b) for a, b in zip(back, (codes, steps, lows)))
    _, s, low = int4_views(torch.from_numpy(cache), values)
    shape = (lambda t: t.flatten(-3, -2)) if values else (lambda t: t)
    assert np.array_equal(shape(s).numpy(), steps) and np.array_equal(shape(low).numpy(), lows)
    both = np.stack([cache, cache])[None]
    got = R.kv_read_int4(torch.from_numpy(both), torch.arange(3))[0, int(values)].numpy()
    assert np.array_equal(got, O.values_of(codes, steps, lows))


@pytest.mark.parametrize("make", [
    lambda: Case((4, 2, 16), [(0, 1), (0, 40), (16, 530)], num_decode=1, seed=17),
    lambda: Case((12, 2, 128), [(0, 1), (32, 1), (4095, 1)], num_decode=3, seed=11),
    lambda: Case((14, 2, 64), [(69999, 1)], num_decode=1, seed=12),
    lambda: Case((12, 2, 128), [(0, 1), (39, 1), (1999, 1)], num_decode=3, seed=15, k_size=300.0),
    lambda: Case((12, 2, 128), [(0, 1), (39, 1), (1999, 1)], num_decode=3, seed=15, k_size=0.0)])
def test_attention_bound_catches_a_lost_result(make):
    """The oracle's bound is a small part of every (row, head)'s values: less than 1/32 of their rms, so
    that a result of zeros, or of other tokens, does not pass."""
    c = make()
    cache = c.cache
    ref, bound = O.paged_attention(c.split()[0], *cache, c.tables, c.lens, c.starts, c.scale)
    rms = lambda x: np.sqrt((x.reshape(c.T, c.H, c.D) ** 2).mean(-1))
    assert (rms(bound) < np.maximum(rms(ref), 2.0 ** -14) / 32).all()


@pytest.mark.parametrize("heads", HEADS)
def test_twins_match_the_oracle(heads):
    c = Case(heads, [(4, 1), (15, 1), (0, 1), (0, 21), (7, 30)], num_decode=3, seed=2, tail_rows=2)
    _, q, k, v, cache, meta = c.on("cpu")
    want = c.cache
    O.write(*c.split()[1:], *want, c.slots)
    R.kv_write_int4(k, v, cache[0, 0], cache[0, 1], meta.slot_mapping)
    assert np.array_equal(cache[0].numpy(), want)
    read = R.kv_read_int4(cache, torch.tensor([1, -1, c.NB, 2])).numpy()
    for j in range(2):
        assert np.array_equal(read[0, j], O.values_of(*O.unpack(want[j], c.D, bool(j)))[[1, 0, 0, 2]])
    n = int(c.starts[-1])
    out = R.paged_attention_int4(q, cache[0, 0], cache[0, 1], meta, c.scale)
    ref, bound = O.paged_attention(c.split()[0], *want, c.tables, c.lens, c.starts, c.scale)
    assert (np.abs(out.double().numpy() - ref) <= bound)[:n].all()


@pytest.mark.parametrize("what", ["short table", "fewer positions", "foreign blocks", "nan k", "nan v"])
def test_attention_twin_keeps_the_contract(what):
    """Tables that do not hold the sequence, rows before its first token, ids outside the cache, tokens
    that are not finite: as the kernels, by the oracle."""
    c = Case((4, 2, 16), [(20, 1), (5, 60), (0, 0), (0, 3)], num_decode=1, seed=41)
    hit = np.zeros((c.T, c.H), bool)
    if what == "short table":
        c.tables = np.ascontiguousarray(c.tables[:, :2])
    elif what == "fewer positions":
        c.lens[1] = 20
    elif what == "foreign blocks":
        c.tables[0, 1], c.tables[1, 1] = c.NB, -1
    cache = c.cache
    if what.startswith("nan"):                           # the second sequence's row at position 33
        k, v = (x[29:30].astype(np.float32).copy() for x in c.split()[1:])
        (k if what == "nan k" else v)[0, 1, 3] = np.inf
        O.write(k, v, *cache, [c.tables[1, 2] * 16 + 1])
        hit[29:61, 2:] = True
    _, q, _, _, _, meta = c.on("cpu")
    t = torch.from_numpy(cache)
    out = R.paged_attention_int4(q, t[0], t[1], meta, c.scale).double().numpy()
    c.tables[(c.tables < 0) | (c.tables >= c.NB)] = 0
    ref, bound = O.paged_attention(c.split()[0], *cache, c.tables, c.lens, c.starts, c.scale)
    rows = np.repeat(hit, c.D, axis=1)
    assert np.isnan(out[rows]).all() and np.isnan(ref[rows]).all() and (np.abs(out - ref) <= bound)[~rows].all()
    if what == "fewer positions":
        assert not out[1:41].any() and out[41:61].any()


def test_rope_twin_matches_the_oracle():
    c = Case((6, 2, 32), [(4, 1), (0, 40)], num_decode=1, seed=3)
    qkv, _, _, _, cache, meta = c.on("cpu")
    cos, sin = rope_tables(32, 1e6, 64, "cpu")
    q = R.rope_kv_write_int4(qkv, torch.from_numpy(c.pos), cos, sin, 6, 2, 32, cache[0, 0], cache[0, 1],
                             meta.slot_mapping)
    qn, kn, vn = c.split()
    cn, sn = cos.numpy()[c.pos], sin.numpy()[c.pos]
    want = c.cache
    O.write(O.rotate(kn, cn, sn), vn, *want, c.slots)
    assert np.array_equal(cache[0].numpy(), want)
    ref = O.rotate(qn, cn, sn)
    assert (np.abs(q.double().numpy() - ref) <= 2.0 ** -11 * np.abs(ref) + 2.0 ** -23 + 2.0 ** -25).all()


@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_the_cache_is_near_that_over_the_rows(heads):
    near_the_rows(R, "cpu", heads)


def _write(**kw):
    a = dict(k=P, v=P, kst=64, ksh=64, vst=64, vsh=64, kc=P, vc=P, nb=4, slots=P, T=1, kvh=1, D=64)
    a.update(kw)
    return N.lib().ts_kv_write_int4(*a.values(), None)


def _rope(**kw):
    a = dict(qkv=P, st=256, pos=P, cos=P, sin=P, mp=16, q=P, kc=P, vc=P, nb=4, slots=P, T=1, h=2, kvh=1, D=64)
    a.update(kw)
    return N.lib().ts_rope_kv_write_int4(*a.values(), None)


def _read(**kw):
    a = dict(cache=P, layers=1, nb=4, kvh=1, D=64, blocks=P, n=1, out=P)
    a.update(kw)
    return N.lib().ts_kv_read_int4(*a.values(), None)


def _attend(**kw):
    a = dict(q=P, qst=128, qsh=64, out=P, ost=128, T=1, kc=P, vc=P, nb=4, bt=P, bts=4, mb=4, sl=P, qsl=P,
             seqs=1, dec=0, mq=1, ms=64, mp=64, h=2, kvh=1, D=64, scale=0.125, ws=None, wsb=0)
    a.update(kw)
    return N.lib().ts_paged_attention_int4(*a.values(), None)


@pytest.mark.parametrize("call,kw,status,text", [
    (_write, dict(T=-1), N.TS_ERR_INVALID_ARG, "num_tokens"),
    (_write, dict(k=None), N.TS_ERR_INVALID_ARG, "null"),
    (_write, dict(slots=None), N.TS_ERR_INVALID_ARG, "null"),
    (_write, dict(kvh=0), N.TS_ERR_INVALID_ARG, "num_kv_heads"),
    (_write, dict(nb=0), N.TS_ERR_INVALID_ARG, "num_blocks"),
    (_write, dict(D=96), N.TS_ERR_UNSUPPORTED, "head_dim 96"),
    (_write, dict(kst=68), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(vsh=-8), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(k=odd), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(vc=odd), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(T=1 << 30), N.TS_ERR_UNSUPPORTED, "tokens"),
    (_rope, dict(cos=None), N.TS_ERR_INVALID_ARG, "null"),
    (_rope, dict(mp=0), N.TS_ERR_INVALID_ARG, "empty table"),
    (_rope, dict(st=252), N.TS_ERR_INVALID_ARG, "aligned"),
    (_rope, dict(st=248), N.TS_ERR_INVALID_ARG, "qkv rows"),
    (_rope, dict(h=0), N.TS_ERR_INVALID_ARG, "num_heads"),
    (_rope, dict(D=48), N.TS_ERR_UNSUPPORTED, "head_dim 48"),
    (_rope, dict(T=1 << 29), N.TS_ERR_UNSUPPORTED, "tokens"),
    (_read, dict(n=-1), N.TS_ERR_INVALID_ARG, "n=-1"),
    (_read, dict(blocks=None), N.TS_ERR_INVALID_ARG, "null"),
    (_read, dict(nb=0), N.TS_ERR_INVALID_ARG, "num_blocks"),
    (_read, dict(D=80), N.TS_ERR_UNSUPPORTED, "head_dim 80"),
    (_read, dict(out=odd), N.TS_ERR_INVALID_ARG, "aligned"),
    (_read, dict(layers=1 << 20, n=1 << 20), N.TS_ERR_UNSUPPORTED, "blocks"),
    (_attend, dict(seqs=-1), N.TS_ERR_INVALID_ARG, "num_seqs"),
    (_attend, dict(dec=1, T=0), N.TS_ERR_INVALID_ARG, "num_decode"),
    (_attend, dict(vc=None), N.TS_ERR_INVALID_ARG, "null"),
    (_attend, dict(D=80), N.TS_ERR_UNSUPPORTED, "head_dim 80"),
    (_attend, dict(h=3, kvh=2), N.TS_ERR_INVALID_ARG, "heads"),
    (_attend, dict(nb=0), N.TS_ERR_INVALID_ARG, "num_blocks"),
    (_attend, dict(seqs=(1 << 20) + 1, ws=P, wsb=1 << 62), N.TS_ERR_UNSUPPORTED, "sequences"),
    (_attend, dict(T=1 << 30, seqs=4, ws=P, wsb=1 << 62), N.TS_ERR_UNSUPPORTED, "tokens"),
    (_attend, dict(mb=(1 << 26) + 1, bts=1 << 27), N.TS_ERR_INVALID_ARG, "max_blocks"),
    (_attend, dict(qst=130), N.TS_ERR_INVALID_ARG, "misaligned"),
    (_attend, dict(ost=64), N.TS_ERR_INVALID_ARG, "misaligned"),
    (_attend, dict(q=odd), N.TS_ERR_INVALID_ARG, "misaligned"),
    (_attend, dict(scale=0.0), N.TS_ERR_INVALID_ARG, "scale"),
    (_attend, dict(scale=float("nan")), N.TS_ERR_INVALID_ARG, "scale"),
])
def test_refusals(call, kw, status, text):
    assert call(**kw) == status and text in N.last_error() and "int4" in N.last_error()


def test_empty_calls_and_workspace_sizes():
    assert _write(T=0) == N.TS_OK and _rope(T=0) == N.TS_OK
    assert _read(n=0) == N.TS_OK and _read(layers=0) == N.TS_OK
    assert _attend(T=0) == N.TS_OK and _attend(seqs=0, T=0) == N.TS_OK
    size = N.lib().ts_paged_attention_int4_workspace_bytes
    assert size(1, 2, 1, 64, 0, 2, 1, 64, 256) == 0 and size(1, 1, 1, 64, 0, 3, 2, 64, 256) == 0
    assert size(64, 64, 1, 256, 0, 12, 2, 128, 256) == 0                 # one split a row
    long = size(4, 4, 1, 32768, 0, 12, 2, 128, 256)
    assert long >= 4 * 12 * 64 * (128 + 2) * 4
    # the host's bounds may be anything
    huge = 2 ** 31 - 1
    assert size(64, 0, huge, huge, huge, 64, 8, 128, 256) == size(64, 0, 4096, 65536, 65536, 64, 8, 128, 256)


def test_python_wrappers_refuse():
    c = Case((2, 1, 64), [(3, 1), (0, 5)], num_decode=1)
    qkv, q, k, v, cache, meta = c.on("cpu")
    layer = cache[0, 0], cache[0, 1]
    cos, sin = rope_tables(64, 1e6, 64, "cpu")
    for call in (lambda: H.kv_write_int4(k, v, *layer, meta.slot_mapping),
                 lambda: H.rope_kv_write_int4(qkv, torch.from_numpy(c.pos), cos, sin, 2, 1, 64, *layer,
                                              meta.slot_mapping),
                 lambda: H.kv_read_int4(cache, torch.arange(2)),
                 lambda: H.paged_attention_int4(q, *layer, meta, 0.1)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    # the cache's and the metadata's checks come before anything is launched
    assert H._int4_cache("x", *layer) == (c.NB, 1, 64)
    for bad in ((layer[0].char(), layer[1]), (layer[0][..., :-8], layer[1][..., :-8]), (layer[0], layer[1][:-1]),
                (cache, cache), (layer[0][::2], layer[1][::2])):
        with pytest.raises(ValueError, match="caches must be"):
            H._int4_cache("x", *bad)
    with pytest.raises(ValueError, match="shorter"):
        H._slots("x", meta.slot_mapping[:3], 6, -1)
    with pytest.raises(ValueError, match="same GPU"):
        H._slots("x", meta.slot_mapping, 6, 0)
    for change in (dict(num_decode=3), dict(num_decode=-1), dict(query_start_loc=meta.query_start_loc[:2]),
                   dict(block_tables=meta.block_tables[:1])):
        with pytest.raises(ValueError, match="metadata"):
            H._int4_meta("x", dataclasses.replace(meta, **change))
    with pytest.raises(ValueError, match="on the GPU"):
        H._on_gpu("x", *layer)


def test_tensors_of_another_gpu_than_the_current_one(monkeypatch):
    """The ops launch on the device of their rows: the calls are made over with it as the current one
    (tensors are stood in for; the caches' check, which these do not pass, comes after)."""
    current, entered = [1], []

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)
            self.was, current[0] = current[0], self.device

        def __exit__(self, *_):
            current[0] = self.was

    class Rows:
        device, dtype = torch.device("cuda", 0), torch.float16

        def __init__(self, *shape):
            self.shape = shape

        def get_device(self):
            return 0

        def stride(self):
            return (1,) * len(self.shape)

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch, "empty", lambda *shape, **_: Rows(*shape))
    flat, rows = Rows(2, 48), Rows(2, 1, 16)
    for call in (lambda c: H.kv_write_int4(rows, rows, c, c, None),
                 lambda c: H.rope_kv_write_int4(flat, flat, flat, flat, 1, 1, 16, c, c, None),
                 lambda c: H.kv_read_int4(c, flat),
                 lambda c: H.paged_attention_int4(rows, c, c, None, 1.0)):
        with pytest.raises(ValueError, match="cache.* must be"):
            call(rows)
        assert entered.pop() == 0 and not entered and current == [1]
        current[0] = 0
        with pytest.raises(ValueError, match="cache.* must be"):
            call(rows)
        assert not entered
        current[0] = 1


def test_cache_container_and_namespaces():
    kv = Int4KVCache.new(3, 5, 2, 32, "cpu")
    kc, vc = kv.layer(1)
    assert kc.shape == vc.shape == (5, 2, 320) and kc.dtype == torch.uint8
    kc.fill_(2)
    assert kv.data[1, 0].eq(2).all() and kv.data[1, 1].eq(0).all() and kv.device.type == "cpu"
    with pytest.raises(ValueError, match="head_dim 48"):
        Int4KVCache.new(1, 1, 1, 48, "cpu")
    ref, hip = get_ops("reference"), get_ops("hip")
    for op in ("kv_write_int4", "rope_kv_write_int4", "kv_read_int4", "paged_attention_int4"):
        assert getattr(ref, op) is getattr(R, op) and getattr(hip, op) is getattr(H, op)


def test_engine_on_the_cpu_with_a_4bit_cache():
    """The greedy engine over the twins: chunked prompts and decode rows through one cache."""
    from turingserve_amd.engine import GreedyEngine
    from turingserve_amd.qwen2 import Qwen2Config, Qwen2Model, random_weights

    cfg = Qwen2Config(64, 96, 2, 4, 2, 300, max_position_embeddings=256)
    model = Qwen2Model(cfg, random_weights(cfg, "cpu", dtype=torch.float32, seed=5), get_ops("reference"))
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (40, 3, 17)]
    eng = GreedyEngine(model, 64, max_num_batched_tokens=24, max_model_len=256, kv_cache_dtype="int4")
    out = eng.generate(prompts, 6)
    assert isinstance(eng.kv, Int4KVCache) and eng.mixed_steps > 0 and [len(o) for o in out] == [6] * 3


def test_a_step_asks_for_its_split_map():
    """A decode step is written alike over each cache: its split map is asked for once and handed to every
    layer's attention. This cache has none, and no other is taken."""
    c = Case((4, 2, 16), [(20, 1), (300, 1)], num_decode=2, seed=70)
    _, q, _, _, cache, meta = c.on("cpu")
    layer = cache[0, 0], cache[0, 1]
    want = R.paged_attention_int4(q, *layer, meta, c.scale)
    for ops in (get_ops("reference"), get_ops("hip")):
        split_map = ops.decode_split_map_int4(meta, c.H, c.KVH, c.D, c.NB, cache.device)
        assert split_map is None
        for other in ((torch.zeros(8, dtype=torch.int32), 32), torch.zeros(8), 0):
            with pytest.raises(ValueError, match="split_map"):
                ops.paged_attention_int4(q, *layer, meta, c.scale, split_map=other)
            with pytest.raises(ValueError, match="split_map"):
                ops.paged_attention_int4(q[:0], *layer, meta, c.scale, split_map=other)
    assert torch.equal(R.paged_attention_int4(q, *layer, meta, c.scale, split_map=None), want)
    with pytest.raises(ValueError, match="GPU"):             # (the map is no reason to refuse the call)
        H.paged_attention_int4(q, *layer, meta, c.scale, split_map=None)


@pytest.mark.parametrize("heads", [(4, 2, 16), (6, 2, 32), (12, 2, 128)])
@pytest.mark.parametrize("kind", TINY)
def test_rope_twin_of_tiny_rows(heads, kind):
    c = tiny_rows(heads, kind)
    h, kvh, d = heads
    qkv, _, _, _, cache, meta = c.on("cpu")
    cos, sin = rope_tables(d, 1e6, 64, "cpu")
    R.rope_kv_write_int4(qkv, torch.from_numpy(c.pos), cos, sin, h, kvh, d, cache[0, 0], cache[0, 1],
                         meta.slot_mapping)
    _, kn, vn = c.split()
    turned = O.rotate(kn, cos.numpy()[c.pos], sin.numpy()[c.pos]).astype(np.float32)
    if kind == TINY[0]:                                  # groups whose least number rounds to -0
        least = turned.reshape(c.T, kvh, O.groups(d), -1).min(-1)
        assert ((least < 0) & (least > -2.0 ** -25)).any()
    want = c.cache
    O.write(turned, vn, *want, c.slots)
    assert np.array_equal(cache[0].numpy(), want)


@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_the_cache_is_that_over_coherent_rows(heads):
    """Write and attention against the rows themselves, where the codes' error is small beside the result; and
    what is no such attention does not pass: zeros, the negated or tripled result, one that ignores K, other
    rows' results (of which those of the same sign may)."""
    c = coherent_rows(heads)
    out, cache = over_the_cache(R, "cpu", c)
    ref, bar = over_the_rows(c, cache)
    assert not outside(c, out, ref, bar).any()
    flat, _ = over_the_cache(R, "cpu", c, scale=c.scale * 1e-6)
    seen = np.concatenate([np.arange(n) for _, n in c.items]) >= 8
    for wrong, part in ((out * 0, 0.9), (-out, 0.9), (3 * out, 0.9), (flat, 0.9), (np.roll(out, 7, 0), 0.25)):
        assert outside(c, wrong, ref, bar)[seen].mean() > part


@pytest.mark.parametrize("D", [16, 32, 128])
def test_values_are_within_the_stated_bound(D):
    """Of fp32 rows (a rotated k): half a step, 15 * 2^-24 where the step is subnormal or 0 (it is rounded
    towards zero by up to 2^-24, the group's end by 15 of these; a normal one by 2^-10 of itself, which half
    a step covers), or what a number lies below its group's low in fp16 by; then the value's own rounding."""
    rng = np.random.default_rng(D)
    rows = [rng.uniform(-1, 1, (40, D)) * size for size in (1e-7, 1e-6, 1e-5, 1e-3, 1.0, 300.0, 60000.0)]
    rows += [rng.uniform(0, 1, (40, D)) * 10.0 ** rng.uniform(-6, 2, (40, 1)) + 10.0 ** rng.uniform(-4, 4, (40, 1))]
    few = np.zeros((3, D))
    few[0, 1], few[1, 1], few[2] = 14 * 2.0 ** -24, 29 * 2.0 ** -24, rng.uniform(1000.2, 1000.3, D)
    x = np.concatenate(rows + [few]).astype(np.float32)
    codes, steps, lows = int4_quantise(torch.from_numpy(x))
    mine = O.quantise(x)
    for a, b in zip(mine, (codes.flatten(-2), steps, lows)):
        assert np.array_equal(a, b.numpy())
    held, x = O.values_of(*mine).astype(np.float64), x.astype(np.float64)
    wide = lambda n: np.repeat(n.astype(np.float64), D // O.groups(D), -1)
    step, low = wide(mine[1]), wide(mine[2])
    half = np.maximum(step * (0.5 + 2.0 ** -16), np.where(step < 2.0 ** -14, 15 * 2.0 ** -24, 0.0))
    assert (low - x <= np.maximum(2.0 ** -11 * np.abs(low), 2.0 ** -25)).all()
    off = np.abs(held - x)
    assert (off <= np.maximum(half, low - x) + np.maximum(2.0 ** -11 * np.abs(held), 2.0 ** -25)).all()
    # and no less: groups of a step of 0, of one of 2^-24, and of steps of 0.02 where fp16 has one number in 0.5
    assert (off[-3:-1, 1] == 14 * 2.0 ** -24).all() and step[-3, 1] == 0 and step[-2, 1] == 2.0 ** -24
    assert (off[-1] > 8 * step[-1]).any()
