"""The 8-bit paged cache on the CPU: the oracle against brute force, the torch twins against the
oracle, and every refusal of the entry points."""

from __future__ import annotations

import ctypes
import dataclasses
import subprocess

import numpy as np
import pytest
import torch

from oracle import int8_cache as O
from tests.int8_cases import HEADS, Case, near_the_rows, roll_back
from turingserve_amd import _native as N
from turingserve_amd import get_ops
from turingserve_amd import hip_ops as H
from turingserve_amd import reference_ops as R
from turingserve_amd.csrc import build as B
from turingserve_amd.quant import Int8KVCache
from turingserve_amd.qwen2 import rope_tables

P = ctypes.c_void_p(256)                 # never dereferenced: the call fails validation first


def test_block_write_by_hand():
    codes, scales = np.full((1, 16, 2), 50, np.int8), np.array([2.0], np.float32)
    O.write_block(np.array([[[127.0, -254.0]]]), codes, scales, 0)          # starts anew: scale 2
    assert scales[0] == 2 and codes[0, 0].tolist() == [64, -127]            # 63.5 to even
    O.write_block(np.array([[[508.0, 3.0]]]), codes, scales, 1)             # doubles the scale
    assert scales[0] == 4 and codes[0, :2].tolist() == [[32, -64], [127, 1]]  # -63.5 to even
    O.write_block(np.array([[[0.0, 4.0]]]), codes, scales, 2)               # no larger row: scale stays
    assert scales[0] == 4 and codes[0, :3].tolist() == [[32, -64], [127, 1], [0, 1]]
    assert (codes[0, 3:] == 50).all()
    O.write_block(np.array([[[np.inf, 1.0]]]), codes, scales, 3)
    assert np.isnan(scales[0]) and codes[0, 3].tolist() == [0, 0] and codes[0, 1, 0] == 127
    O.write_block(np.zeros((1, 1, 2)), codes, scales, 0)                    # a new owner
    assert scales[0] == 0 and codes[0, 0].tolist() == [0, 0]


def test_write_in_pieces_holds_every_row_within_its_steps():
    """Rows appended one by one: each is off by half a step of the final scale, plus half a step at
    each requantisation, of which there are at most as many as scales seen."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((16, 1, 8))
    codes, scales = np.zeros((1, 16, 8), np.int8), np.zeros(1, np.float32)
    grew = 0
    for r in range(16):
        was = scales[0]
        O.write_block(np.moveaxis(x[r:r + 1], 0, 1), codes, scales, r)
        grew += scales[0] > was
    err = np.abs(codes[0].astype(np.float64) * scales[0] - x[:, 0])
    assert err.max() <= 0.5 * scales[0] * grew * (1 + 1e-5)


def _of_different_size():
    c = Case((12, 2, 128), [(99, 1), (1999, 1), (15, 1), (0, 90)], num_decode=3, seed=16)
    c.scales[1] = np.exp2(np.random.default_rng(0).integers(-40, 10, c.scales[1].shape)).astype(np.float32)
    c.scales[1, c.tables[2, 0]] = 2.0 ** -20
    c.scales[1, c.tables[1, ::3]] = 0
    return c


def _small_ahead_of_large():
    c = Case((14, 2, 64), [(0, 90), (0, 90)], seed=38)
    c.scales[1, c.tables] = 2.0 ** 8
    c.scales[1, c.tables[0, 0]] = 2.0 ** -12
    c.scales[1, c.tables[1, 0]] = 2.0 ** -17
    return c


@pytest.mark.parametrize("make", [
    _of_different_size, _small_ahead_of_large,
    lambda: Case((4, 2, 16), [(0, 1), (0, 40), (16, 530)], num_decode=1, seed=17),
    lambda: Case((12, 2, 128), [(0, 1), (32, 1), (4095, 1)], num_decode=3, seed=11),
    lambda: Case((14, 2, 64), [(69999, 1)], num_decode=1, seed=12),
    lambda: Case((12, 2, 128), [(0, 1), (39, 1), (1999, 1)], num_decode=3, seed=15, k_size=1e5),
    lambda: Case((12, 2, 128), [(0, 1), (39, 1), (1999, 1)], num_decode=3, seed=15, k_size=0.0)])
def test_attention_bound_catches_a_lost_result(make):
    """The oracle's bound is a small part of every (row, head)'s values: less than 1/32 of their rms (or
    of fp16's smallest normal number), so that a result of zeros, or of other tokens, does not pass."""
    c = make()
    ref, bound = O.paged_attention(c.split()[0], c.codes, c.scales, c.tables, c.lens, c.starts, c.scale)
    rms = lambda x: np.sqrt((x.reshape(c.T, c.H, c.D) ** 2).mean(-1))
    assert (rms(bound) < np.maximum(rms(ref), 2.0 ** -14) / 32).all()


@pytest.mark.parametrize("heads", HEADS)
def test_twins_match_the_oracle(heads):
    c = Case(heads, [(4, 1), (15, 1), (0, 1), (0, 21), (7, 30)], num_decode=3, seed=2)
    qkv, q, k, v, cache, meta = c.on("cpu")
    _, kn, vn = c.split()
    want_c, want_s = c.codes.copy(), c.scales.copy()
    for j, x in enumerate((kn, vn)):
        O.write(x, want_c[j], want_s[j], c.tables, c.lens, c.starts)
    R.kv_write_int8(k, v, *cache, meta)
    assert np.array_equal(torch.stack(cache[:2]).numpy(), want_c)
    assert np.array_equal(torch.stack(cache[2:]).numpy(), want_s)
    out = R.paged_attention_int8(q, *cache, meta, c.scale)
    ref, bound = O.paged_attention(c.split()[0], want_c, want_s, c.tables, c.lens, c.starts, c.scale)
    assert (np.abs(out.double().numpy() - ref) <= bound).all()


@pytest.mark.parametrize("what", ["short table", "fewer positions", "foreign blocks", "nan", "inf"])
def test_attention_twin_keeps_the_contract(what):
    """Tables that do not hold the sequence, rows before its first token, ids outside the cache, blocks
    without a finite scale: as the kernels, by the oracle."""
    c = Case((4, 2, 16), [(20, 1), (5, 60), (0, 0), (0, 3)], num_decode=1, seed=41)
    hit = np.zeros((c.T, c.H), bool)
    if what == "short table":
        c.tables = np.ascontiguousarray(c.tables[:, :2])
    elif what == "fewer positions":
        c.lens[1] = 20
    elif what == "foreign blocks":
        c.tables[0, 1], c.tables[1, 1] = c.NB, -1
    else:
        c.scales[0 if what == "inf" else 1, c.tables[1, 2], 1] = float(what)
        hit[1 + 27:61, 2:] = True                        # positions 32 and later of the second sequence
    _, q, _, _, cache, meta = c.on("cpu")
    out = R.paged_attention_int8(q, *cache, meta, c.scale).double().numpy()
    c.tables[(c.tables < 0) | (c.tables >= c.NB)] = 0
    clean = np.where(np.isfinite(c.scales), c.scales, 0)
    ref, bound = O.paged_attention(c.split()[0], c.codes, clean, c.tables, c.lens, c.starts, c.scale)
    rows = np.repeat(hit, c.D, axis=1)
    assert np.isnan(out[rows]).all() and (np.abs(out - ref) <= bound)[~rows].all()
    if what == "fewer positions":
        assert not out[1:41].any() and out[41:61].any()


def test_twins_of_sequences_without_rows():
    c = Case((4, 2, 16), [(20, 1), (40, 0), (0, 0), (5, 20)], num_decode=1, seed=5)
    _, q, k, v, cache, meta = c.on("cpu")
    R.kv_write_int8(k, v, *cache, meta)
    want = c.codes.copy(), c.scales.copy()
    for j, x in enumerate(c.split()[1:]):
        O.write(x, want[0][j], want[1][j], c.tables, c.lens, c.starts)
    assert np.array_equal(torch.stack(cache[:2]).numpy(), want[0])
    assert np.array_equal(torch.stack(cache[2:]).numpy(), want[1])
    assert R.paged_attention_int8(q, *cache, meta, c.scale).shape == (c.T, c.H * c.D)


def test_rope_twin_matches_the_oracle():
    c = Case((6, 2, 32), [(4, 1), (0, 21), (7, 30)], num_decode=1, seed=3)
    qkv, _, _, _, cache, meta = c.on("cpu")
    cos, sin = rope_tables(32, 1e6, 64, "cpu")
    q = R.rope_kv_write_int8(qkv, torch.from_numpy(c.pos), cos, sin, 6, 2, 32, *cache, meta)
    qn, kn, vn = c.split()
    cn, sn = cos.numpy()[c.pos], sin.numpy()[c.pos]
    want_c, want_s = c.codes.copy(), c.scales.copy()
    O.write(O.rotate(kn, cn, sn), want_c[0], want_s[0], c.tables, c.lens, c.starts)
    O.write(vn, want_c[1], want_s[1], c.tables, c.lens, c.starts)
    assert np.array_equal(torch.stack(cache[:2]).numpy(), want_c)
    assert np.array_equal(torch.stack(cache[2:]).numpy(), want_s)
    assert np.array_equal(q.numpy(), O.rotate(qn, cn, sn).astype(np.float32).astype(np.float16))


@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_the_cache_is_near_that_over_the_rows(heads):
    near_the_rows(R, "cpu", heads)


def test_rows_that_are_taken_back_keep_their_say():
    roll_back(R, "cpu")


def _write(**kw):
    a = dict(k=P, v=P, kst=64, ksh=64, vst=64, vsh=64, kc=P, vc=P, ks=P, vs=P, nb=4, bt=P, bts=4,
             mb=4, sl=P, qsl=P, seqs=1, dec=0, mq=1, T=1, kvh=1, D=64)
    a.update(kw)
    return N.lib().ts_kv_write_int8(*a.values(), None)


def _rope(**kw):
    a = dict(qkv=P, st=256, pos=P, cos=P, sin=P, mp=16, q=P, kc=P, vc=P, ks=P, vs=P, nb=4, bt=P,
             bts=4, mb=4, sl=P, qsl=P, seqs=1, dec=0, mq=1, T=1, h=2, kvh=1, D=64)
    a.update(kw)
    return N.lib().ts_rope_kv_write_int8(*a.values(), None)


def _attend(**kw):
    a = dict(q=P, qst=128, qsh=64, out=P, ost=128, T=1, kc=P, vc=P, ks=P, vs=P, nb=4, bt=P, bts=4,
             mb=4, sl=P, qsl=P, seqs=1, dec=0, mq=1, ms=64, mp=64, h=2, kvh=1, D=64, scale=0.125,
             ws=None, wsb=0)
    a.update(kw)
    return N.lib().ts_paged_attention_int8(*a.values(), None)


odd = ctypes.c_void_p(258)


@pytest.mark.parametrize("call,kw,status,text", [
    (_write, dict(T=-1), N.TS_ERR_INVALID_ARG, "num_tokens"),
    (_write, dict(k=None), N.TS_ERR_INVALID_ARG, "null"),
    (_write, dict(vs=None), N.TS_ERR_INVALID_ARG, "null"),
    (_write, dict(dec=2), N.TS_ERR_INVALID_ARG, "num_decode"),
    (_write, dict(D=96), N.TS_ERR_UNSUPPORTED, "head_dim 96"),
    (_write, dict(bts=3), N.TS_ERR_INVALID_ARG, "bt_stride"),
    (_write, dict(mb=0), N.TS_ERR_INVALID_ARG, "max_blocks"),
    (_write, dict(kst=67), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(k=odd), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(vc=odd), N.TS_ERR_INVALID_ARG, "aligned"),
    (_write, dict(seqs=1 << 30, mq=1 << 20), N.TS_ERR_UNSUPPORTED, "workgroups"),
    (_rope, dict(cos=None), N.TS_ERR_INVALID_ARG, "null"),
    (_rope, dict(mp=0), N.TS_ERR_INVALID_ARG, "empty table"),
    (_rope, dict(st=252), N.TS_ERR_INVALID_ARG, "aligned"),
    (_rope, dict(st=248), N.TS_ERR_INVALID_ARG, "qkv rows"),
    (_rope, dict(h=0), N.TS_ERR_INVALID_ARG, "num_heads"),
    (_rope, dict(D=48), N.TS_ERR_UNSUPPORTED, "head_dim 48"),
    (_attend, dict(seqs=-1), N.TS_ERR_INVALID_ARG, "num_seqs"),
    (_attend, dict(dec=1, T=0), N.TS_ERR_INVALID_ARG, "num_decode"),
    (_attend, dict(ks=None), N.TS_ERR_INVALID_ARG, "null"),
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
    assert call(**kw) == status and text in N.last_error()


@pytest.mark.parametrize("kw", [
    dict(seqs=1 << 20, dec=1 << 20, T=1 << 20, h=32, kvh=32, D=16, qst=512, qsh=16, ost=512, ms=1 << 14),   # splits
    dict(seqs=1 << 20, T=1 << 20, h=512, kvh=4, D=16, qst=8192, qsh=16, ost=8192, ms=1 << 14, mp=1 << 14),  # of chunks
    dict(seqs=1, T=1 << 20, mq=1 << 20, ms=1 << 21, mp=1 << 21, mb=1 << 17, bts=1 << 17, h=64, kvh=8, qst=4096,
         ost=4096),                                                                                        # steps
])
def test_more_work_than_is_counted_is_refused_before_the_device_is_asked(kw):
    """(It used to end where the count did, with the rest of the rows never written.)"""
    assert _attend(**kw, ws=P, wsb=1 << 62) == N.TS_ERR_UNSUPPORTED and "tables of" in N.last_error()


def test_split_edges_up_to_the_longest_table(tmp_path):
    """The kernel's own rule, compiled for the host: the splits of up to 2^26 blocks (the longest table
    that the entry point takes) follow one another, cover every block and differ by one at most."""
    src = tmp_path / "edges.hip"
    src.write_text("""#include <cstdio>
#include "decode_int8.h"
int main() {
  const int sizes[] = {1, 15, 63, 64, 65, 1023, 1025, 4375, (1 << 25) - 1, 1 << 25, (1 << 25) + 1,
                       (1 << 26) - 63, (1 << 26) - 1, 1 << 26};
  for (int nb : sizes)
    for (int splits = 1; splits <= ts::kI8MaxSplits; ++splits) {
      std::printf("%d %d", nb, splits);
      for (int i = 0; i <= splits; ++i) std::printf(" %d", ts::i8_split_begin(nb, i, splits));
      std::printf("\\n");
    }
}
""")
    exe = tmp_path / "edges"
    subprocess.run([B.hipcc(), *B.COMMON_FLAGS, "--offload-host-only", f"-I{B.HERE}", str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 14 * 64
    for line in lines:
        nb, splits, *edges = map(int, line.split())
        sizes = np.diff(edges)
        assert edges[0] == 0 and edges[-1] == nb and len(sizes) == splits
        assert sizes.min() >= 0 and sizes.max() - sizes.min() <= 1


def test_empty_calls_and_workspace_sizes():
    assert _write(T=0) == N.TS_OK and _rope(T=0) == N.TS_OK
    assert _attend(T=0) == N.TS_OK and _attend(seqs=0, T=0) == N.TS_OK
    size = N.lib().ts_paged_attention_int8_workspace_bytes
    assert size(1, 2, 1, 64, 0, 2, 1, 64, 256) == 0 and size(1, 1, 1, 64, 0, 3, 2, 64, 256) == 0
    assert size(64, 64, 1, 256, 0, 12, 2, 128, 256) == 0                 # one split a row
    long = size(4, 4, 1, 32768, 0, 12, 2, 128, 256)
    assert long >= 4 * 12 * 64 * (128 + 2) * 4
    assert size(8, 8, 1, 32768, 0, 12, 2, 128, 256) > long
    # the host's bounds may be anything
    huge = 2 ** 31 - 1
    assert size(64, 0, huge, huge, huge, 64, 8, 128, 256) == size(64, 0, 4096, 65536, 65536, 64, 8, 128, 256)
    # chunks of several tiles of 16 rows leave no more partials than one tile, but for a split a tile
    tile = 16 * 64 * (128 + 2) * 4 * 4
    assert tile <= size(4, 0, 16, 32768, 32768, 8, 8, 128, 256) / 8 < 1.01 * tile
    assert tile <= size(4, 0, 128, 32768, 32768, 8, 8, 128, 256) / 8 < 1.15 * tile


def test_python_wrappers_refuse():
    c = Case((2, 1, 64), [(3, 1), (0, 5)], num_decode=1)
    qkv, q, k, v, cache, meta = c.on("cpu")
    cos, sin = rope_tables(64, 1e6, 64, "cpu")
    for call in (lambda: H.kv_write_int8(k, v, *cache, meta),
                 lambda: H.rope_kv_write_int8(qkv, torch.from_numpy(c.pos), cos, sin, 2, 1, 64, *cache, meta),
                 lambda: H.paged_attention_int8(q, *cache, meta, 0.1)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    # the cache's and the metadata's checks come before anything is launched
    bad = [(cache[0].float(), *cache[1:]), (cache[0][:, :, :8], cache[1][:, :, :8], *cache[2:]),
           (*cache[:3], cache[3].double()), (*cache[:3], cache[3][:-1]),
           (cache[0].transpose(0, 1), cache[1].transpose(0, 1), *cache[2:])]
    for cc in bad:
        with pytest.raises(ValueError):
            H._int8_args("x", *cc, meta, torch.device("cpu"))
    for change in (dict(num_decode=3), dict(query_start_loc=meta.query_start_loc[:2]),
                   dict(block_tables=meta.block_tables[:1])):
        with pytest.raises(ValueError, match="metadata"):
            H._int8_args("x", *cache, dataclasses.replace(meta, **change), torch.device("cpu"))
    with pytest.raises(ValueError, match="same GPU"):
        H._int8_args("x", *cache, meta, torch.device("cuda", 0))


def test_tensors_of_another_gpu_than_the_current_one(monkeypatch):
    """The ops launch on the device of their rows: the calls are made over with it as the current one
    (tensors are stood in for; the caches' check, which these do not pass, comes after)."""
    current, entered = [1], []

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)
            self.was, current[0] = current[0], self.device.index

        def __exit__(self, *_):
            current[0] = self.was

    class Rows:
        is_cuda, device, dtype = True, torch.device("cuda", 0), torch.float16

        def __init__(self, *shape):
            self.shape = shape

        def dim(self):
            return len(self.shape)

        def stride(self, _):
            return 1

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch, "empty", lambda *shape, **_: Rows(*shape))
    flat, rows = Rows(2, 48), Rows(2, 1, 16)
    for call in (lambda c: H.kv_write_int8(rows, rows, c, c, c, c, None),
                 lambda c: H.rope_kv_write_int8(flat, flat, flat, flat, 1, 1, 16, c, c, c, c, None),
                 lambda c: H.paged_attention_int8(rows, c, c, c, c, None, 1.0)):
        with pytest.raises(ValueError, match="caches must be"):
            call(rows)
        assert entered.pop() == torch.device("cuda", 0) and not entered and current == [1]
        current[0] = 0
        with pytest.raises(ValueError, match="caches must be"):
            call(rows)
        assert not entered
        current[0] = 1


def test_cache_container_and_namespaces():
    kv = Int8KVCache.new(3, 5, 2, 32, "cpu")
    kc, vc, ks, vs = kv.layer(1)
    assert kc.shape == vc.shape == (5, 2, 16, 32) and ks.shape == vs.shape == (5, 2)
    ks.fill_(2.0)
    assert kv.scales[1, 0].eq(2).all() and kv.scales[1, 1].eq(0).all() and kv.device.type == "cpu"
    ref, hip = get_ops("reference"), get_ops("hip")
    for op in ("kv_write_int8", "rope_kv_write_int8", "paged_attention_int8"):
        assert getattr(ref, op) is getattr(R, op) and getattr(hip, op) is getattr(H, op)


def test_engine_on_the_cpu_with_an_8bit_cache():
    """The greedy engine over the twins: chunked prompts and decode rows through one cache; an
    unknown cache type is refused."""
    from turingserve_amd.engine import GreedyEngine
    from turingserve_amd.qwen2 import Qwen2Config, Qwen2Model, random_weights

    cfg = Qwen2Config(64, 96, 2, 4, 2, 300, max_position_embeddings=256)
    model = Qwen2Model(cfg, random_weights(cfg, "cpu", dtype=torch.float32, seed=5), get_ops("reference"))
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (40, 3, 17)]
    eng = GreedyEngine(model, 64, max_num_batched_tokens=24, max_model_len=256, kv_cache_dtype="int8")
    out = eng.generate(prompts, 6)
    assert isinstance(eng.kv, Int8KVCache) and eng.mixed_steps > 0 and [len(o) for o in out] == [6] * 3
    with pytest.raises(ValueError, match="fp8"):
        GreedyEngine(model, 64, kv_cache_dtype="fp8")
