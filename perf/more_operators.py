"""The operators of the 4-bit paged KV cache: their cases, inputs, plain forms and 64-bit results.

The cache holds, for each token, KV head and group of 32 channels, 4-bit codes and two fp16 numbers,
step and low; a code stands for fp16(low + code * step), rounded once. A group's low is its least
value in fp16, its step (largest value - low) / 15 in fp32, rounded towards zero to fp16, and a code
rint((value - low) / step) within 0 .. 15 (0 where the step is 0). Four operators share it:

write    New K/V rows, each into the block and row that its position names. With `rope`, q and k are
         rotated (rotate-half, tables in fp32) on the way: q is returned and the rotated k, rounded
         once to 32 bits, is quantised. The pass returns the cache's values, read back.
read     The values of blocks of every layer's cache, as fp16.
decode   Attention of one query row per sequence over its cached rows.
prefill  Causal attention of several query rows per sequence (prompt chunks on a cached prefix,
         the rows of a speculative step), with or without decode rows beside them.

Several layers with caches of their own stand in one pass, as in a model. Sequence lengths follow
from the case alone (spread evenly over the logarithm of their range); the seed shuffles them and
draws every value. Batches of single rows are replayed from a graph, as graphs.DecodeGraphs serves
them; the others are eager calls, as the engine makes them.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 16
GROUP = 32
THETA = 1e6
HEADS = [(12, 2, 128), (14, 2, 64), (28, 4, 128), (8, 8, 64)]


# ---------------------------------------------------------------------------- the cases
def _case(name, kind, heads, layers, decodes=0, ctx=(1, 1), chunks=0, q=(1, 1), prefix=(0, 0),
          rope=False):
    h, kvh, d = heads
    return dict(name=name, kind=kind, heads=h, kv_heads=kvh, head_dim=d, layers=layers,
                decodes=decodes, ctx_lo=ctx[0], ctx_hi=ctx[1], chunks=chunks, q_lo=q[0], q_hi=q[1],
                prefix_lo=prefix[0], prefix_hi=prefix[1], rope=rope)


def listed():
    g6, g7, wide, _ = HEADS
    return [
        # a decode batch's new rows, each appended somewhere inside its sequence's last block
        _case("write_append_64_d128", "write", g6, 8, decodes=64, ctx=(128, 4096), rope=True),
        # a 2048-token chunk of a long prompt
        _case("write_chunk_2048_d128", "write", g6, 2, chunks=1, q=(2048, 2048),
              prefix=(4096, 4096), rope=True),
        # several prompts of odd lengths that go on inside a block, rows rotated beforehand
        _case("write_ragged_d64", "write", g7, 2, chunks=5, q=(90, 1100), prefix=(0, 1500)),
        # one user's prefix handed on to a worker whose cache is fp16
        _case("read_1_prefix_d128", "read", g6, 4, decodes=1, ctx=(1500, 1500)),
        # a whole batch's caches, moved out of the card's memory
        _case("read_32_d64", "read", g7, 8, decodes=32, ctx=(200, 8192)),
        # one user's chat, well into its context: latency of a small launch
        _case("decode_1_d128", "decode", g6, 4, decodes=1, ctx=(6000, 6000)),
        # a full decode batch at the 1.5B attention shape, chat lengths
        _case("decode_64_d128", "decode", g6, 4, decodes=64, ctx=(128, 4096)),
        # a few long documents: contexts up to the model's 32768 positions
        _case("decode_4_long", "decode", g6, 4, decodes=4, ctx=(8000, 32768)),
        # one 2048-token chunk of a long prompt on its cached prefix
        _case("prefill_2048_d128", "prefill", g6, 2, chunks=1, q=(2048, 2048), prefix=(4096, 4096)),
        # several prompts of mixed lengths, some with a cached prefix
        _case("prefill_ragged_d64", "prefill", g7, 2, chunks=5, q=(90, 1100), prefix=(0, 1500)),
        # speculative verification: a few drafted rows for each of 16 sequences
        _case("verify_16x5_d128", "prefill", wide, 2, chunks=16, q=(5, 5), prefix=(300, 3000)),
        # continuous batching: 48 decoding sequences beside one 512-token prompt chunk
        _case("mixed_48_512_d128", "prefill", g6, 4, decodes=48, ctx=(256, 4096), chunks=1,
              q=(512, 512), prefix=(200, 200)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _drawn(rng)
        w = work(case)                                    # no more than the largest listed ones
        if w["flops"] < 120e9 and w["bytes"] < 400e6:
            return case


def _drawn(rng):
    kind = rng.choice(["write", "write", "read", "decode", "decode", "decode", "prefill", "prefill",
                       "prefill"])
    heads = rng.choice(HEADS)
    row_bytes = 2 * heads[1] * heads[2]
    if kind in ("decode", "read") or (kind == "write" and rng.random() < 0.5):
        hi = _log(rng, 100, 32768)
        lo = _log(rng, max(1, hi // 50), hi)
        most = min(128, int(50e6 / (row_bytes * (lo + hi) / 2)))
        case = _case("", kind, heads, rng.choice([1, 2, 4]), decodes=_log(rng, 1, max(1, most)),
                     ctx=(lo, hi), rope=kind == "write" and rng.random() < 0.7)
    else:
        q_hi = _log(rng, 2, 2048)
        q_lo = _log(rng, max(1, q_hi // 8), q_hi)
        prefix_hi = rng.choice([0, _log(rng, 16, 4000)])
        prefix_lo = rng.choice([0, prefix_hi // 3])
        mixed = kind == "prefill" and rng.random() < 0.4
        ctx_hi = _log(rng, 50, 4096)
        case = _case("", kind, heads, rng.choice([1, 2]),
                     decodes=_log(rng, 1, 48) if mixed else 0,
                     ctx=(max(1, ctx_hi // 10), ctx_hi) if mixed else (1, 1),
                     chunks=rng.randint(1, max(1, min(16, 2048 // q_hi))), q=(q_lo, q_hi),
                     prefix=(prefix_lo, prefix_hi), rope=kind == "write" and rng.random() < 0.7)
    case.pop("name")
    return case


def _spread(n, lo, hi):
    """n lengths spread evenly over the logarithm of [lo, hi]."""
    if n == 0 or hi == 0:
        return [0] * n
    lo = max(lo, 1)
    return [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]


def _lengths(case):
    """(cached, new) rows of each sequence: decode rows, then chunks, the longest chunks on the
    shortest prefixes. In an order without a seed."""
    dec = [(c - 1, 1) for c in _spread(case["decodes"], case["ctx_lo"], case["ctx_hi"])]
    n, lo, hi = case["chunks"], case["prefix_lo"], case["prefix_hi"]
    pre = [lo + (hi - lo) * (n - 1 - i) // (n - 1) if n > 1 else hi for i in range(n)]
    return dec, list(zip(pre, _spread(n, case["q_lo"], case["q_hi"])))


def work(case):
    h, kvh, d, layers = case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
    dec, chunks = _lengths(case)
    items = dec + chunks
    rows = sum(n for _, n in items)
    values = 2 * kvh * d                                  # of one token, K and V
    row = values // 2 + 4 * values // GROUP               # bytes: codes, a step and a low a group
    blocks = sum(-(-(c + n) // BLOCK) for c, n in items)
    if case["kind"] == "write":
        # new rows read in 16 bits and written as codes, and the blocks that they fall in read
        # back; with rope, q read and written and the tables' rows
        touched = sum((c + n - 1) // BLOCK - c // BLOCK + 1 for c, n in items)
        nbytes = rows * (2 * values + row) + touched * BLOCK * (row + 2 * values)
        flops = rows * values * 4 + touched * BLOCK * values * 2
        if case["rope"]:
            nbytes += rows * (2 * h * d * 2 + d * 4)
            flops += rows * (h + kvh) * d * 3
        return dict(bytes=layers * nbytes, flops=layers * flops)
    if case["kind"] == "read":
        return dict(bytes=layers * blocks * BLOCK * (row + 2 * values),
                    flops=layers * blocks * BLOCK * values * 2)
    cached = sum(c + n for c, n in items)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in items)   # (query row, visible key)
    nbytes = cached * row + blocks * 4 + 2 * rows * h * d * 2
    return dict(bytes=layers * nbytes, flops=layers * 4 * pairs * h * d)


# ---------------------------------------------------------------------------- inputs
def _batch(case, seed):
    """The step's metadata (host lists and device tensors) with a shuffled block table. A write
    touches only the blocks that its new rows fall in: the blocks before them stand as block 0 in
    the tables, so that the cache holds what the operator returns and nothing else."""
    g = torch.Generator().manual_seed(seed)
    items = []
    for part in _lengths(case):
        items += [part[i] for i in torch.randperm(len(part), generator=g).tolist()]
    first = [c // BLOCK if case["kind"] == "write" else 0 for c, _ in items]
    last = [-(-(c + n) // BLOCK) for c, n in items]
    blocks = sum(b - a for a, b in zip(first, last)) + 1      # block 0 is the null block
    free = (torch.randperm(blocks - 1, generator=g) + 1).to(torch.int32)
    tables = torch.zeros(len(items), max(last), dtype=torch.int32)
    starts, at = [0], 0
    for b, (c, n) in enumerate(items):
        tables[b, first[b]:last[b]] = free[at:at + last[b] - first[b]]
        at += last[b] - first[b]
        starts.append(starts[-1] + n)
    pos = torch.cat([torch.arange(c, c + n) for c, n in items])
    lens = [c + n for c, n in items]
    nd = case["decodes"]
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(items=items, blocks=blocks, starts=starts, tables=tables.cuda(), used=free.cuda(),
                positions=pos.cuda(), query_start_loc=torch.tensor(starts, **i32),
                seq_lens=torch.tensor(lens, **i32), num_decode=nd,
                max_query_len=max(n for _, n in items), max_seq_len=max(lens),
                max_prefill_seq_len=max(lens[nd:], default=0))


def _inputs(case, seed):
    """(batch, qkv rows [layers, T, (H + 2 KVH) D] fp16, cached rows [layers, 2, blocks, KVH, 16, D]
    fp16 that the cache was written with): K's channels differ in size, a few of them by much, and
    some sit away from zero; V's do not. Old and new rows are alike."""
    b = _batch(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, kvh, d, layers = case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
    rows = b["starts"][-1]
    qkv = torch.empty(layers, rows, (h + 2 * kvh) * d, dtype=torch.float16, device="cuda")
    old = torch.empty(layers, 2, b["blocks"], kvh, BLOCK, d, dtype=torch.float16, device="cuda")
    for i in range(layers):
        size = torch.exp(0.5 * torch.randn(kvh, d, generator=g, device="cuda"))
        mean = size * torch.randn(kvh, d, generator=g, device="cuda") * 0.5
        x = torch.randn(rows, h + 2 * kvh, d, generator=g, device="cuda")
        x[:, h:h + kvh] = x[:, h:h + kvh] * size + mean
        x[:, h + kvh:] *= 0.7
        qkv[i] = x.flatten(1)
        x = torch.randn(2, b["blocks"], kvh, BLOCK, d, generator=g, device="cuda")
        old[i, 0] = x[0] * size[:, None] + mean[:, None]
        old[i, 1] = x[1] * 0.7
    return b, qkv, old


def _tables(case, b):
    """(cos, sin) [positions, D / 2] fp32."""
    d = case["head_dim"]
    freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.outer(torch.arange(b["max_seq_len"], dtype=torch.float64), freq)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def prepare(case, seed):
    b, qkv, old = _inputs(case, seed)
    h, kvh, d, layers = case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
    rows = qkv.shape[1]
    state = dict(case=case, batch=b, qkv=qkv, scale=d ** -0.5,
                 q=qkv[:, :, :h * d].view(layers, rows, h, d),
                 k=qkv[:, :, h * d:(h + kvh) * d].view(layers, rows, kvh, d),
                 v=qkv[:, :, (h + kvh) * d:].view(layers, rows, kvh, d))
    if case["rope"]:
        state["cos"], state["sin"] = _tables(case, b)
    if not own:
        state["codes"], state["steps"], state["lows"] = _quantise(old.float())
        return state
    from turingserve_amd import get_ops
    from turingserve_amd.metadata import AttentionMetadata
    from turingserve_amd.quant import Int4KVCache

    ops = state["ops"] = get_ops("hip")
    cache = state["cache"] = Int4KVCache.new(layers, b["blocks"], kvh, d, "cuda")
    # what the cache was written with: slot after slot
    n = b["blocks"] * BLOCK
    for i in range(layers):
        k, v = (old[i, j].transpose(1, 2).reshape(n, kvh, d) for j in range(2))
        ops.kv_write_int4(k, v, *cache.layer(i), torch.arange(n, device="cuda"))
    state["meta"] = AttentionMetadata(
        query_start_loc=b["query_start_loc"], seq_lens=b["seq_lens"], block_tables=b["tables"],
        slot_mapping=_slots(b), num_decode=b["num_decode"], max_query_len=b["max_query_len"],
        max_seq_len=b["max_seq_len"], max_prefill_seq_len=b["max_prefill_seq_len"])
    if case["chunks"] == 0 and case["kind"] != "read":    # single rows: a captured step
        with torch.inference_mode():
            _run_own(state)
            torch.cuda.synchronize()
            state["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(state["graph"]):
                state["out"] = _run_own(state)
    return state


def _slots(b):
    """The slot of every new row, [T] int64."""
    owner = torch.repeat_interleave(torch.arange(len(b["items"])),
                                    torch.tensor([n for _, n in b["items"]])).cuda()
    pos = b["positions"]
    return b["tables"][owner, pos // BLOCK].long() * BLOCK + pos % BLOCK


# ---------------------------------------------------------------------------- one pass
def run(state):
    if own:
        if "graph" in state:
            state["graph"].replay()
            return state["out"]
        return _run_own(state)
    case = state["case"]
    if case["kind"] == "write":
        return _write_plain(state)
    if case["kind"] == "read":
        return _values(*(state[x][:, :, state["batch"]["used"]] for x in ("codes", "steps", "lows")))
    return [_attend_plain(state, i) for i in range(case["layers"])]


def _run_own(s):
    case, ops, meta, cache = s["case"], s["ops"], s["meta"], s["cache"]
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "read":
        return ops.kv_read_int4(cache.data, s["batch"]["used"])
    out = []
    if case["kind"] != "write":
        # a pure-decode step's plan, shared by its layers
        split_map = (ops.decode_split_map_int4(meta, h, kvh, d, s["batch"]["blocks"], s["q"].device)
                     if case["chunks"] == 0 else None)
        for i in range(case["layers"]):
            out.append(ops.paged_attention_int4(s["q"][i], *cache.layer(i), meta, s["scale"],
                                                split_map=split_map))
        return out
    for i in range(case["layers"]):
        if case["rope"]:
            out.append(ops.rope_kv_write_int4(s["qkv"][i], s["batch"]["positions"], s["cos"],
                                              s["sin"], h, kvh, d, *cache.layer(i),
                                              meta.slot_mapping))
        else:
            ops.kv_write_int4(s["k"][i], s["v"][i], *cache.layer(i), meta.slot_mapping)
    return dict(q=out, cache=ops.kv_read_int4(cache.data, s["batch"]["used"]))


# ---------------------------------------------------------------------------- the plain forms
def _quantise(x):
    """x [..., D] in 32 bits -> codes [..., D / 32, 32], steps and lows [..., D / 32]."""
    x = x.unflatten(-1, (-1, GROUP))
    lows = x.amin(-1).half()
    span = (x.amax(-1) - lows.float()).clamp_min(0) / torch.tensor(15.0, device=x.device)
    steps = span.half()                                   # to the nearest, then towards zero
    steps = (steps.view(torch.int16) - (steps.float() > span).to(torch.int16)).view(torch.float16)
    ratio = (x - lows.float()[..., None]) / steps.float()[..., None]
    codes = torch.where(steps[..., None] > 0, torch.round(ratio).clamp(0, 15), 0)
    return codes.to(torch.uint8), steps, lows


def _values(codes, steps, lows):
    """What the codes stand for, [..., D] fp16."""
    return (codes.float() * steps.float()[..., None] + lows.float()[..., None]).half().flatten(-2)


def _rotate(x, cos, sin):
    """Rotate-half RoPE of x [..., D] by tables that broadcast to [..., D / 2]."""
    half = x.shape[-1] // 2
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)


def _write_plain(s):
    case, b = s["case"], s["batch"]
    k, v, q = s["k"].float(), s["v"].float(), []
    if case["rope"]:
        cos = s["cos"][b["positions"]][:, None]
        sin = s["sin"][b["positions"]][:, None]
        q = list(_rotate(s["q"].float(), cos, sin).half())
        # a quotient next to a border between two codes: the last bit of k decides
        k = _rotate(k.double(), cos.double(), sin.double()).float()
    slot = _slots(b)
    for j, x in enumerate((k, v)):                        # [L, T, KVH, D]
        for name, new in zip(("codes", "steps", "lows"), _quantise(x)):
            s[name][:, j, slot // BLOCK, :, slot % BLOCK] = new.transpose(0, 1)
    return dict(q=q, cache=_values(*(s[x][:, :, b["used"]] for x in ("codes", "steps", "lows"))))


def _cached(s, i, j, table):
    """K's (j = 0) or V's values in the blocks of `table`, in 32 bits."""
    return _values(*(s[x][i, j][table] for x in ("codes", "steps", "lows"))).float()


def _attend_plain(s, i):
    case, b = s["case"], s["batch"]
    q = s["q"][i]
    out = torch.empty(q.shape[0], case["heads"] * case["head_dim"], dtype=torch.float16,
                      device="cuda")
    nd = case["decodes"]
    if nd:
        out[:nd] = _decode_plain(s, i, nd)
    for seq in range(nd, len(b["items"])):
        lo, hi = b["starts"][seq], b["starts"][seq + 1]
        out[lo:hi] = _chunk_plain(s, i, seq, q[lo:hi])
    return out


def _decode_plain(s, i, nd):
    """Rows [0, nd): every sequence padded to the longest."""
    case, b = s["case"], s["batch"]
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    lens = b["seq_lens"][:nd].long()
    width = -(-max(c + n for c, n in b["items"][:nd]) // BLOCK)
    table = b["tables"][:nd, :width].long()
    k, v = (_cached(s, i, j, table).transpose(1, 2).reshape(nd, kvh, width * BLOCK, d)
            for j in range(2))                            # from [S, W, KVH, 16, D]
    q = s["q"][i][:nd].float().view(nd, kvh, h // kvh, d)
    scores = (q @ k.transpose(2, 3).contiguous()) * s["scale"]
    hidden = torch.arange(width * BLOCK, device="cuda") >= lens[:, None, None, None]
    scores = scores.masked_fill(hidden, -torch.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return ((p @ v) / p.sum(-1, keepdim=True)).reshape(nd, h * d).half()


def _chunk_plain(s, i, seq, q):
    """The rows of one sequence's chunk."""
    case, b = s["case"], s["batch"]
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    cached, new = b["items"][seq]
    length = cached + new
    table = b["tables"][seq, :-(-length // BLOCK)].long()
    k, v = (_cached(s, i, j, table).transpose(0, 1).reshape(kvh, -1, d)[:, :length]
            for j in range(2))                            # from [W, KVH, 16, D]
    g = h // kvh
    q = q.float().view(new, kvh, g, d).permute(1, 2, 0, 3).reshape(kvh, g * new, d)
    scores = (q @ k.transpose(1, 2).contiguous()).view(kvh, g, new, length) * s["scale"]
    hidden = (torch.arange(length, device="cuda")[None, :]
              > torch.arange(cached, length, device="cuda")[:, None])
    scores = scores.masked_fill(hidden, -torch.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (p.view(kvh, g * new, length) @ v.contiguous()) / p.sum(-1).view(kvh, g * new, 1)
    return o.view(kvh, g, new, d).permute(2, 0, 1, 3).reshape(new, h * d).half()


# ---------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    b, qkv, old = _inputs(case, seed)
    h, kvh, d, layers = case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
    cache = torch.stack([_held64(x.double()) for x in old])    # what the written rows stand for
    x = qkv.double().view(*qkv.shape[:2], h + 2 * kvh, d)
    q, k, v = x.split([h, kvh, kvh], dim=2)
    if case["kind"] == "read":
        return cache[:, :, b["used"]]
    if case["kind"] == "write":
        q_out = []
        if case["rope"]:
            cos, sin = (t.double()[b["positions"]][None, :, None] for t in _tables(case, b))
            q, k = _turn64(q, cos, sin), _turn64(k, cos, sin).float().double()
            q_out = list(q)
        tables = b["tables"].tolist()
        for j, rows in enumerate((_held64(k), _held64(v))):
            for seq, (cached, new) in enumerate(b["items"]):
                for blk in range(cached // BLOCK, (cached + new - 1) // BLOCK + 1):
                    lo, hi = max(cached, BLOCK * blk), min(cached + new, BLOCK * (blk + 1))
                    at = b["starts"][seq] - cached
                    cache[:, j, tables[seq][blk], :, lo - BLOCK * blk:hi - BLOCK * blk] = \
                        rows[:, at + lo:at + hi].transpose(1, 2)
        return dict(q=q_out, cache=cache[:, :, b["used"]])
    return [_attend64(case, b, q[i], cache[i]) for i in range(layers)]


def _turn64(x, cos, sin):
    half = x.shape[-1] // 2
    out = torch.empty_like(x)
    out[..., :half] = x[..., :half] * cos - x[..., half:] * sin
    out[..., half:] = x[..., half:] * cos + x[..., :half] * sin
    return out


def _held64(x):
    """The values that the cache holds for rows x [..., D]: what is defined in 16 and 32 bits is
    rounded to them, every operation is made in 64."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], GROUP):
        g = x[..., at:at + GROUP]
        low = g.min(-1, keepdim=True).values.half().double()
        span = (torch.clamp((g.max(-1, keepdim=True).values - low).float().double(), min=0) / 15).float()
        # the binary exponent of an fp16's unit in the last place: 10 below its own, -24 at least
        unit = torch.ldexp(torch.ones_like(low), (torch.frexp(span).exponent - 11).clamp_min(-24))
        step = torch.floor(span.double() / unit) * unit
        code = ((g - low).float().double() / step).float().round().clamp(0, 15)
        out[..., at:at + GROUP] = torch.where(step > 0, code.double() * step, 0.0) + low
    return out.half().double()


def _attend64(case, b, q, cache):
    """q [T, H, D] and one layer's values -> [T, H * D], a sequence and a KV head at a time."""
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    g = h // kvh
    out = torch.empty(q.shape[0], h, d, dtype=torch.float64, device="cuda")
    for seq, (cached, new) in enumerate(b["items"]):
        lo, length = b["starts"][seq], cached + new
        blocks = b["tables"][seq, :-(-length // BLOCK)].long()
        last = torch.arange(cached, length, device="cuda").repeat_interleave(g)
        late = torch.arange(length, device="cuda")[None, :] > last[:, None]
        for head in range(kvh):
            k, v = (cache[j, blocks, head].reshape(-1, d)[:length] for j in range(2))
            rows = q[lo:lo + new, head * g:(head + 1) * g].reshape(new * g, d)
            score = torch.mm(rows, k.t().contiguous()) / math.sqrt(d)
            score[late] = -math.inf
            out[lo:lo + new, head * g:(head + 1) * g] = \
                torch.mm(torch.softmax(score, dim=1), v).view(new, g, d)
    return out.view(q.shape[0], h * d)
