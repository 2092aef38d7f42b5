"""The ``reference`` op namespace: pure-PyTorch twins of every op (CPU or GPU).

These restate ops/reference.py:13-111 with the same numerics (fp32 math where the twins use it,
the HF cast order for the norms), so ``get_ops("reference")`` behaves like the reference's
``--kernels reference`` switch. They are slow and simple; the ``hip`` namespace is checked
against them.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from turingserve_amd.quant import LinearWeight, dequantize


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """RMS in fp32, cast back to x.dtype, then times the weight (ops/reference.py:13-16)."""
    x32 = x.float()
    y = x32 * torch.rsqrt(x32.pow(2).mean(-1, keepdim=True) + eps)
    return w * y.to(x.dtype)


def rmsnorm_residual(x: torch.Tensor, residual: torch.Tensor | None, w: torch.Tensor,
                     eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """residual <- x + residual (in x.dtype), out = rmsnorm(residual) (ops/reference.py:19-23)."""
    new_res = x if residual is None else x + residual
    return rmsnorm(new_res, w, eps), new_res


def silu_mul(gu: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for gu = [gate | up] (ops/reference.py:26-28)."""
    i = gu.shape[-1] // 2
    return F.silu(gu[..., :i]) * gu[..., i:]


def rope_(qkv: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
          H: int, KVH: int, D: int) -> None:
    """In-place rotate-half RoPE on the q and k heads of qkv [T, (H + 2 KVH) D]; the fp32 tables
    are cast to the activation dtype first (ops/reference.py:31-42)."""
    T = qkv.shape[0]
    c = cos[positions].to(qkv.dtype)[:, None, :]
    s = sin[positions].to(qkv.dtype)[:, None, :]
    qk = qkv[:, : (H + KVH) * D].view(T, H + KVH, D)
    half = D // 2
    x1, x2 = qk[..., :half], qk[..., half:]
    o1 = x1 * c - x2 * s
    o2 = x2 * c + x1 * s
    qk[..., :half] = o1
    qk[..., half:] = o2


def linear(x: torch.Tensor, lw: LinearWeight) -> torch.Tensor:
    """Dequantise to x.dtype (if int8), then F.linear (ops/reference.py:45-47)."""
    w = dequantize(lw.w, lw.scale, x.dtype) if lw.quantized else lw.w
    return F.linear(x, w, lw.b)


def kv_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             slot_mapping: torch.Tensor) -> None:
    """cache[slot // 16, :, slot % 16, :] = row for slot >= 0 (ops/reference.py:50-57)."""
    keep = slot_mapping >= 0
    slots = slot_mapping[keep]
    blk, off = slots // 16, slots % 16
    k_cache[blk, :, off, :] = k[keep]
    v_cache[blk, :, off, :] = v[keep]


def attention_with_mask(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        scale: float) -> torch.Tensor:
    """q [Tq, H, D], k/v [Tk, KVH, D] -> [Tq, H*D]; fp32 math with an explicit bottom-right
    causal mask j <= (Tk - Tq) + i (ops/reference.py:60-77)."""
    Tq, H, D = q.shape
    Tk, KVH, _ = k.shape
    G = H // KVH
    qf = q.float().permute(1, 0, 2)
    kf = k.float().repeat_interleave(G, dim=1).permute(1, 0, 2)
    vf = v.float().repeat_interleave(G, dim=1).permute(1, 0, 2)
    scores = torch.matmul(qf, kf.transpose(1, 2).contiguous()) * scale
    i = torch.arange(Tq, device=q.device)[:, None]
    j = torch.arange(Tk, device=q.device)[None, :]
    scores = scores.masked_fill(~(j <= (Tk - Tq) + i), float("-inf"))
    p = torch.softmax(scores, dim=-1)
    out = torch.matmul(p, vf).permute(1, 0, 2)
    return out.reshape(Tq, H * D).to(q.dtype)


def dense_causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           scale: float) -> torch.Tensor:
    """Causal attention with q_len == kv_len (ops/reference.py:80-91)."""
    T, H, D = q.shape
    G = H // k.shape[1]
    kk = k.repeat_interleave(G, dim=1)
    vv = v.repeat_interleave(G, dim=1)
    out = F.scaled_dot_product_attention(
        q.permute(1, 0, 2)[None], kk.permute(1, 0, 2)[None], vv.permute(1, 0, 2)[None],
        is_causal=True, scale=scale)
    return out[0].permute(1, 0, 2).reshape(T, H * D)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, meta,
                    scale: float) -> torch.Tensor:
    """Per-sequence gather of the paged cache, then attention_with_mask; rows of sequences with
    seq_len 0 stay 0 (ops/reference.py:94-111)."""
    T, H, D = q.shape
    KVH = k_cache.shape[1]
    out = torch.zeros(T, H * D, dtype=q.dtype, device=q.device)
    qsl = meta.query_start_loc.tolist()
    for b, seq_len in enumerate(meta.seq_lens.tolist()):
        qs, qe = qsl[b], qsl[b + 1]
        if seq_len == 0 or qe == qs:
            continue
        nb = -(-seq_len // 16)
        blocks = meta.block_tables[b, :nb].long()
        kk = k_cache[blocks].permute(0, 2, 1, 3).reshape(nb * 16, KVH, D)[:seq_len]
        vv = v_cache[blocks].permute(0, 2, 1, 3).reshape(nb * 16, KVH, D)[:seq_len]
        out[qs:qe] = attention_with_mask(q[qs:qe], kk, vv, scale)
    return out


def kv_write_int8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor, meta) -> None:
    """Twin of the quantising write into an 8-bit paged cache (codes [NB, KVH, 16, D] int8, scales
    [NB, KVH] fp32), a block at a time. k, v [T, KVH, D] in any floating type."""
    qsl, tables = meta.query_start_loc.tolist(), meta.block_tables.tolist()
    for b, length in enumerate(meta.seq_lens.tolist()):
        start = length - (qsl[b + 1] - qsl[b])
        if start == length:
            continue
        for j in range(max(start, 0) // 16, -(-length // 16)):
            if j >= len(tables[b]) or not 0 <= tables[b][j] < k_cache.shape[0]:
                continue
            lo, hi = max(start, 16 * j), min(length, 16 * (j + 1))
            rows = slice(qsl[b] + lo - start, qsl[b] + hi - start)
            for x, codes, scales in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
                _write_block(x[rows].transpose(0, 1).float(), codes[tables[b][j]],
                             scales[tables[b][j]], max(lo, 0) - 16 * j)


def _write_block(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, at: int) -> None:
    """Rows x [KVH, n, D] fp32 into rows at .. at + n - 1 of one block, in place."""
    was = scales.clone() if at > 0 else torch.zeros_like(scales)
    top = x.abs().amax((1, 2))
    scale = torch.maximum(was, top / torch.full_like(top, 127.0))
    scale = torch.where(torch.isfinite(top), scale, torch.nan)
    for h, (old, new) in enumerate(zip(was.tolist(), scale.tolist())):
        if new > old:
            codes[h, :at] = torch.round(codes[h, :at].float() * (was[h] / scale[h])).to(torch.int8)
        codes[h, at:at + x.shape[1]] = \
            torch.round(x[h] / scale[h]).clamp(-127, 127).to(torch.int8) if new > 0 else 0
    scales.copy_(scale)


def rope_kv_write_int8(qkv: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor,
                       sin: torch.Tensor, H: int, KVH: int, D: int, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                       meta) -> torch.Tensor:
    """Twin: rotate-half RoPE of q (returned, [T, H, D], rounded once) and k (rounded to fp32), then
    kv_write_int8 of the rotated k and of v."""
    T, half = qkv.shape[0], D // 2
    pos = positions[:T].clamp(0, cos.shape[0] - 1)
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    x = qkv[:, :(H + 2 * KVH) * D].view(T, H + 2 * KVH, D)
    x1, x2 = x[:, :H + KVH, :half].double(), x[:, :H + KVH, half:].double()
    qk = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).float()
    kv_write_int8(qk[:, H:], x[:, H + KVH:], k_cache, v_cache, k_scale, v_scale, meta)
    return qk[:, :H].to(qkv.dtype)


def paged_attention_int8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         k_scale: torch.Tensor, v_scale: torch.Tensor, meta,
                         scale: float) -> torch.Tensor:
    """Twin: the sequences' blocks as fp32 values, then causal attention over the tokens that the table
    holds (block ids outside the cache read block 0). Rows that see no token are zeros, rows that see a
    block whose K or V scale is not finite NaN."""
    T, H, D = q.shape
    NB, KVH = k_scale.shape
    out = torch.zeros(T, H * D, dtype=q.dtype, device=q.device)
    qsl = meta.query_start_loc.tolist()
    for b, seq_len in enumerate(meta.seq_lens.tolist()):
        qs, qe = qsl[b], qsl[b + 1]
        held = min(seq_len, 16 * meta.block_tables.shape[1])
        if held <= 0 or qe <= qs:
            continue
        blocks = meta.block_tables[b, :-(-held // 16)].long()
        blocks = torch.where((blocks >= 0) & (blocks < NB), blocks, 0)
        bad = ~(torch.isfinite(k_scale[blocks]) & torch.isfinite(v_scale[blocks]))
        kk, vv = ((c[blocks].float() * s[blocks].masked_fill(bad, 0.0)[:, :, None, None])
                  .permute(1, 0, 2, 3).reshape(KVH, -1, D)[:, :held].repeat_interleave(H // KVH, 0)
                  for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        bad = bad.repeat_interleave(16, 0)[:held].T.repeat_interleave(H // KVH, 0)      # [H, held]
        last = torch.arange(seq_len - (qe - qs), seq_len, device=q.device)               # a row's own position
        seen = torch.arange(held, device=q.device) <= last[:, None]                      # [rows, held]
        scores = torch.matmul(q[qs:qe].float().permute(1, 0, 2), kk.transpose(1, 2).contiguous()) * scale
        p = torch.softmax(scores.masked_fill(~seen, float("-inf")), dim=-1).masked_fill(~seen, 0.0)
        o = torch.matmul(p, vv).permute(1, 0, 2)
        o = o.masked_fill((seen[:, None] & bad).any(-1)[:, :, None], float("nan"))
        out[qs:qe] = o.reshape(qe - qs, H * D).to(q.dtype)
    return out
