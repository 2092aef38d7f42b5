"""The W8A16 weight format: per-output-row symmetric int8 with an fp32 scale; the 8-bit and 4-bit
paged K/V caches.

Restates quant/int8.py:8-16 and the LinearWeight container of model/layers.py:21-31. The GEMM
also accepts fp16 scales (the W8A16 benchmark configuration draws them in fp16; widening fp16
to fp32 is exact).
"""

from __future__ import annotations

from dataclasses import dataclass, field

import torch


@dataclass
class LinearWeight:
    """``w`` is [N, K] fp16/fp32, or int8 with a per-row ``scale`` [N] (W8A16); ``b`` [N] or None."""

    w: torch.Tensor
    b: torch.Tensor | None = None
    scale: torch.Tensor | None = None

    @property
    def quantized(self) -> bool:
        return self.scale is not None


def quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """W [N, K] -> (int8 [N, K], fp32 scale [N]); scale = max|W[n, :]| / 127 clamped to 1e-8."""
    scale = (w.abs().amax(dim=1) / 127.0).clamp_min(1e-8).float()
    wq = torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8)
    return wq, scale


def dequantize(wq: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return (wq.to(torch.float32) * scale.float()[:, None]).to(dtype)


@dataclass
class Int8KVCache:
    """The 8-bit paged KV cache of every layer: codes [L, 2, num_blocks, KVH, 16, D] int8 and one
    fp32 scale per (layer, K or V, block, KV head), [L, 2, num_blocks, KVH]; a code stands for
    code * scale. Per token and layer it takes KVH * (2 D + 0.5) bytes where fp16 takes
    KVH * 4 D."""

    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def new(cls, num_layers: int, num_blocks: int, num_kv_heads: int, head_dim: int,
            device) -> "Int8KVCache":
        shape = (num_layers, 2, num_blocks, num_kv_heads)
        return cls(torch.zeros(*shape, 16, head_dim, dtype=torch.int8, device=device),
                   torch.zeros(*shape, dtype=torch.float32, device=device))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def layer(self, index: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """(k_cache, v_cache, k_scale, v_scale) of one layer, as the ops take them."""
        c, s = self.codes[index], self.scales[index]
        return c[0], c[1], s[0], s[1]


INT4_GROUP = 32                          # channels that share a step and a low
# The channels of an octet (8 channels, one 32-bit word) in the order of the word's nibbles: even
# channels in the low half, odd ones in the high half, so that a mask leaves two neighbours as fp16
# mantissas.
INT4_NIBBLES = (0, 2, 4, 6, 1, 3, 5, 7)


def int4_unit_bytes(head_dim: int) -> int:
    """Bytes of one block of one KV head in the 4-bit cache: 16 rows of codes, then 16 rows of (step,
    low) for each group of min(32, head_dim) channels."""
    return 16 * head_dim // 2 + 16 * (head_dim // min(head_dim, INT4_GROUP)) * 4


def int4_head_dim(unit_bytes: int) -> int | None:
    """The head_dim of a 4-bit cache by its units' bytes (None: of no such cache)."""
    return _INT4_DIMS.get(unit_bytes)


_INT4_DIMS = {int4_unit_bytes(d): d for d in (16, 32, 64, 128, 256)}


def int4_quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [..., D] fp32 -> codes [..., G, D / G] uint8, steps and lows [..., G] fp16. low: the group's least
    value in fp16; step: (largest - low) / 15, rounded towards zero to fp16, so that no code stands for
    more than the largest value; code: rint((x - low) / step) within 0 .. 15, 0 where the step is 0."""
    x = x.unflatten(-1, (-1, min(x.shape[-1], INT4_GROUP)))
    lows = x.amin(-1).half() + 0.0                             # (-0 as 0)
    span = (x.amax(-1) - lows.float()).clamp_min(0) + 0.0      # (here too)
    span = span / torch.full_like(span, 15.0)
    steps = span.half()
    steps = (steps.view(torch.int16) - (steps.float() > span).to(torch.int16)).view(torch.float16)
    codes = torch.round((x - lows.float()[..., None]) / steps.float()[..., None]).clamp(0, 15)
    return torch.where(steps[..., None] > 0, codes, 0).to(torch.uint8), steps, lows


def int4_views(cache: torch.Tensor, values: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, steps, lows) of a contiguous cache [..., unit bytes], as views: the codes' bytes
    [..., 16, D / 8, 4] and the numbers [..., 16, G], rows and octets or groups in that order. K's units
    are row-major, the step and low of a group side by side; V's (values) hold the 16 rows of an
    octet together, and of each group and four rows the steps, then the lows."""
    D = int4_head_dim(cache.shape[-1])
    G = D // min(D, INT4_GROUP)
    codes, numbers = cache[..., :8 * D], cache[..., 8 * D:].view(torch.float16)
    if not values:
        numbers = numbers.unflatten(-1, (16, G, 2))
        return codes.unflatten(-1, (16, D // 8, 4)), numbers[..., 0], numbers[..., 1]
    numbers = numbers.unflatten(-1, (G, 4, 2, 4)).movedim(-4, -1)         # [..., 4, 2, 4, G]
    steps, lows = (numbers[..., :, j, :, :] for j in range(2))            # [..., 4, 4, G]
    return codes.unflatten(-1, (D // 8, 16, 4)).transpose(-3, -2), steps, lows


@dataclass(frozen=True)
class Int4KVCache:
    """The 4-bit paged KV cache of every layer: uint8 [L, 2, num_blocks, KVH, bytes], the bytes of a block
    of one KV head holding its 16 rows' codes and, for each row and group of 32 channels, fp16 step
    and low (int4_views); a code stands for fp16(low + code * step). Per token and layer it takes
    KVH * 1.25 D bytes (1.5 D at head_dim 16) where fp16 takes KVH * 4 D."""

    data: torch.Tensor
    layers: tuple = field(init=False, repr=False, compare=False)     # (k_cache, v_cache) of each layer

    def __post_init__(self) -> None:
        object.__setattr__(self, "layers", tuple(tuple(x.unbind()) for x in self.data.unbind()))

    @classmethod
    def new(cls, num_layers: int, num_blocks: int, num_kv_heads: int, head_dim: int,
            device) -> "Int4KVCache":
        if head_dim not in (16, 32, 64, 128, 256):
            raise ValueError(f"4-bit cache: head_dim {head_dim} (16, 32, 64, 128, 256)")
        return cls(torch.zeros(num_layers, 2, num_blocks, num_kv_heads, int4_unit_bytes(head_dim),
                               dtype=torch.uint8, device=device))

    @property
    def device(self) -> torch.device:
        return self.data.device

    def layer(self, index: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(k_cache, v_cache) of one layer, views of data, as the ops take them."""
        return self.layers[index]
