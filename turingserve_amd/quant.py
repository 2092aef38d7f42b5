"""The W8A16 weight format: per-output-row symmetric int8 with an fp32 scale.

Restates quant/int8.py:8-16 and the LinearWeight container of model/layers.py:21-31. The GEMM
also accepts fp16 scales (the W8A16 benchmark configuration draws them in fp16; widening fp16
to fp32 is exact).
"""

from __future__ import annotations

from dataclasses import dataclass

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
