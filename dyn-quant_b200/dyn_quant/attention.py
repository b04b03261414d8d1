"""Attention layer of a decode step on the split GEMV and the 4-bit KV cache.

The projections are DynQuantLinear layers (each token's vector with its own
outlier mask): wq, wk and wv read the same x, so they are stacked into one
[(q_heads + 2 kv_heads) head_dim, d_model] matrix, one call for the three.  The
new keys and values go from that call's output straight into the cache
(Int4KVCache.append reads the slice in place), the queries attend over it, and
wo projects the heads' outputs back.
"""
from __future__ import annotations

from typing import Callable

import torch

from dyn_quant import DynQuantLinear
from dyn_quant.kv_cache import Int4KVCache


class Int4Attention(torch.nn.Module):
    """Grouped-query attention with quantized projections and a 4-bit KV cache.

    load_weights(wq, wk, wv, wo) quantizes the FP16 projections ([q_heads
    head_dim, d_model], [kv_heads head_dim, d_model] twice, [d_model, q_heads
    head_dim]); forward(x, cache) runs one step: x [n_seqs, d_model] (one new
    token per sequence) or [n_seqs, T, d_model]."""

    def __init__(self, d_model: int, n_heads: int, n_kv_heads: int, head_dim: int = 128,
                 outlier_k: float = 3.0) -> None:
        super().__init__()
        if n_heads % n_kv_heads != 0:
            raise RuntimeError(f"n_heads={n_heads} must be a multiple of n_kv_heads={n_kv_heads}")
        self.d_model, self.n_heads, self.n_kv_heads, self.head_dim = d_model, n_heads, n_kv_heads, head_dim
        self.wqkv = DynQuantLinear(d_model, (n_heads + 2 * n_kv_heads) * head_dim, outlier_k)
        self.wo = DynQuantLinear(n_heads * head_dim, d_model, outlier_k)

    def load_weights(self, wq: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, wo: torch.Tensor) -> None:
        q, kv = self.n_heads * self.head_dim, self.n_kv_heads * self.head_dim
        for name, w, shape in (("wq", wq, (q, self.d_model)), ("wk", wk, (kv, self.d_model)),
                               ("wv", wv, (kv, self.d_model)), ("wo", wo, (self.d_model, q))):
            if tuple(w.shape) != shape:
                raise RuntimeError(f"{name} must be {list(shape)}, got {list(w.shape)}")
        self.wqkv.load_weight(torch.cat([wq, wk, wv]).contiguous())
        self.wo.load_weight(wo)

    def forward(self, x: torch.Tensor, cache: Int4KVCache,
                rotate: Callable[[torch.Tensor, torch.Tensor, torch.Tensor], tuple] | None = None,
                counts: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
        """One step over `cache` (which gains the new tokens).

        rotate(q, k, positions) -> (q, k), if given, applies the model's rotary
        embedding: q [n_seqs, T, n_heads, head_dim], k [n_seqs, T, n_kv_heads,
        head_dim] float16, positions int32 [n_seqs, T].  counts: int32 [n_seqs],
        tokens of x that are real (default: all); rows behind them attend to
        nothing.  accumulate: see Int4KVCache.attend."""
        n, t = x.shape[0], (x.shape[1] if x.dim() == 3 else 1)
        if x.shape[-1] != self.d_model or x.dim() not in (2, 3) or n != cache.n_seqs:
            raise RuntimeError(f"x must be [{cache.n_seqs}, {self.d_model}] or [{cache.n_seqs}, T, {self.d_model}], "
                               f"got {tuple(x.shape)}")
        if t == 0:
            return x.to(torch.float16)
        h, g = self.n_heads, self.n_kv_heads
        qkv = self.wqkv(x.reshape(n * t, self.d_model)).view(n, t, h + 2 * g, self.head_dim)
        q, k, v = qkv[:, :, :h], qkv[:, :, h:h + g], qkv[:, :, h + g:]
        if rotate is not None:
            first = cache.lengths + cache.evicted
            q, k = rotate(q, k, first[:, None] + torch.arange(t, dtype=torch.int32, device=x.device))
        cache.append(k, v, counts=counts)
        y = cache.attend(q, counts=counts, accumulate=accumulate)
        return self.wo(y.reshape(n * t, h * self.head_dim)).view(*x.shape[:-1], self.d_model)
