"""The attention block of a quantised model: projection of queries, keys and values with int4 weights, storing into the paged 8-bit
cache with the position rotation, attention over the cache, output projection (no counterpart in the reference).

    block = CachedAttention(W4A16Linear.from_float(w_qkv), W4A16Linear.from_float(w_out), heads, kv_heads, *rotation(positions, head_dim))
    cache = PagedKVCache(pages, kv_heads, head_dim)
    y = block(x, cache, block_table, lengths)      # x: the new tokens' hidden states, one row each

Four launches for a decode step (one more where sequences are cut into parts, and for each projection whose K is summed in runs), all on the current
stream, none that looks at a length on the host: a step may be captured into a HIP graph and replayed with other contents of ``x``, ``block_table`` and ``lengths``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import QuadmulError
from .kv_cache import PagedKVCache
from .linear import W4A16Linear


def rotation(positions: int, pairs_times_two: int, base: float = 10000.0, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin of ``position / base^(2 i / d)`` for ``d = pairs_times_two`` elements, ``[positions, d / 2]`` float32, worked out in 64 bits."""
    inverse = base ** (-torch.arange(0, pairs_times_two, 2, device=device, dtype=torch.float64) / pairs_times_two)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


class CachedAttention(torch.nn.Module):
    """``qkv`` projects to ``heads`` queries, then ``kv_heads`` keys, then as many values, each ``head_dim`` wide; ``out`` takes the heads' outputs side by side.
    ``cos`` and ``sin`` as :func:`quadmul_amd.kv_cache.append` takes them, or None."""

    def __init__(self, qkv: W4A16Linear, out: W4A16Linear, heads: int, kv_heads: int, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                 interleaved: bool = False, scale: Optional[float] = None, window: int = 0):
        super().__init__()
        if heads < 1 or kv_heads < 1 or heads % kv_heads or qkv.out_features % (heads + 2 * kv_heads):
            raise QuadmulError("CachedAttention: heads must be a multiple of kv_heads, and qkv's outputs one of heads + 2 kv_heads")
        if (cos is None) != (sin is None):
            raise QuadmulError("CachedAttention: cos and sin go together")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, qkv.out_features // (heads + 2 * kv_heads)
        if out.in_features != heads * self.head_dim:
            raise QuadmulError(f"CachedAttention: out must take {heads * self.head_dim} features")
        self.qkv, self.out = qkv, out
        self.interleaved, self.scale, self.window = interleaved, scale, window
        self.register_buffer("cos", cos)
        self.register_buffer("sin", sin)

    def forward(self, x: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, lengths: torch.Tensor, query_start: Optional[torch.Tensor] = None,
                max_query: int = 0, max_length: int = 0) -> torch.Tensor:
        """``x`` [tokens, hidden]: the new tokens of every sequence, packed; ``lengths`` counts them in. The other arguments are those of
        :func:`quadmul_amd.kv_cache.append` and :func:`quadmul_amd.kv_cache.attend`."""
        wide, narrow = self.heads * self.head_dim, self.kv_heads * self.head_dim
        q, k, v = self.qkv(x).split((wide, narrow, narrow), dim=1)
        q, k, v = (t.unflatten(1, (-1, self.head_dim)) for t in (q, k, v))
        if self.cos is None:
            cache.append(k, v, block_table, lengths, query_start, max_query=max_query)
        else:
            q = cache.append(k, v, block_table, lengths, query_start, q=q, cos=self.cos, sin=self.sin, interleaved=self.interleaved, max_query=max_query)
        o = cache.attend(q, block_table, lengths, query_start, scale=self.scale, window=self.window, max_query=max_query, max_length=max_length)
        return self.out(o.flatten(1))
