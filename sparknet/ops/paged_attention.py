"""Decode attention over a paged 8-bit KV cache (grouped-query, head_dim 64 or 128).

``paged_decode_attention(q, cache, block_tables, lengths)``: each sequence's newest T
tokens attend to its keys.  ``q`` is ``[B, heads, head_dim]`` (T = 1) or
``[B, T, heads, head_dim]``, bf16 or fp16; ``block_tables`` ``[B, width]`` int32 names the
pages; ``lengths`` ``[B]`` int32 counts the keys, the T new tokens (appended before)
included.  Token t sees the keys ``j <= lengths[b] - T + t``; with ``window`` w > 0, only
the last w of them.

Rows that see no key (an empty or padded sequence, ``lengths[b] < T``) give 0 and a
log-sum-exp of -inf.  Keys behind a sequence's length are never used, whatever their
pages hold.  Lengths beyond the table's width count as its width; a table entry that
names no page of the cache holds no keys.

Scores, softmax statistics and the sum over the values are in fp32; the only roundings
before the last are those of the softmax weights to fp16.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from .kv_cache import Fp8KVCache


def paged_decode_attention(q: torch.Tensor, cache: Fp8KVCache, block_tables: torch.Tensor, lengths: torch.Tensor, *,
                           scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None,
                           return_lse: bool = False):
    """softmax(q k^T * scale) v over the pages of each sequence; ``scale`` defaults to
    ``head_dim ** -0.5``.  Returns out, or ``(out, lse)`` with the natural log-sum-exp
    ``[B, (T,) heads]`` in float32."""
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    out, lse = cache._pool.attention(q, block_tables, lengths, scale, window, out, return_lse)
    return (out, lse) if return_lse else out


__all__ = ["paged_decode_attention"]
