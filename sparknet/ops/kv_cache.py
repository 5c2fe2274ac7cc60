"""Paged KV cache in 8 bits: pages of e4m3 codes with one scale for each (page, KV head).

    cache = Fp8KVCache(num_pages, kv_heads, page_size=64, head_dim=128, device="cuda")
    kv_append(cache, k, v, slots)          # k, v [n, kv_heads, head_dim] bf16 / fp16
    k, v = kv_read(cache, slots)           # back, exactly code * scale

``cache.k`` / ``cache.v`` are ``[num_pages, kv_heads, page_size, head_dim]``
``float8_e4m3fn``, ``cache.k_scale`` / ``cache.v_scale`` ``[num_pages, kv_heads]`` float32;
a value is ``code * scale``.  A token's *slot* is ``page * page_size + place in the page``
(:func:`sparknet.ops.plan_pages` makes them).

Scales are powers of two, the smallest (from 2^-100 up) that brings a block's largest
finite magnitude to at most 448.  While a page fills, its scale only grows; codes already
there are then rewritten as ``RN(code * old / new)``, which is exact except for values
below 2^-6 of the new scale.  A run of rows that begins at place 0 starts its page, and
its scale, afresh.  Infinities are stored as the largest value, NaN as NaN.

The rows that one call adds to a page must be consecutive rows with consecutive slots, as
the tokens of a sequence are: each run of rows is one block's work, and two runs for one
page would race for its scale.  ``plan_pages`` makes no others; ``check=True`` reads
hand-made slots back first and raises ``ValueError`` for such a call (it synchronises).
Rows with a slot below 0 or outside the pool are skipped by the append and read as zeros.

Calls run on the current stream of the cache's device and order like any other kernel:
a caller that appends on one stream and attends on another synchronises the two.  They
allocate nothing but what they return, and can be captured into CUDA graphs.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native

PAGE_SIZES = (16, 32, 64, 128)


class Fp8KVCache:
    """A pool of e4m3 pages for one layer's keys and values."""

    def __init__(self, num_pages: int, kv_heads: int, *, page_size: int = 64, head_dim: int = 128, device="cuda"):
        device = torch.device(device)
        shape = (int(num_pages), int(kv_heads), int(page_size), int(head_dim))
        k, v = (torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        ks, vs = (torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        self._adopt(k, v, ks, vs)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor) -> "Fp8KVCache":
        """A cache over existing tensors (not copied).  Scales must be positive."""
        cache = cls.__new__(cls)
        cache._adopt(k, v, k_scale, v_scale)
        return cache

    def _adopt(self, k, v, k_scale, v_scale):
        self._pool = _native.load().KvPool(k, v, k_scale, v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.device = k.device

    def nbytes(self) -> int:
        """Bytes of the codes and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))

    def attention_launches(self, sequences: int, heads: int, width: int, tokens: int = 1) -> int:
        """Kernels that ``paged_decode_attention`` launches for these shapes: 1 or 2."""
        return self._pool.attention_launches(sequences, tokens, heads, width)

    def check(self) -> None:
        """Synchronise and raise if an attention kernel over this cache gave up on a load."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        code = int(self._pool.err.item())
        if code:
            self._pool.err.zero_()
            raise RuntimeError(f"paged_decode_attention failed: error {code} (an mbarrier wait timed out)")


def _check_slots(cache: Fp8KVCache, slots: torch.Tensor) -> None:
    """Raise if two separate runs of ``slots`` fall into one page."""
    s = slots.long().cpu()
    real = (s >= 0) & (s < cache.num_pages * cache.page_size)
    begins = real.clone()
    begins[1:] &= ~(real[:-1] & (s[1:] == s[:-1] + 1) & (s[1:] % cache.page_size != 0))
    pages = s[begins] // cache.page_size
    if pages.unique().numel() != pages.numel():
        raise ValueError("slots hold two separate runs of rows for one page")


def kv_append(cache: Fp8KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
              check: bool = False) -> None:
    """Write rows ``k``, ``v`` ``[n, kv_heads, head_dim]`` (bf16 or fp16, rows contiguous, other
    strides multiples of 8 elements) to ``slots`` ``[n]`` (int32)."""
    if check:
        _check_slots(cache, slots)
    cache._pool.append(k, v, slots)


def rope_kv_append(cache: Fp8KVCache, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                   positions: torch.Tensor, slots: torch.Tensor, q_out: Optional[torch.Tensor] = None, *,
                   check: bool = False) -> torch.Tensor:
    """Split a fused projection ``qkv`` ``[n, (heads + 2 kv_heads) * head_dim]`` (q heads, k
    heads, v heads), rotate q and k, append k and v, and return the rotated q
    ``[n, heads, head_dim]``.

    ``cos`` / ``sin`` are ``[positions, head_dim / 2]`` float32 (rotate-half form) and
    ``positions`` ``[n]`` int32 their rows (clamped into the tables).  The rotation is in
    fp32; q is rounded once to ``qkv``'s type, k once to its code.  q is rotated for skipped
    rows too."""
    if check:
        _check_slots(cache, slots)
    return cache._pool.rope_append(qkv, cos, sin, positions, slots, q_out)


def kv_read(cache: Fp8KVCache, slots: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16,
            k_out: Optional[torch.Tensor] = None,
            v_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[n, kv_heads, head_dim]`` of ``slots`` ``[n]`` (int32, any order, repeats
    allowed) as bfloat16, float16 or float32.  Exact in bfloat16 and float32."""
    return cache._pool.read(slots, dtype, k_out, v_out)


__all__ = ["Fp8KVCache", "PAGE_SIZES", "kv_append", "kv_read", "rope_kv_append"]
