"""Pages of a paged KV cache, planned on the GPU from the requests' lengths.

:func:`plan_pages` turns ``lengths`` (tokens held) and ``new_tokens`` into the step's block
tables, slots and positions in one launch, without the host reading a length: it can
be captured into a CUDA graph with the step.  :class:`PageTable` keeps the state and
updates it in place.

Token rows are packed: request r's ``new_tokens[r]`` rows begin at ``starts[r]``.  Free
pages are a stack ``free_pages[:free_count]``.  The pages of ``finished`` requests go
back first, in request order; a finished request counts as empty and may bring new
tokens.  New pages are then popped in request order.  A request is granted its tokens
if it needs no page, or if the pages that the requests up to and including it need are
there; one that would pass its table's width, or ``max_tokens``, is refused and does not
count.  A refused request keeps its length, and its rows have slot -1, as have rows behind
the last.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _native


class PagePlan(NamedTuple):
    """What a step needs to know about its pages (int32, on the GPU)."""

    slots: torch.Tensor        # [max_tokens] slot of each token row, -1: none
    positions: torch.Tensor    # [max_tokens] position of each token row in its sequence, 0 behind the last
    starts: torch.Tensor       # [requests + 1] first token row of each request
    lengths: torch.Tensor      # [requests] tokens held after the step
    granted: torch.Tensor      # [requests] new tokens that got slots: new_tokens or 0
    free_count: torch.Tensor   # [1] pages free after the step


def plan_pages(lengths: torch.Tensor, new_tokens: torch.Tensor, block_tables: torch.Tensor,
               free_pages: torch.Tensor, free_count: torch.Tensor, *, page_size: int, max_tokens: int,
               finished: Optional[torch.Tensor] = None, lengths_out: Optional[torch.Tensor] = None,
               free_count_out: Optional[torch.Tensor] = None) -> PagePlan:
    """Plan one step for up to 4096 requests.

    ``lengths``, ``new_tokens`` ``[requests]`` int32 (negative counts as 0); ``block_tables``
    ``[requests, width]`` int32, new entries written in place; ``free_pages`` int32, the
    stack, with room for every page of the pool (pushes past its end are dropped);
    ``free_count`` ``[1]`` int32; ``finished`` ``[requests]`` bool or None.  ``lengths_out``
    may be ``lengths`` and ``free_count_out`` may be ``free_count``."""
    return PagePlan(*_native.load().plan_pages(lengths, new_tokens, block_tables, free_pages, free_count,
                                               page_size, max_tokens, finished, lengths_out, free_count_out))


class PageTable:
    """Block tables, lengths and the free list of one page pool.

    One table serves every layer's cache of the same page size: a page number means the
    same tokens in each."""

    def __init__(self, num_pages: int, *, page_size: int, max_requests: int, max_pages: int, device="cuda"):
        if num_pages < 1 or max_requests < 1 or max_pages < 1:
            raise ValueError("num_pages, max_requests and max_pages must be at least 1")
        i32 = {"dtype": torch.int32, "device": torch.device(device)}
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.block_tables = torch.zeros((max_requests, max_pages), **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)

    def extend(self, new_tokens: torch.Tensor, max_tokens: int,
               finished: Optional[torch.Tensor] = None) -> PagePlan:
        """Free the finished requests' pages, take pages for the new tokens, and update the
        tables, lengths and free list in place.  ``plan.lengths`` is ``self.lengths``."""
        return plan_pages(self.lengths, new_tokens, self.block_tables, self.free_pages, self.free_count,
                          page_size=self.page_size, max_tokens=max_tokens, finished=finished,
                          lengths_out=self.lengths, free_count_out=self.free_count)


__all__ = ["PagePlan", "PageTable", "plan_pages"]
