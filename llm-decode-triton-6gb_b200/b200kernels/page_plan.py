"""Page tables kept on the GPU: which page every new token of a step goes to, from the requests' lengths alone.

No counterpart in the reference, whose cache is one contiguous tensor; next to the paged caches of this package (``paged.py``,
``paged_int4.py``), whose appends and attention take ``page_table``, ``positions``, ``seq_ids`` and ``seqlens`` as they come
out of here. Nothing goes through the host, so that a whole step -- plan, appends, attention, draft verification -- is one CUDA graph:

    tables = PageTables.empty(num_pages, page_size, batch, pages_per_seq, "cuda")
    plan = tables.step(cached, new, max_tokens)        # int32 [batch]: tokens cached, tokens of this step
    q_rot = paged_rope_append(kv, q, k, v, plan.positions, tables.page_table, cos, sin, seq_ids=plan.seq_ids)
    ... paged_attention(kv, q_rot.view(B, T, H, D), tables.page_table, plan.seqlens)

The last line is right where every sequence was granted T tokens. Tokens lie one sequence's behind another's: with other numbers of
new tokens, or a sequence that is refused, the queries are gathered by ``starts``, and a refused sequence, whose ``seqlens`` stays
``cached``, is given no keys, or it would attend with another's queries (its row of the output is then zeros):

    rows = (plan.starts[:-1, None] + torch.arange(T, device="cuda")).clamp(max=max_tokens - 1).view(-1)   # [B T]
    lens = torch.where(plan.granted > 0, plan.seqlens, 0)
    ... paged_attention(kv, q_rot[rows].view(B, T, H, D), tables.page_table, lens)       # T new tokens, or none

A request that ends, or whose drafts were refused, gives its pages back by the next step's lengths (0 and 0: all of them).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_BATCH = 8192


class StepPlan(NamedTuple):
    """A step's tokens, one sequence's behind another's; rows past the last token are -1 (padding for the appends)."""
    positions: torch.Tensor   # int64 [max_tokens]
    seq_ids: torch.Tensor     # int32 [max_tokens]
    slots: torch.Tensor       # int64 [max_tokens]: page * page_size + offset
    seqlens: torch.Tensor     # int32 [B]: cached + new, or cached where the sequence is refused (none of the step's queries are its own)
    starts: torch.Tensor      # int32 [B + 1]: its tokens are [starts[b], starts[b + 1])
    granted: torch.Tensor     # int32 [B]: new, or -1 where refused

    @classmethod
    def empty(cls, batch: int, max_tokens: int, device) -> "StepPlan":
        new = lambda n, t: torch.empty(n, dtype=t, device=device)  # noqa: E731
        return cls(new(max_tokens, torch.int64), new(max_tokens, torch.int32), new(max_tokens, torch.int64),
                   new(batch, torch.int32), new(batch + 1, torch.int32), new(batch, torch.int32))


class PageTables:
    """The page tables of a batch and the pages that nobody holds, all int32 on one device and changed in place:
    ``page_table`` [B, pages_per_seq]; ``held`` [B], the pages of each sequence (the table's entries before it);
    ``free`` [num_pages], a ring of free pages; ``ring`` [2], the index of its first one and their number."""

    def __init__(self, page_table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, ring: torch.Tensor, page_size: int):
        if not 1 <= page_size <= 1024:
            raise ValueError(f"pages hold 1..1024 positions, got {page_size}")
        if page_table.dim() != 2 or page_table.shape[0] > MAX_BATCH:
            raise ValueError(f"page_table is [B, pages] of at most {MAX_BATCH} sequences, got {tuple(page_table.shape)}")
        self.page_table, self.held, self.free, self.ring, self.page_size = page_table, held, free, ring, page_size

    @classmethod
    def empty(cls, num_pages: int, page_size: int, batch: int, pages_per_seq: int, device) -> "PageTables":
        """Nobody holds a page; all of them are free."""
        return cls(torch.full((batch, pages_per_seq), -1, dtype=torch.int32, device=device),
                   torch.zeros(batch, dtype=torch.int32, device=device),
                   torch.arange(num_pages, dtype=torch.int32, device=device),
                   torch.tensor([0, num_pages], dtype=torch.int32, device=device), page_size)

    def step(self, cached: torch.Tensor, new: torch.Tensor, max_tokens: int | None = None, out: StepPlan | None = None,
             flags: int = 0) -> StepPlan:
        """cached, new int32 [B] (negative counts as 0) -> the plan of the step's tokens, in ``out`` or new tensors of
        ``max_tokens`` rows. Every sequence then holds ceil((cached + new) / page_size) pages: missing ones are taken from the
        ring's front in the sequences' order, surplus ones put behind its end (their entries become -1). A sequence
        whose pages or tokens do not fit -- the table's row, the free pages or the ``max_tokens`` left behind the sequences before
        it, refused ones counted -- keeps its state and gets no token: ``granted`` is -1 there. Calls on the same tables must not overlap."""
        if out is None:
            if max_tokens is None:
                raise ValueError("max_tokens or out is needed")
            out = StepPlan.empty(self.page_table.shape[0], max_tokens, self.page_table.device)
        elif max_tokens is not None and max_tokens != out.positions.shape[0]:
            raise ValueError(f"out holds {out.positions.shape[0]} tokens, not {max_tokens}")
        r = _lib.binding().page_plan(self.page_table, self.held, self.free, self.ring, self.page_size, cached, new, *out, flags)
        if r != _lib.B2D_OK:
            raise _lib.B2DError("b2d_page_plan", r)
        return out
