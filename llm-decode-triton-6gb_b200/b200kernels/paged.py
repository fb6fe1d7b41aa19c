"""Paged KV cache: append with the rotation on the way, and attention of the newest tokens over the pages.

No counterpart in the reference, whose cache is one contiguous ``[B, KVH, S, D]`` tensor; next to the
contiguous ``rope_kv_append`` (``glue.py``) and ``decode_attention`` of this package:

* ``PagedKV(k_pages, v_pages)`` -- one layer's pool, ``[num_pages, KVH, page_size, D]`` (any strides with a
  contiguous last dim; a ``[num_pages, page_size, KVH, D]`` pool is passed as ``pool.transpose(1, 2)``).
  Position p of sequence b lies in page ``page_table[b, p // page_size]``, slot ``p % page_size``;
* ``paged_rope_append`` -- (RMS norms of the query and key heads,) rotary embedding, keys and values into
  their pages;
* ``paged_attention`` -- T tokens per sequence (1: plain decode; more: drafts verified at once), causal among
  themselves, with an optional prefix that the whole batch shares, read and multiplied once.

    kv = PagedKV(k_pages, v_pages)
    q_rot = paged_rope_append(kv, q, k, v, positions, page_table, cos, sin)
    out = paged_attention(kv, q_rot.view(B, T, H, D), page_table, seqlens)

Work runs in ``libb200decode.so`` on the tensors' device and torch's current stream there; there is no
fallback. Every call can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib


MAX_PAGE_SIZE = 1024


class PagedKV:
    """One layer's paged cache: a view of the caller's pools (nothing is copied or allocated). Page ids
    outside [0, num_pages) are never followed."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise ValueError(f"k/v pages are [num_pages, KVH, page_size, D], got {tuple(k_pages.shape)} and "
                             f"{tuple(v_pages.shape)}")
        if k_pages.dtype not in (torch.float16, torch.bfloat16) or v_pages.dtype != k_pages.dtype:
            raise TypeError(f"k/v pages are both fp16 or both bf16, got {k_pages.dtype} and {v_pages.dtype}")
        if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
            raise ValueError("the last dimension of the pages must be contiguous")
        if not 1 <= k_pages.shape[2] <= MAX_PAGE_SIZE or k_pages.shape[1] == 0:
            raise ValueError(f"pages hold 1..{MAX_PAGE_SIZE} positions of at least one head, got {tuple(k_pages.shape)}")
        if max(k_pages.shape) >= 2 ** 31:
            raise ValueError(f"too many pages, heads or elements (2^31 or more): {tuple(k_pages.shape)}")
        if v_pages.device != k_pages.device:
            raise ValueError(f"k/v pages are on {k_pages.device} and {v_pages.device}")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k_pages.shape
        self.dtype, self.device = k_pages.dtype, k_pages.device
        self.desc = _lib.PagedKvDesc(k_pages.data_ptr(), *k_pages.stride()[:3], v_pages.data_ptr(),
                                     *v_pages.stride()[:3], self.num_pages, self.page_size, self.kv_heads,
                                     self.head_dim, _lib.dtype_code(self.dtype))
        self._desc = ctypes.addressof(self.desc)
        self._index = self.device.index if self.device.type == "cuda" else -1


def paged_rope_append(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                      page_table: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      q_out: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None,
                      q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                      eps: float = 1e-6, flags: int = 0) -> torch.Tensor:
    """q [N, H, D], k / v [N, KVH, D] (projection outputs; strided views are fine), positions int64 [N],
    page_table int32 [B, pages], cos / sin [S_max, D] in the cache's dtype or fp32 -> q_out [N, H, D] (may be
    q itself, overlaps no other input); the rotated keys and the values are written to their pages. Token i belongs to sequence
    ``seq_ids[i]`` (int32 [N]) or, without them, ``i // (N // B)``. ``q_weight`` / ``k_weight`` [D]: RMS norm
    of every head before the rotation. fp32 between loads and stores, one rounding. A token whose sequence is
    outside [0, B) or whose position is outside [0, S_max) is padding: nothing of it is written. Two tokens
    of a call must not share a slot; pools whose pages, or whose keys and values, are one memory are refused."""
    r = _lib.binding().rope_append(kv._desc, q, k, v, positions, page_table, cos, sin, q_out, seq_ids, q_weight, k_weight,
                                   eps, flags, kv._index)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_paged_rope_append", r)
    return r


def paged_attention(kv: PagedKV, q: torch.Tensor, page_table: torch.Tensor, seqlens: torch.Tensor,
                    scale: float | None = None, prefix_table: torch.Tensor | None = None, prefix_len: int = 0,
                    max_len: int = 0, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    workspace: torch.Tensor | None = None, flags: int = 0) -> torch.Tensor:
    """q [B, T, H, D], page_table int32 [B, pages], seqlens int32 [B] (cached keys, the T new tokens included)
    -> [B, T, H, D] in ``out_dtype`` (q's dtype or torch.float32). Query t of sequence b sees the keys before
    position ``seqlens[b] - T + 1 + t``; one that sees none gives zeros. Lengths past the table's pages (and the prefix)
    are cut to them. ``prefix_table`` int32 [pages] and
    ``prefix_len``: the first ``prefix_len`` positions of every sequence lie in these pages (the entries of
    ``page_table`` for them are not read, and need not be there) and are computed once for the batch -- fast where
    pages hold 8, 16, 32 or a multiple of 64 positions and ``prefix_len`` is a multiple of the page (of 64 for larger
    pages); other sizes are right, but take slower copies for the whole call. ``max_len``: an upper bound of
    ``seqlens`` known to the host, which only guides the split. ``workspace``: contiguous scratch of
    ``paged_attention_workspace`` bytes, 16-byte aligned, not shared by calls that may overlap; without it
    one is allocated per call."""
    r = _lib.binding().attention(kv._desc, q, page_table, seqlens, scale, prefix_table, prefix_len, max_len, out, out_dtype,
                                 workspace, flags, kv._index)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_paged_attention", r)
    return r


def paged_attention_workspace(kv: PagedKV, q: torch.Tensor, page_table: torch.Tensor, prefix_len: int = 0,
                              max_len: int = 0) -> torch.Tensor:
    """Scratch for ``paged_attention`` calls of these sizes (for callers that keep their buffers)."""
    return _lib.binding().attention_workspace(kv._desc, q, page_table, prefix_len, max_len)
