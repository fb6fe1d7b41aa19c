"""Paged KV cache in 4 bits: append with rotation and quantisation on the way, reads, and attention over the codes.

No counterpart in the reference, which holds 4-bit weights but a 16-bit cache; next to ``PagedKV``, ``paged_rope_append`` and
``paged_attention`` (``paged.py``), with the same page tables (``page_plan.PageTables`` keeps them on the GPU):

* ``PagedKVInt4.empty(num_pages, KVH, page_size, D, dtype, device)`` -- one layer's pool. Per position, head and run of
  ``group_size`` elements x: m = round16(min x), s = round16((max x - m) * (1 / 15)), codes rint((x - m) / s) in 0..15; the entry
  stands for m + s c. 4.5 (group 64) or 5 (group 32) bits an element of D = 128 against 16;
* ``paged_int4_append`` -- (RMS norms of the query and key heads,) rotary embedding in either pair layout, of all or the
  first part of a head, keys and values quantised into their pages;
* ``paged_int4_attention`` -- T tokens per sequence, causal among themselves, as ``paged_attention``;
* ``paged_int4_read`` -- the values of cached positions in 16 or 32 bits (the next chunk of a prompt, a move to another cache);
* ``rotary_tables`` -- cos and sin of the usual scalings for long contexts.

    kv = PagedKVInt4.empty(num_pages, KVH, 16, D, torch.bfloat16, "cuda")
    cos, sin = rotary_tables(max_len, D, theta, scaling=config.rope_scaling, device="cuda")
    q_rot = paged_int4_append(kv, q, k, v, positions, page_table, cos, sin)
    out = paged_int4_attention(kv, q_rot.view(B, T, H, D), page_table, seqlens)

Work runs in ``libb200decode.so`` on the tensors' device and torch's current stream there; there is no fallback. Every call
can be captured in a CUDA graph. Inference only: no gradients.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

TILE = 16   # positions of a tile: a page is a whole number of them
MAX_PAGE_SIZE = 1024


class PagedKVInt4:
    """One layer's pool: a view of the caller's uint8 ``pages`` [num_pages, KVH, page bytes] (any strides with a contiguous
    last dimension; nothing is copied). ``dtype`` is that of the model's activations and of the scales. The order of the
    bytes inside a page is the library's own. Page ids outside [0, num_pages) are never followed."""

    def __init__(self, pages: torch.Tensor, page_size: int, head_dim: int, dtype: torch.dtype, group_size: int = 64):
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"dtype is fp16 or bf16, got {dtype}")
        if pages.dtype != torch.uint8:
            raise TypeError(f"pages are uint8, got {pages.dtype}")
        block = self.page_bytes(page_size, head_dim, group_size)
        if pages.dim() != 3 or pages.shape[2] != block:
            raise ValueError(f"pages are [num_pages, KVH, {block}], got {tuple(pages.shape)}")
        if pages.stride(2) != 1:
            raise ValueError("the last dimension of the pages must be contiguous")
        if pages.shape[1] == 0 or max(pages.shape[:2]) >= 2 ** 31:
            raise ValueError(f"no heads, or 2^31 or more pages or heads: {tuple(pages.shape)}")
        self.pages, self.page_size, self.head_dim, self.group_size, self.dtype = pages, page_size, head_dim, group_size, dtype
        self.num_pages, self.kv_heads = pages.shape[:2]
        self.device, self._block = pages.device, block
        self.desc = _lib.Int4KvDesc(pages.data_ptr(), pages.stride(0), pages.stride(1), self.num_pages, page_size,
                                    self.kv_heads, head_dim, group_size, _lib.dtype_code(dtype))
        self._desc = ctypes.addressof(self.desc)
        self._index = self.device.index if self.device.type == "cuda" else -1

    @staticmethod
    def page_bytes(page_size: int, head_dim: int, group_size: int = 64) -> int:
        """Bytes of one page of one head (keys and values)."""
        if head_dim not in (64, 128) or group_size not in (32, 64):
            raise ValueError(f"heads of 64 or 128 in groups of 32 or 64, got {head_dim} and {group_size}")
        if page_size % TILE or not TILE <= page_size <= MAX_PAGE_SIZE:
            raise ValueError(f"pages hold a multiple of {TILE} positions up to {MAX_PAGE_SIZE}, got {page_size}")
        return page_size * (head_dim + 8 * (head_dim // group_size))

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype, device,
              group_size: int = 64) -> "PagedKVInt4":
        """A new pool; its contents are those of zeros."""
        block = cls.page_bytes(page_size, head_dim, group_size)
        return cls(torch.zeros(num_pages, kv_heads, block, dtype=torch.uint8, device=device), page_size, head_dim, dtype,
                   group_size)


def rotary_tables(max_len: int, rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, device="cpu",
                  dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin [max_len, rotary_dim / 2] for ``paged_int4_append``: angles position * theta^(-2 i / rotary_dim), formed in
    64 bits. ``scaling``: a model's ``rope_scaling`` of type "linear", "llama3" or "yarn" (with its keys ``factor``,
    ``original_max_position_embeddings``, ...), whose frequencies and attention factor go into the tables."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim is even, got {rotary_dim}")
    freq = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    gain = 1.0
    kind = (scaling or {}).get("rope_type", (scaling or {}).get("type", "default"))
    if kind == "linear":
        freq = freq / scaling["factor"]
    elif kind == "llama3":
        # long wavelengths are stretched by the factor, short ones stay, those between are blended
        turns = scaling["original_max_position_embeddings"] * freq / (2 * math.pi)
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = keep * freq + (1 - keep) * freq / scaling["factor"]
    elif kind == "yarn":
        # by the number of turns within the original length: beta_fast and more stay, beta_slow and fewer are stretched
        factor, original = scaling["factor"], scaling["original_max_position_embeddings"]

        def index(turns):   # the (fractional) pair that makes so many turns
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = index(scaling.get("beta_fast") or 32), index(scaling.get("beta_slow") or 1)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        stretch = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = (1 - stretch) * freq + stretch * freq / factor

        def strength(weight):
            return 0.1 * weight * math.log(factor) + 1.0 if factor > 1 else 1.0

        gain = scaling.get("attention_factor")
        if gain is None:
            m, every = scaling.get("mscale"), scaling.get("mscale_all_dim")
            gain = strength(m) / strength(every) if m and every else strength(1)
    elif kind != "default":
        raise ValueError(f"scaling of type {kind!r} is not one of default, linear, llama3, yarn")
    angle = torch.arange(max_len, dtype=torch.float64)[:, None] * freq
    return (gain * angle.cos()).to(device, dtype), (gain * angle.sin()).to(device, dtype)


def paged_int4_append(kv: PagedKVInt4, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                      page_table: torch.Tensor, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                      interleaved: bool = False, q_out: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None,
                      q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                      flags: int = 0) -> torch.Tensor | None:
    """q [N, H, D], k / v [N, KVH, D] (projection outputs; strided views are fine), positions int64 [N], page_table int32
    [B, pages] -> q_out [N, H, D] (may be q itself, overlaps no other input); the rotated keys and the values are quantised
    into their pages. cos / sin [S_max, R / 2] in the cache's dtype or fp32 turn the first R elements of a head (R a multiple of
    16): pairs (d, d + R / 2), or neighbours with ``interleaved``; without them nothing is turned. q may be None: keys and values
    alone (another cache's contents). Token i belongs to sequence ``seq_ids[i]`` (int32 [N]) or, without them, ``i // (N // B)``.
    ``q_weight`` / ``k_weight`` [D]: RMS norm of every head before the rotation. A token whose sequence is outside [0, B) or
    whose position is negative or outside [0, S_max) is padding: nothing of it is written; one whose position is outside the
    page table, or whose page is outside the pool, gets its q_out only. Two tokens of a call must not share a slot. A run of
    keys or values with an infinity or a NaN is cached as NaN."""
    r = _lib.binding().int4_append(kv._desc, q, k, v, positions, page_table, cos, sin, interleaved, q_out, seq_ids, q_weight,
                                   k_weight, eps, flags, kv._index, kv._block)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_int4_append", r)
    return r


def paged_int4_read(kv: PagedKVInt4, positions: torch.Tensor, page_table: torch.Tensor, seq_ids: torch.Tensor | None = None,
                    k_out: torch.Tensor | bool | None = None, v_out: torch.Tensor | bool | None = None,
                    out_dtype: torch.dtype | None = None, flags: int = 0) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """What the cache holds at N positions, addressed as by ``paged_int4_append`` -> (k, v) [N, KVH, D] in ``out_dtype`` (the
    cache's dtype or torch.float32; that of given outputs). ``k_out`` / ``v_out``: where to write (they share no
    element), False: leave it out. Rows of padding (a sequence outside [0, B), a position outside the page table) are left as they were; a page id outside the pool
    gives zeros."""
    r = _lib.binding().int4_read(kv._desc, positions, page_table, seq_ids, k_out, v_out, out_dtype, flags, kv._index)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_int4_read", r)
    return r


def paged_int4_attention(kv: PagedKVInt4, q: torch.Tensor, page_table: torch.Tensor, seqlens: torch.Tensor,
                         scale: float | None = None, max_len: int = 0, out: torch.Tensor | None = None,
                         out_dtype: torch.dtype | None = None, workspace: torch.Tensor | None = None,
                         flags: int = 0) -> torch.Tensor:
    """q [B, T, H, D], page_table int32 [B, pages], seqlens int32 [B] (cached keys, the T new tokens included) ->
    [B, T, H, D] in ``out_dtype`` (q's dtype or torch.float32). Query t of sequence b sees the keys before position
    ``seqlens[b] - T + 1 + t``; one that sees none gives zeros. Lengths past the table's pages are cut to them. T and H / KVH up to 16.
    ``max_len``: an upper bound of ``seqlens`` known to the host, which only guides the split. ``out`` may be q itself and
    overlaps no other input. ``workspace``: contiguous scratch of ``paged_int4_attention_workspace`` bytes, 16-byte
    aligned, not shared by calls that may overlap; without it one is allocated per call. A weight times its value's s is
    rounded to fp16: by 2^-11, or by 2^-30 of the row's largest such term where it is below 2^-19 of that. bf16 only: values whose s is
    2^111 or more, queries of 2^114 or more and scores of 2^126 or more may give infinities, NaN or zeros though the exact result is finite."""
    r = _lib.binding().int4_attention(kv._desc, q, page_table, seqlens, scale, max_len, out, out_dtype, workspace, flags,
                                      kv._index)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_int4_attention", r)
    return r


def paged_int4_attention_workspace(kv: PagedKVInt4, q: torch.Tensor, page_table: torch.Tensor, max_len: int = 0) -> torch.Tensor:
    """Scratch for ``paged_int4_attention`` calls of these sizes (for callers that keep their buffers); empty where none is needed.
    Sizes that the call refuses are refused here."""
    r = _lib.binding().int4_workspace(kv._desc, q, page_table, max_len)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_int4_attention", r)
    return r
