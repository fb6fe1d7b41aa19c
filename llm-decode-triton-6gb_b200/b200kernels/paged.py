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
        if v_pages.device != k_pages.device:
            raise ValueError(f"k/v pages are on {k_pages.device} and {v_pages.device}")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k_pages.shape
        self.dtype, self.device = k_pages.dtype, k_pages.device
        self.desc = _lib.PagedKvDesc(k_pages.data_ptr(), *k_pages.stride()[:3], v_pages.data_ptr(),
                                     *v_pages.stride()[:3], self.num_pages, self.page_size, self.kv_heads,
                                     self.head_dim, _lib.dtype_code(self.dtype))
        self._ref = ctypes.byref(self.desc)


def _table(kv: PagedKV, table: torch.Tensor, name: str, dim: int) -> None:
    if table.dtype != torch.int32 or table.dim() != dim or (table.numel() and table.stride(-1) != 1):
        raise ValueError(f"{name} is int32, {dim}-D, contiguous in its last dimension; got {table.dtype}, "
                         f"{tuple(table.shape)}")


def _same_device(device: torch.device, **tensors) -> int:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    return _lib.cuda_index(device)


def paged_rope_append(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                      page_table: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      q_out: torch.Tensor | None = None, seq_ids: torch.Tensor | None = None,
                      q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                      eps: float = 1e-6, flags: int = 0) -> torch.Tensor:
    """q [N, H, D], k / v [N, KVH, D] (projection outputs; strided views are fine), positions int64 [N],
    page_table int32 [B, pages], cos / sin [S_max, D] in the cache's dtype or fp32 -> q_out [N, H, D] (may be
    q itself); the rotated keys and the values are written to their pages. Token i belongs to sequence
    ``seq_ids[i]`` (int32 [N]) or, without them, ``i // (N // B)``. ``q_weight`` / ``k_weight`` [D]: RMS norm
    of every head before the rotation. fp32 between loads and stores, one rounding. A token whose sequence is
    outside [0, B) or whose position is outside [0, S_max) is padding: nothing of it is written. Two tokens
    of a call must not share a slot."""
    N, H, D = q.shape
    B, per_seq = page_table.shape
    if D != kv.head_dim or k.shape != (N, kv.kv_heads, D) or v.shape != k.shape or H % kv.kv_heads:
        raise ValueError(f"incompatible shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)} for a cache of "
                         f"{kv.kv_heads} heads of {kv.head_dim}")
    if q.dtype != kv.dtype or k.dtype != kv.dtype or v.dtype != kv.dtype:
        raise TypeError(f"q/k/v dtypes {q.dtype}, {k.dtype}, {v.dtype} differ from the cache's {kv.dtype}")
    if positions.dtype != torch.int64 or positions.shape != (N,) or (N > 1 and positions.stride(0) != 1):
        raise ValueError(f"positions is a contiguous int64 [{N}], got {positions.dtype} {tuple(positions.shape)}")
    _table(kv, page_table, "page_table", 2)
    if seq_ids is None:
        if N and (B == 0 or N % B):
            raise ValueError(f"{N} tokens do not divide over {B} sequences: pass seq_ids")
    elif seq_ids.dtype != torch.int32 or seq_ids.shape != (N,) or (N > 1 and seq_ids.stride(0) != 1):
        raise ValueError(f"seq_ids is a contiguous int32 [{N}], got {seq_ids.dtype} {tuple(seq_ids.shape)}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != D or cos.stride() != sin.stride() or cos.stride(1) != 1:
        raise ValueError(f"cos / sin are [S_max, {D}] of one layout, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    if cos.dtype != sin.dtype or cos.dtype not in (kv.dtype, torch.float32):
        raise TypeError(f"cos / sin are {kv.dtype} or torch.float32, got {cos.dtype}, {sin.dtype}")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (D,) or w.dtype != kv.dtype or w.stride(0) != 1):
            raise ValueError(f"q_weight / k_weight are contiguous [{D}] of {kv.dtype}, got {w.dtype} {tuple(w.shape)}")
    if q_out is None:
        q_out = torch.empty((N, H, D), device=q.device, dtype=q.dtype)
    elif q_out.shape != q.shape or q_out.dtype != q.dtype:
        raise ValueError(f"q_out is {tuple(q.shape)} of {q.dtype}, got {tuple(q_out.shape)} of {q_out.dtype}")
    if D and (q.stride(2) != 1 or k.stride(2) != 1 or v.stride(2) != 1 or q_out.stride(2) != 1):
        raise ValueError("the last dimension of q, k, v and q_out must be contiguous")
    index = _same_device(kv.device, q=q, k=k, v=v, positions=positions, page_table=page_table, cos=cos, sin=sin,
                         q_out=q_out, seq_ids=seq_ids, q_weight=q_weight, k_weight=k_weight)
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), q_out.stride()
    _lib.call_on(index, "b2d_paged_rope_append", kv._ref, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1],
                 v.data_ptr(), vs[0], vs[1], positions.data_ptr(), _lib.ptr(seq_ids), page_table.data_ptr(),
                 page_table.stride(0), per_seq, B, cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0],
                 _lib.dtype_code(cos.dtype), _lib.ptr(q_weight), _lib.ptr(k_weight), eps, q_out.data_ptr(), os[0],
                 os[1], N, H, flags)
    return q_out


def paged_attention(kv: PagedKV, q: torch.Tensor, page_table: torch.Tensor, seqlens: torch.Tensor,
                    scale: float | None = None, prefix_table: torch.Tensor | None = None, prefix_len: int = 0,
                    max_len: int = 0, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    workspace: torch.Tensor | None = None, flags: int = 0) -> torch.Tensor:
    """q [B, T, H, D], page_table int32 [B, pages], seqlens int32 [B] (cached keys, the T new tokens included)
    -> [B, T, H, D] in ``out_dtype`` (q's dtype or torch.float32). Query t of sequence b sees the keys before
    position ``seqlens[b] - T + 1 + t``; one that sees none gives zeros. ``prefix_table`` int32 [pages] and
    ``prefix_len``: the first ``prefix_len`` positions of every sequence lie in these pages (the entries of
    ``page_table`` for them are not read) and are computed once for the batch. ``max_len``: an upper bound of
    ``seqlens`` known to the host, which only guides the split. ``workspace``: uint8 scratch of
    ``paged_attention_workspace`` bytes, 16-byte aligned, not shared by calls that may overlap; without it
    one is allocated per call."""
    B, T, H, D = q.shape
    if D != kv.head_dim or H % kv.kv_heads or page_table.shape[0] != B:
        raise ValueError(f"incompatible shapes q{tuple(q.shape)} page_table{tuple(page_table.shape)} for a cache of "
                         f"{kv.kv_heads} heads of {kv.head_dim}")
    if q.dtype != kv.dtype:
        raise TypeError(f"q is {q.dtype}, the cache {kv.dtype}")
    _table(kv, page_table, "page_table", 2)
    if seqlens.dtype != torch.int32 or seqlens.shape != (B,) or (B > 1 and seqlens.stride(0) != 1):
        raise ValueError(f"seqlens is a contiguous int32 [{B}], got {seqlens.dtype} {tuple(seqlens.shape)}")
    if prefix_len:
        if prefix_table is None:
            raise ValueError("prefix_len without prefix_table")
        _table(kv, prefix_table, "prefix_table", 1)
        if prefix_len < 0 or prefix_len > prefix_table.shape[0] * kv.page_size:
            raise ValueError(f"prefix_len {prefix_len} is outside the {prefix_table.shape[0]} pages of prefix_table")
    if out is None:
        out = torch.empty((B, T, H, D), device=q.device, dtype=out_dtype or q.dtype)
    elif out.shape != q.shape or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out is {tuple(q.shape)} of {out_dtype or q.dtype}, got {tuple(out.shape)} of {out.dtype}")
    if D and (q.stride(3) != 1 or out.stride(3) != 1):
        raise ValueError("the last dimension of q and out must be contiguous")
    index = _same_device(kv.device, q=q, page_table=page_table, seqlens=seqlens, out=out,
                         prefix_table=prefix_table if prefix_len else None, workspace=workspace)
    per_seq = page_table.shape[1]
    if workspace is None:
        nbytes = _workspace_bytes(kv, index, B, T, H, per_seq, prefix_len, max_len)
        if nbytes:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    qs, os = q.stride(), out.stride()
    _lib.call_on(index, "b2d_paged_attention", kv._ref, q.data_ptr(), qs[0], qs[1], qs[2], page_table.data_ptr(),
                 page_table.stride(0), per_seq, seqlens.data_ptr(), prefix_table.data_ptr() if prefix_len else None,
                 prefix_len, max_len, B, T, H, D ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1],
                 os[2], _lib.dtype_code(out.dtype), None if workspace is None else workspace.data_ptr(),
                 0 if workspace is None else workspace.numel(), flags)
    return out


def _workspace_bytes(kv, index, B, T, H, per_seq, prefix_len, max_len) -> int:
    with _lib.on_device(index):
        return _lib.load().b2d_paged_attention_workspace_bytes(kv._ref, B, T, H, per_seq, prefix_len, max_len)


def paged_attention_workspace(kv: PagedKV, q: torch.Tensor, page_table: torch.Tensor, prefix_len: int = 0,
                              max_len: int = 0) -> torch.Tensor:
    """Scratch for ``paged_attention`` calls of these sizes (for callers that keep their buffers)."""
    nbytes = _workspace_bytes(kv, _lib.cuda_index(kv.device), *q.shape[:3], page_table.shape[1], prefix_len, max_len)
    return torch.empty(nbytes, dtype=torch.uint8, device=kv.device)
