"""float64 definitions of the paged-cache and draft-verification operators.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``): the product never imports this. The reference has no
paged cache and no speculative decoding; the attention formula is its stock one (``gqa_decode_ref``: fp32 SDPA
on repeated KV heads, ``profiling/kernels/bench_attention.py:40-41``) with a causal limit per query.
"""
from __future__ import annotations

import numpy as np


def gather_keys(pages, table, n):
    """pages [num_pages, KVH, page_size, D], table [pages] -> the first n positions, [KVH, n, D]. A page id
    outside the pool reads as zeros."""
    ps = pages.shape[2]
    out = np.zeros((pages.shape[1], n, pages.shape[3]))
    for p in range(n):
        page = int(table[p // ps])
        if 0 <= page < pages.shape[0]:
            out[:, p] = pages[page, :, p % ps]
    return out


def paged_attention_ref(q, k_pages, v_pages, page_table, seqlens, scale, prefix_table=None, prefix_len=0):
    """q [B, T, H, D], pages [num_pages, KVH, page_size, D], float64 -> (out [B, T, H, D], mass, reach):
    ``mass`` = sum_j p_j |v_j| / sum_j p_j per element and ``reach`` = max_j scale sum_d |q_d k_jd| per
    (b, t, h), from which the tests derive rounding bounds."""
    q = np.asarray(q, np.float64)
    B, T, H, D = q.shape
    KVH, ps = k_pages.shape[1], k_pages.shape[2]
    G = H // KVH
    out, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, T, H))
    for b in range(B):
        n = int(seqlens[b])
        if n <= 0:
            continue
        npre = min(n, prefix_len)
        k, v = (np.concatenate([gather_keys(p, prefix_table, npre) if npre else np.zeros((KVH, 0, D)),
                                gather_keys(p, page_table[b], n)[:, npre:] if n > npre else np.zeros((KVH, 0, D))], 1)
                for p in (k_pages, v_pages))
        for t in range(T):
            lim = n - T + 1 + t
            if lim <= 0:
                continue
            for h in range(H):
                kk, vv = k[h // G, :lim], v[h // G, :lim]
                s = kk @ q[b, t, h] * scale
                p = np.exp(s - s.max())
                out[b, t, h] = (p / p.sum()) @ vv
                mass[b, t, h] = (p / p.sum()) @ np.abs(vv)
                reach[b, t, h] = (np.abs(kk) @ np.abs(q[b, t, h])).max() * abs(scale)
    return out, mass, reach


def rope_ref(x, cos, sin, weight=None, eps=0.0):
    """x [N, heads, D], cos / sin [N, D] (rows of each token's position) -> (y, size): the rotated (and, with
    a weight, first normalised) heads and the size |x' cos| + |rot(x') sin| of the two terms."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    half = x.shape[-1] // 2
    rot = np.concatenate([-x[..., half:], x[..., :half]], -1)
    a, b = x * cos[:, None], rot * sin[:, None]
    return a + b, np.abs(a) + np.abs(b)


def verify_ref(draft, target, uniforms, draft_probs=None, draft_lens=None):
    """draft [B, K] ids, target [B, K+1, V], uniforms [B, K+1] -> (tokens [B, K+1], accepted [B])."""
    B, K = draft.shape
    V = target.shape[2]
    tokens, accepted = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int32)
    for b in range(B):
        n = K if draft_lens is None else min(max(int(draft_lens[b]), 0), K)
        a = 0
        while a < n:
            x = int(draft[b, a])
            if not 0 <= x < V:
                break
            q = 1.0 if draft_probs is None else float(draft_probs[b, a, x])
            if not float(uniforms[b, a]) * q < float(target[b, a, x]):
                break
            a += 1
        p = np.asarray(target[b, a], np.float64)
        w = p.copy()
        if a < n:
            if draft_probs is not None:
                w = p - np.asarray(draft_probs[b, a], np.float64)
            elif 0 <= draft[b, a] < V:
                w[draft[b, a]] = 0.0
        w = np.where(w > 0, w, 0.0)
        if not w.sum() > 0:
            w = np.where(p > 0, p, 0.0)
        run = np.cumsum(w)
        above = np.nonzero((run > float(uniforms[b, K]) * run[-1]) & (w > 0))[0]
        some = np.nonzero(w > 0)[0]
        tokens[b, :a] = draft[b, :a]
        tokens[b, a] = above[0] if above.size else some[-1] if some.size else -1
        accepted[b] = a
    return tokens, accepted
