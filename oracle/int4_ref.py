"""Definitions of the 4-bit paged cache's operators and of page planning.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``): the product never imports this. The reference has neither. The
quantiser's steps are IEEE fp32 by definition and are followed as such; everything behind it is float64 (attention:
``paged_ref.paged_attention_ref`` on the values that the codes stand for).
"""
from __future__ import annotations

import numpy as np
import torch


def quantise_ref(x, group, dtype):
    """x fp32 [..., D] (numpy) -> (codes, s, m), the latter two fp32 [..., D / group] of dtype's values."""
    def round16(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).float().numpy()
    x = np.asarray(x, np.float32)
    x = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        m = round16(x.min(-1))
        s = round16(np.maximum((x.max(-1) - m) * (np.float32(1) / np.float32(15)), np.float32(0)))   # torch's x / 15 on a GPU
        c = np.where(s[..., None] > 0, np.clip(np.rint((x - m[..., None]) / s[..., None]), 0, 15), 0)
    odd = ~np.isfinite(x).all(-1) | ~np.isfinite(m) | ~np.isfinite(s)
    s, m, c = np.where(odd, np.nan, s), np.where(odd, np.nan, m), np.where(odd[..., None], 0, c)
    return c.astype(np.uint8), s.astype(np.float32), m.astype(np.float32)


def values_ref(codes, s, m, D):
    """What codes stand for, in fp32 as the read gives them (one rounding of m + s c): [..., D]."""
    v = m[..., None].astype(np.float64) + s[..., None].astype(np.float64) * codes
    return v.astype(np.float32).reshape(*v.shape[:-2], D)


def size_ref(codes, s, m, D):
    """|m| + s c, the size of an entry's two terms."""
    v = np.abs(m[..., None].astype(np.float64)) + s[..., None].astype(np.float64) * codes
    return v.reshape(*v.shape[:-2], D)


def turn_ref(x, cos, sin, interleaved, weight=None, eps=0.0, exact32=False):
    """x [N, heads, D], cos / sin [N, R / 2] of each token -> the normed and turned heads, in float64, or (``exact32``) in
    the fp32 steps that the definition of a cached key has."""
    t = np.float32 if exact32 else np.float64
    x = np.asarray(x).astype(t)
    if weight is not None:
        r = 1 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        x = (x * r.astype(t)) * np.asarray(weight).astype(t)
    if cos is None:
        return x
    cos, sin = np.asarray(cos).astype(t)[:, None], np.asarray(sin).astype(t)[:, None]
    R = 2 * cos.shape[-1]
    y = x.copy()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        y[..., 0:R:2], y[..., 1:R:2] = ya, yb
    else:
        y[..., :R // 2], y[..., R // 2:R] = ya, yb
    return y


def plan_ref(page_table, held, free, ring, cached, new, page_size, max_tokens):
    """One step of the page tables, sequence by sequence; lists / arrays of ints in, a dict of new ones out."""
    table = np.array(page_table, np.int64)
    (B, W), P = table.shape, len(free)
    free_out, held_out = np.array(free, np.int64), np.array(held, np.int64)
    first, count = (int(ring[0]) % P, min(max(int(ring[1]), 0), P)) if P else (0, 0)
    out = {"positions": np.full(max_tokens, -1, np.int64), "seq_ids": np.full(max_tokens, -1, np.int32),
           "slots": np.full(max_tokens, -1, np.int64), "seqlens": np.zeros(B, np.int32), "starts": np.zeros(B + 1, np.int32),
           "granted": np.zeros(B, np.int32)}
    asked_pages = asked_tokens = taken = given = n = 0
    for b in range(B):
        c, f = max(int(cached[b]), 0), max(int(new[b]), 0)
        h = min(max(int(held[b]), 0), W)
        target = -(-(c + f) // page_size)
        ok = target <= W
        if ok:
            need = max(target - h, 0)
            asked_pages += need
            asked_tokens += f
            ok = (need == 0 or asked_pages <= count) and (f == 0 or asked_tokens <= max_tokens)
        out["starts"][b] = n
        out["granted"][b] = f if ok else -1
        out["seqlens"][b] = c + f if ok else c
        if not ok:
            continue
        for i in range(h, target):
            table[b, i] = free[(first + taken) % P]
            taken += 1
        for i in range(target, h):
            if count + given < P:
                free_out[(first + count + given) % P] = table[b, i]
            given += 1
            table[b, i] = -1
        held_out[b] = target
        for p in range(c, c + f):
            page = int(table[b, p // page_size])
            out["positions"][n], out["seq_ids"][n] = p, b
            if 0 <= page < P:
                out["slots"][n] = page * page_size + p % page_size
            n += 1
    out["starts"][B] = n
    out.update(page_table=table, held=held_out, free=free_out,
               ring=np.array([(first + taken) % P if P else 0, min(count - taken + given, P)]))
    return out
