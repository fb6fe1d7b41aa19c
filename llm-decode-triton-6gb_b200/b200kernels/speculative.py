"""Verification of drafted tokens (speculative sampling), next to the greedy ``lm_head_argmax``.

No counterpart in the reference, which decodes one token at a time. ``verify_drafts`` accepts the leading
drafts with ``u * q(x) < p(x)`` and draws one more token, from ``max(p - q, 0)`` at the first refused position
or from ``p`` behind the last draft, so the tokens are distributed as the target model's own. Work runs in
``libb200decode.so`` (``b2d_verify_drafts``); there is no fallback.
"""
from __future__ import annotations

import torch

from . import _lib

MAX_DRAFTS = 31


def verify_drafts(draft_tokens: torch.Tensor, target_probs: torch.Tensor, uniforms: torch.Tensor,
                  draft_probs: torch.Tensor | None = None, draft_lens: torch.Tensor | None = None,
                  tokens: torch.Tensor | None = None, accepted: torch.Tensor | None = None, flags: int = 0):
    """draft_tokens int64 [B, K] (K <= 31), target_probs [B, K+1, V], uniforms fp32 [B, K+1] in [0, 1) ->
    (tokens int64 [B, K+1], accepted int32 [B]). Row b of ``tokens`` holds the accepted drafts, the drawn
    token, then -1. ``draft_probs`` [B, K, V] are what the drafts were drawn from (same dtype as
    ``target_probs``: fp32, fp16 or bf16); None means drafts that were not sampled (probability 1 on each).
    ``draft_lens`` int32 [B]: drafts per sequence (default K). ``uniforms[b, i]`` decides draft i,
    ``uniforms[b, K]`` draws the token: the first v whose running sum of weights exceeds it times their sum,
    in 64 bits. Pass ``tokens`` / ``accepted`` to reuse buffers."""
    if draft_tokens.dim() != 2 or draft_tokens.dtype != torch.int64:
        raise ValueError(f"draft_tokens is int64 [B, K], got {draft_tokens.dtype} {tuple(draft_tokens.shape)}")
    B, K = draft_tokens.shape
    if K > MAX_DRAFTS:
        raise ValueError(f"at most {MAX_DRAFTS} drafts per sequence, got {K}")
    if target_probs.dim() != 3 or target_probs.shape[:2] != (B, K + 1) or target_probs.shape[2] == 0:
        raise ValueError(f"target_probs is [{B}, {K + 1}, V], got {tuple(target_probs.shape)}")
    V = target_probs.shape[2]
    if target_probs.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"target_probs is fp32, fp16 or bf16, got {target_probs.dtype}")
    if target_probs.stride(2) != 1 and V > 1:
        raise ValueError("the last dimension of target_probs must be contiguous")
    sd = (0, 0)
    if draft_probs is not None:
        if draft_probs.shape != (B, K, V):
            raise ValueError(f"draft_probs is [{B}, {K}, {V}], got {tuple(draft_probs.shape)}")
        if draft_probs.dtype != target_probs.dtype:
            raise TypeError(f"draft_probs is {draft_probs.dtype}, target_probs {target_probs.dtype}")
        if draft_probs.stride(2) != 1 and V > 1:
            raise ValueError("the last dimension of draft_probs must be contiguous")
        sd = draft_probs.stride()
    if uniforms.dtype != torch.float32 or uniforms.shape != (B, K + 1):
        raise ValueError(f"uniforms is fp32 [{B}, {K + 1}], got {uniforms.dtype} {tuple(uniforms.shape)}")
    if draft_lens is not None and (draft_lens.dtype != torch.int32 or draft_lens.shape != (B,) or
                                   (B > 1 and draft_lens.stride(0) != 1)):
        raise ValueError(f"draft_lens is a contiguous int32 [{B}], got {draft_lens.dtype} {tuple(draft_lens.shape)}")
    if tokens is None:
        tokens = torch.empty((B, K + 1), dtype=torch.int64, device=target_probs.device)
    elif tokens.dtype != torch.int64 or tokens.shape != (B, K + 1):
        raise ValueError(f"tokens is int64 [{B}, {K + 1}], got {tokens.dtype} {tuple(tokens.shape)}")
    if accepted is None:
        accepted = torch.empty(B, dtype=torch.int32, device=target_probs.device)
    elif accepted.dtype != torch.int32 or accepted.shape != (B,) or (B > 1 and accepted.stride(0) != 1):
        raise ValueError(f"accepted is a contiguous int32 [{B}], got {accepted.dtype} {tuple(accepted.shape)}")
    if (K > 1 and draft_tokens.stride(1) != 1) or (K and (uniforms.stride(1) != 1 or tokens.stride(1) != 1)):
        raise ValueError("the last dimension of draft_tokens, uniforms and tokens must be contiguous")
    device = target_probs.device
    for name, t in (("draft_tokens", draft_tokens), ("draft_probs", draft_probs), ("uniforms", uniforms),
                    ("draft_lens", draft_lens), ("tokens", tokens), ("accepted", accepted)):
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, target_probs on {device}")
    index = _lib.cuda_index(device)
    st = target_probs.stride()
    _lib.call_on(index, "b2d_verify_drafts", draft_tokens.data_ptr(), draft_tokens.stride(0) if B > 1 else K,
                 _lib.ptr(draft_lens), target_probs.data_ptr(), st[0], st[1], _lib.ptr(draft_probs), sd[0], sd[1],
                 _lib.dtype_code(target_probs.dtype), uniforms.data_ptr(), uniforms.stride(0) if B > 1 else K + 1,
                 tokens.data_ptr(), tokens.stride(0) if B > 1 else K + 1, accepted.data_ptr(), B, K, V, flags)
    return tokens, accepted
