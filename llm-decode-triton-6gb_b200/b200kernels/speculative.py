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
    r = _lib.binding().verify(draft_tokens, target_probs, uniforms, draft_probs, draft_lens, tokens, accepted, flags)
    if r.__class__ is int:
        raise _lib.B2DError("b2d_verify_drafts", r)
    return r
