"""Speculative decoding: drafted tokens checked against the target model's
probabilities (csrc/kernels/speculative.hip; the fake backend runs
csrc/core/paged_ref.cpp).

The target scores a request's last token and its K drafts in one batch
(paged.attention takes the K + 1 rows), which gives K + 1 rows of probabilities;
``verify_draft`` keeps the longest prefix of drafts the target agrees with and
draws one more token, so that the tokens are distributed as the target's own.
"""
from __future__ import annotations

import torch

from .._native import lib
from .paged import _ELEM, _ints, _where


def _rows(name: str, t: torch.Tensor, shape: tuple) -> None:
    if t.dim() != 3 or tuple(t.shape) != shape or t.dtype not in _ELEM or (t.shape[2] > 1 and t.stride(2) != 1) \
            or any(n > 1 and s < 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"verify_draft: {name} must be f32, bf16 or fp16 {list(shape)} with contiguous rows")


def verify_draft(target_probs: torch.Tensor, draft_probs: torch.Tensor | None, draft_tokens: torch.Tensor,
                 u: torch.Tensor, u_last: torch.Tensor, counts: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """target_probs [B, K + 1, V], draft_probs [B, K, V] (None: the drafts were certain,
    e.g. greedy), draft_tokens int32 [B, K], u f32 [B, K] and u_last f32 [B] uniform in
    [0, 1), counts int32 [B] (drafts of each request, default K) -> tokens int32
    [B, K + 1], accepted int32 [B].

    Draft j stays while ``u[j] * draft_probs[j][x] < target_probs[j][x]``. ``accepted``
    m is the first that does not (or the count); tokens are the m drafts, then the
    smallest i whose running sum of max(target_probs[m] - draft_probs[m], 0) passes
    ``u_last`` times the whole (of target_probs[m] alone where no draft is left or
    nothing remains), then -1. Rows need not be normalised. A token outside the
    vocabulary is refused; a NaN or negative probability weighs nothing; a row
    without any weight gives -1."""
    if target_probs.dim() != 3 or target_probs.shape[1] < 1 or not 1 <= target_probs.shape[2] < 2**31:
        raise ValueError("verify_draft: target_probs must be [B, K + 1, V]")
    B, K, V = target_probs.shape[0], target_probs.shape[1] - 1, target_probs.shape[2]
    if B > 65535 or K > 65535:
        raise ValueError("verify_draft: at most 65535 requests and drafts")
    _rows("target_probs", target_probs, (B, K + 1, V))
    if draft_probs is not None:
        _rows("draft_probs", draft_probs, (B, K, V))
        if draft_probs.dtype != target_probs.dtype:
            raise ValueError(f"verify_draft: {draft_probs.dtype} drafts against a {target_probs.dtype} target")
    _ints("verify_draft", "draft_tokens", draft_tokens, (B, K))
    for name, t, shape in (("u", u, (B, K)), ("u_last", u_last, (B,))):
        if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"verify_draft: {name} must be contiguous f32 {list(shape)}")
    if counts is not None:
        _ints("verify_draft", "counts", counts, (B,))
    dev, stream = _where("verify_draft", target_probs, draft_probs=draft_probs, draft_tokens=draft_tokens, u=u,
                         u_last=u_last, counts=counts)
    chunks = -(-V // lib.verify_chunk())
    sums = torch.empty(B * chunks * 2, dtype=torch.float64, device=target_probs.device)
    out = torch.empty(B * (K + 2), dtype=torch.int32, device=target_probs.device)
    tokens, accepted = out[:B * (K + 1)].view(B, K + 1), out[B * (K + 1):]
    q = draft_probs
    lib.verify_draft(dev, stream, target_probs.data_ptr(), target_probs.stride(0), target_probs.stride(1),
                     q.data_ptr() if q is not None and K else 0, q.stride(0) if q is not None else 0,
                     q.stride(1) if q is not None else 0, draft_tokens.data_ptr(), u.data_ptr(), u_last.data_ptr(),
                     counts.data_ptr() if counts is not None else 0, tokens.data_ptr(), accepted.data_ptr(),
                     sums.data_ptr(), sums.numel() * 8, B, K, V, _ELEM[target_probs.dtype])
    return tokens, accepted
