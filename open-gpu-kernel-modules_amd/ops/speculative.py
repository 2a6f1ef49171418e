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
from .paged import _ELEM, _ints, _per_layout, _where


@_per_layout
def _layout(dtype, shape, stride, q_dtype, q_shape, q_stride):
    if len(shape) != 3 or shape[1] < 1 or not 1 <= shape[2] <= 2**30:
        raise ValueError("verify_draft: target_probs must be [B, K + 1, V]")
    B, K, V = shape[0], shape[1] - 1, shape[2]
    if B > 65535 or K > 65535:
        raise ValueError("verify_draft: at most 65535 requests and drafts")
    for name, d, got, st, want in (("target_probs", dtype, shape, stride, (B, K + 1, V)),
                                   ("draft_probs", q_dtype, q_shape, q_stride, (B, K, V))):
        if d is not None and (got != want or d not in _ELEM or (V > 1 and st[2] != 1)):
            raise ValueError(f"verify_draft: {name} must be f32, bf16 or fp16 {list(want)} with contiguous rows")
    if q_dtype not in (None, dtype):
        raise ValueError(f"verify_draft: {q_dtype} drafts against a {dtype} target")
    return B, K, V, -(-V // lib.verify_chunk())


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
    p, q = target_probs, draft_probs
    if q is None:
        B, K, V, chunks = _layout(p.dtype, p.shape, p.stride(), None, None, None)
        q_ptr, q_batch, q_row, given = 0, 0, 0, p
    else:
        B, K, V, chunks = _layout(p.dtype, p.shape, p.stride(), q.dtype, q.shape, q.stride())
        q_ptr, (q_batch, q_row, _), given = q.data_ptr(), q.stride(), q
    _ints("verify_draft", "draft_tokens", draft_tokens, (B, K))
    if u.dtype is not torch.float32 or u.shape != (B, K) or not u.is_contiguous():
        raise ValueError(f"verify_draft: u must be contiguous f32 [{B}, {K}]")
    if u_last.dtype is not torch.float32 or u_last.shape != (B,) or not u_last.is_contiguous():
        raise ValueError(f"verify_draft: u_last must be contiguous f32 [{B}]")
    counted = u if counts is None else counts
    if counts is not None:
        _ints("verify_draft", "counts", counts, (B,))
    dev, stream = _where("verify_draft", p, given, draft_tokens, u, u_last, counted)
    # workspace and outputs in one allocation: f64 sums by chunk, tokens, accepted
    sums = 2 * B * chunks
    out = draft_tokens.new_empty((sums + B * (K + 2),))
    _, tokens, accepted = out.split_with_sizes((sums, B * (K + 1), B))
    p_batch, p_row, _ = p.stride()
    lib.verify_draft(dev, stream, p.data_ptr(), p_batch, p_row, q_ptr, q_batch, q_row, draft_tokens.data_ptr(),
                     u.data_ptr(), u_last.data_ptr(), 0 if counts is None else counts.data_ptr(), tokens.data_ptr(),
                     accepted.data_ptr(), out.data_ptr(), B, K, V, _ELEM[p.dtype])
    return tokens.view(B, K + 1), accepted
