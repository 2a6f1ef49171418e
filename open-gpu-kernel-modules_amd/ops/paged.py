"""Serving ops over a paged KV cache (csrc/kernels/paged_ops.hip, paged_attn.hip):
requests of different lengths in one batch, each with its own pages.

  plan(...)       where every new token of a step goes: pages from a free list, block tables, slots
  rope_kv(...)    RoPE of q and k at each row's own position + append of k / v into the pages
  attention(...)  causal attention of each request's new rows (one token, a few drafted
                  ones, a prompt chunk, all in one call) over its pages

``fused.rope_kv`` / ``fused.attention`` are the contiguous-cache forms of the same
ops (one position and one length for the whole batch). The fake backend runs the
C++ references (csrc/core/paged_ref.cpp).

Page pool: [2, num_pages, hkv, page_size, hd] (k then v), bf16 or fp16; page_size
a power of two of 16 .. 256; the three outer strides are free, so a layer's slice
of a larger pool is fine. Block table: int32 [B, width], row b lists the pages of
request b in order. Lengths and tables stay on the device: no op reads them back,
so a step can be captured into a graph and replayed over changed lengths.
Everything runs on the current stream of the tensors' device; a workspace is
allocated per call on that stream, so calls on other streams and captured graphs
share none.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from .._native import lib

_ELEM = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I32 = torch.int32

# The checks of shapes, strides and types of a call run once per layout: a decode
# step calls these ops with the same layouts over and over, and on the smallest
# ones the host is what limits the rate. Nothing of a tensor's content, address
# or identity is kept.
_per_layout = functools.lru_cache(maxsize=512)


def _where(op: str, first: torch.Tensor, *others: torch.Tensor) -> tuple[int, int]:
    """(device index, stream) of a call, (-1, 0) on the host. Every tensor has to be
    on the first one's device; the binding checks that the backend runs there."""
    if first.is_cuda:
        dev = first.get_device()
        for t in others:
            if t.get_device() != dev:
                raise ValueError(f"{op}: tensors on {first.device} and {t.device}")
        return dev, torch._C._cuda_getCurrentRawStream(dev)
    for t in others:
        if t.device != first.device:
            raise ValueError(f"{op}: tensors on {first.device} and {t.device}")
    if first.device.type != "cpu":
        raise ValueError(f"{op}: tensors must be on a GPU")
    return -1, 0


def _ints(op: str, name: str, t: torch.Tensor, shape: tuple) -> None:
    if t.dtype is not _I32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{op}: {name} must be contiguous int32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def _check_table(op: str, dtype, shape, stride, B: int) -> None:
    if dtype is not _I32 or len(shape) != 2 or shape[0] != B or shape[1] < 1 or (
            shape[1] > 1 and stride[1] != 1) or (B > 1 and stride[0] < shape[1]):
        raise ValueError(f"{op}: block_table must be int32 [{B}, width] with rows apart")


def _check_page_size(op: str, size: int) -> None:
    if size < 16 or size > 256 or size & (size - 1):
        raise ValueError(f"{op}: page size must be a power of two of 16 .. 256 tokens, got {size}")


def _check_pool(op: str, dtype, shape, stride, rows_dtype) -> None:
    if len(shape) != 5 or shape[0] != 2 or dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{op}: pages must be bf16 or fp16 [2, num_pages, hkv, page_size, hd]")
    _, num, hkv, size, hd = shape
    _check_page_size(op, size)
    if num * size > 2**31 - 1 or num < 1 or hkv < 1 or hkv > 65535:
        raise ValueError(f"{op}: the pool must hold 1 .. 2^31 - 1 slots of 1 .. 65535 heads")
    if stride[4] != 1 or stride[3] != hd or any(n > 1 and st % 8 for n, st in zip(shape[:3], stride[:3])):
        raise ValueError(f"{op}: a page's rows must be contiguous and 16-byte aligned")
    if rows_dtype != dtype:
        raise ValueError(f"{op}: {rows_dtype} rows over {dtype} pages")


def _unaligned(op: str):
    raise ValueError(f"{op}: tensors must be 16-byte aligned")


class Plan(NamedTuple):
    """One step of a batch, all int32 on the device. ``granted[b]`` is 0 where
    request b's tokens do not fit its table row, where its rows end behind
    n_tokens, or where it lacks pages and those asked for up to it, its own among
    them, are more than the free list has: its lengths and pages then stay as they
    were and its rows have position and slot -1.

    Pages are asked for in request order, and a request that finds too few keeps its
    place: those behind it that lack pages are refused too, however few they lack,
    so that small requests never overtake a large one for good. (One that does not
    fit its table row or the batch asks for none.) A server therefore puts running
    requests before those it admits, and takes a refused admission out of the next
    batches (0 new tokens) until pages came back."""

    cu_q: torch.Tensor         # [B + 1] first row of each request
    kv_lens: torch.Tensor      # [B] cached tokens after the step
    page_counts: torch.Tensor  # [B] pages held after the step
    granted: torch.Tensor      # [B]
    positions: torch.Tensor    # [n_tokens], -1 in rows behind the last request
    slots: torch.Tensor        # [n_tokens] page * page_size + row, -1: store nothing
    free_start: torch.Tensor   # [1] first unused entry of free_pages after the step


def plan(new_lens: torch.Tensor, kv_lens: torch.Tensor, page_counts: torch.Tensor, block_table: torch.Tensor,
         free_pages: torch.Tensor, free_start: torch.Tensor, page_size: int, n_tokens: int) -> Plan:
    """Place ``new_lens[b]`` new tokens (0 allowed) behind the ``kv_lens[b]`` cached
    ones of each request, whose rows follow each other in a batch of ``n_tokens``
    rows. Pages a request lacks are taken, in request order, from
    ``free_pages[free_start:]`` and written into ``block_table`` (in place) behind
    the ``page_counts[b]`` it holds - a count of its own, since a request whose
    drafts were refused keeps pages beyond its length. One launch; at most
    4096 requests. Negative lengths and counts are taken as 0."""
    B, n_free = _plan_layout(new_lens.shape, block_table.dtype, block_table.shape, block_table.stride(),
                             free_pages.shape, page_size, n_tokens)
    shape = (B,)
    _ints("plan", "new_lens", new_lens, shape)
    _ints("plan", "kv_lens", kv_lens, shape)
    _ints("plan", "page_counts", page_counts, shape)
    _ints("plan", "free_pages", free_pages, (n_free,))
    _ints("plan", "free_start", free_start, (1,))
    dev, stream = _where("plan", new_lens, kv_lens, page_counts, block_table, free_pages, free_start)
    # one allocation for the seven outputs
    out = new_lens.new_empty(4 * B + 2 * n_tokens + 2)
    lib.paged_plan(dev, stream, new_lens.data_ptr(), kv_lens.data_ptr(), page_counts.data_ptr(),
                   block_table.data_ptr(), block_table.stride(0), free_pages.data_ptr(), free_start.data_ptr(),
                   out.data_ptr(), B, block_table.shape[1], n_free, page_size, n_tokens)
    return Plan(*out.split_with_sizes((B + 1, B, B, B, n_tokens, n_tokens, 1)))


@_per_layout
def _plan_layout(lens, table_dtype, table, table_stride, free, page_size, n_tokens):
    if len(lens) != 1 or len(free) != 1:
        raise ValueError("plan: lengths and free_pages must be lists")
    B, most = lens[0], lib.paged_plan_max_requests()
    _check_table("plan", table_dtype, table, table_stride, B)
    _check_page_size("plan", page_size)
    if B > most or not 0 <= n_tokens < 2**31 or table[1] * page_size >= 2**31 or free[0] >= 2**31:
        raise ValueError(f"plan: at most {most} requests; rows and positions below 2^31")
    return B, free[0]


def rope_kv(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pages: torch.Tensor, positions: torch.Tensor,
            slots: torch.Tensor, hq: int, hkv: int) -> torch.Tensor:
    """qkv [n, (hq + 2 hkv) hd] -> rotated q [n, hq, hd]; the rotated k and the v of
    row t are stored into slot ``slots[t]`` of the pool. cos / sin: f32 [max_pos,
    hd / 2] (rotate-half). A row with position -1 is padding: its q is 0 and
    nothing is stored, as for a slot outside the pool; a position behind the
    tables gives NaN. Slots of one call are distinct (of two rows with one slot
    either's values may stay); the pool's pages share no memory."""
    n, hd, num, size, max_pos = _rope_layout(qkv.dtype, qkv.shape, qkv.stride(), pages.dtype, pages.shape,
                                             pages.stride(), cos.dtype, cos.shape, cos.stride(), sin.dtype, sin.shape,
                                             sin.stride(), hq, hkv)
    shape = (n,)
    _ints("rope_kv", "positions", positions, shape)
    _ints("rope_kv", "slots", slots, shape)
    dev, stream = _where("rope_kv", qkv, cos, sin, pages, positions, slots)
    q = qkv.new_empty((n, hq, hd))
    x, c, s, p = qkv.data_ptr(), cos.data_ptr(), sin.data_ptr(), pages.data_ptr()
    if (x | c | s | p) & 15:
        _unaligned("rope_kv")
    kv_stride, page_stride, head_stride = pages.stride()[:3]
    lib.paged_rope(dev, stream, x, qkv.stride(0), c, s, positions.data_ptr(), slots.data_ptr(), q.data_ptr(), p,
                   kv_stride, page_stride, head_stride, n, hq, hkv, hd, num, size, max_pos, _ELEM[qkv.dtype])
    return q


@_per_layout
def _rope_layout(dtype, qkv, qkv_stride, pool_dtype, pool, pool_stride, cos_dtype, cos, cos_stride, sin_dtype, sin,
                 sin_stride, hq, hkv):
    _check_pool("rope_kv", pool_dtype, pool, pool_stride, dtype)
    _, num, heads, size, hd = pool
    span = 0  # an element of one page may not be an element of another: the rows are written
    for st, n in sorted((st, n) for n, st in zip(pool[:4], pool_stride[:4]) if n > 1):
        if st < max(span, hd):
            raise ValueError("rope_kv: the pool's pages overlap")
        span = st * (n - 1) + max(span, hd)
    if hkv != heads or hq < 1 or hd % 16:
        raise ValueError(f"rope_kv: {hkv} kv heads over a pool of {heads}, hd {hd} (a multiple of 16)")
    if len(qkv) != 2 or qkv[1] != (hq + 2 * hkv) * hd or qkv_stride[1] != 1 or (qkv[0] > 1 and qkv_stride[0] % 8):
        raise ValueError("rope_kv: qkv must be [n, (hq + 2 hkv) hd] with contiguous, 16-byte aligned rows")
    for name, d, shape, stride in (("cos", cos_dtype, cos, cos_stride), ("sin", sin_dtype, sin, sin_stride)):
        if d is not torch.float32 or len(shape) != 2 or shape[1] * 2 != hd or stride != (hd // 2, 1) \
                or shape != cos or not 1 <= shape[0] < 2**31:
            raise ValueError(f"rope_kv: {name} must be contiguous f32 [max_pos, {hd // 2}]")
    return qkv[0], hd, num, size, cos[0]


def attention(q: torch.Tensor, pages: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor,
              block_table: torch.Tensor, max_q: int | None = None, max_kv: int | None = None,
              scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [n, hq, hd] (rotated), rows [cu_q[b], cu_q[b + 1]) of request b being its last
    new tokens of the ``kv_lens[b]`` cached ones -> [n, hq * hd]: row i of a request
    sees its tokens 0 .. kv_lens - rows + i. A row that sees nothing gives 0. ``cu_q``
    ascends; bounds outside q are cut to it, and rows of no request (those behind
    cu_q[B]) are left as they are in ``out``. What no row sees (the rest of a
    last page, a later token) cannot reach a result, NaN or not. Rows that would
    need a page outside the pool or beyond their table row give NaN.

    Scores, maxima, sums and the result before its one rounding are f32. A single
    token's probabilities (of up to 32 query heads a kv head), and a draft's where no
    request of the batch may have more than 32 rows per kv head (``max_q``), are
    multiplied with twice the type's bits, so that such a call is as exact as
    ``fused.attention``. Those of longer chunks are rounded to the type, which adds an
    error of up to half a step of it relative to sum p |v|.

    ``max_q`` / ``max_kv``: the host's bounds of rows and length per request; they
    only choose how the work is split (default: n and the table's width). ``out``
    shares no memory with q or the pool. Limits: 65535 requests, 2^30 tokens each."""
    n, B, hq, hkv, hd, num, size, width = _attention_layout(
        q.dtype, q.shape, q.stride(), pages.dtype, pages.shape, pages.stride(), kv_lens.shape, block_table.dtype,
        block_table.shape, block_table.stride())
    _ints("attention", "kv_lens", kv_lens, (B,))
    _ints("attention", "cu_q", cu_q, (B + 1,))
    max_q = n if max_q is None else min(max(int(max_q), 1), n)
    max_kv = width * size if max_kv is None else min(max(int(max_kv), 1), width * size)
    if out is None:
        out = q.new_empty((n, hq * hd))
    elif out.dtype != q.dtype or tuple(out.shape) != (n, hq * hd) or out.stride(1) != 1 or (
            n > 1 and (out.stride(0) % 8 or out.stride(0) < hq * hd)):
        raise ValueError(f"attention: out must be {q.dtype} [{n}, {hq * hd}] with contiguous, aligned rows")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not 1e-30 < abs(scale) < 1e30:
        raise ValueError(f"attention: scale {scale}")
    dev, stream = _where("attention", q, pages, cu_q, kv_lens, block_table, out)
    part, part_bytes = 0, 0
    if dev >= 0:
        part_bytes = lib.paged_attn_workspace(n, B, hq, hkv, hd, max_q, max_kv)
        if part_bytes:
            work = q.new_empty(part_bytes // 2)
            part = work.data_ptr()
    x, p, y = q.data_ptr(), pages.data_ptr(), out.data_ptr()
    if (x | p | y) & 15:
        _unaligned("attention")
    q_stride, q_head_stride, _ = q.stride()
    kv_stride, page_stride, head_stride = pages.stride()[:3]
    lib.paged_attn(dev, stream, x, q_stride, q_head_stride, p, kv_stride, page_stride, head_stride, cu_q.data_ptr(),
                   kv_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), y, out.stride(0), n, B, hq, hkv,
                   hd, num, size, width, scale, _ELEM[q.dtype], max_q, max_kv, part, part_bytes)
    return out


@_per_layout
def _attention_layout(dtype, q, q_stride, pool_dtype, pool, pool_stride, lens, table_dtype, table, table_stride):
    _check_pool("attention", pool_dtype, pool, pool_stride, dtype)
    _, num, hkv, size, hd = pool
    if hd not in (64, 128):
        raise ValueError(f"attention: head dim 64 or 128, got {hd}")
    if len(q) != 3 or q[2] != hd or q[1] < 1 or q[1] % hkv:
        raise ValueError(f"attention: q must be [n, hq, {hd}] with hq a multiple of {hkv}")
    if q_stride[2] != 1 or any(c > 1 and s % 8 for c, s in zip(q[:2], q_stride[:2])):
        raise ValueError("attention: q's heads must be contiguous and 16-byte aligned")
    if q[0] * q[1] >= 2**31:
        raise ValueError("attention: fewer than 2^31 rows x heads")
    if len(lens) != 1 or lens[0] > 65535:
        raise ValueError("attention: kv_lens must list at most 65535 requests")
    _check_table("attention", table_dtype, table, table_stride, lens[0])
    if table[1] * size > 2**30:
        raise ValueError("attention: at most 2^30 tokens per request")
    return q[0], lens[0], q[1], hkv, hd, num, size, table[1]
