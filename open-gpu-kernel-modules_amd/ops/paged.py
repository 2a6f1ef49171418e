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

import math
from dataclasses import dataclass

import torch

from .._native import lib

_ELEM = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _where(op: str, first: torch.Tensor, **tensors: torch.Tensor) -> tuple[int, int]:
    """(device index, stream) of a call. Every tensor has to be on the first
    one's device, and that has to be the runtime backend's kind of device."""
    for name, t in tensors.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{op}: {name} is on {t.device}, expected {first.device}")
    if lib.backend_name() == "fake":
        if first.device.type != "cpu":
            raise ValueError(f"{op}: the fake backend takes CPU tensors")
        return 0, 0
    if first.device.type != "cuda":
        raise ValueError(f"{op}: tensors must be on a GPU")
    dev = first.device.index
    return dev, int(torch.cuda.current_stream(dev).cuda_stream)


def _ints(op: str, name: str, t: torch.Tensor, shape: tuple) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{op}: {name} must be contiguous int32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def _table(op: str, table: torch.Tensor, B: int) -> None:
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or table.shape[1] < 1 or (
            table.shape[1] > 1 and table.stride(1) != 1) or (B > 1 and table.stride(0) < table.shape[1]):
        raise ValueError(f"{op}: block_table must be int32 [{B}, width] with rows apart")


def _page_size(op: str, size: int) -> None:
    if size < 16 or size > 256 or size & (size - 1):
        raise ValueError(f"{op}: page size must be a power of two of 16 .. 256 tokens, got {size}")


def _pool(op: str, pages: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if pages.dim() != 5 or pages.shape[0] != 2 or pages.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{op}: pages must be bf16 or fp16 [2, num_pages, hkv, page_size, hd]")
    _, num, hkv, size, hd = pages.shape
    _page_size(op, size)
    if num * size > 2**31 - 1 or num < 1 or hkv < 1:
        raise ValueError(f"{op}: the pool must hold 1 .. 2^31 - 1 slots of at least one head")
    if pages.stride(4) != 1 or pages.stride(3) != hd or any(
            n > 1 and (st % 8 or st < 0) for n, st in zip(pages.shape[:3], pages.stride()[:3])) or pages.data_ptr() % 16:
        raise ValueError(f"{op}: a page's rows must be contiguous and 16-byte aligned")
    if like is not None and like.dtype != pages.dtype:
        raise ValueError(f"{op}: {like.dtype} rows over {pages.dtype} pages")


@dataclass
class Plan:
    """One step of a batch, all int32 on the device. ``granted[b]`` is 0 where
    request b's pages did not fit the free list or its table row, or its rows
    did not fit n_tokens: its lengths and pages then stay as they were and its
    rows have position and slot -1."""

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
    B = new_lens.shape[0] if new_lens.dim() == 1 else -1
    for name, t in (("new_lens", new_lens), ("kv_lens", kv_lens), ("page_counts", page_counts)):
        _ints("plan", name, t, (B,))
    _table("plan", block_table, B)
    _page_size("plan", page_size)
    if free_pages.dim() != 1:
        raise ValueError("plan: free_pages must be a list of pages")
    _ints("plan", "free_pages", free_pages, (free_pages.shape[0],))
    _ints("plan", "free_start", free_start, (1,))
    width = block_table.shape[1]
    if B > lib.paged_plan_max_requests() or not 0 <= n_tokens < 2**31 or width * page_size >= 2**31 \
            or free_pages.shape[0] >= 2**31:
        raise ValueError(f"plan: at most {lib.paged_plan_max_requests()} requests; rows and positions below 2^31")
    dev, stream = _where("plan", new_lens, kv_lens=kv_lens, page_counts=page_counts, block_table=block_table,
                         free_pages=free_pages, free_start=free_start)
    # one allocation for the seven outputs
    sizes = (B + 1, B, B, B, n_tokens, n_tokens, 1)
    parts = torch.empty(sum(sizes), dtype=torch.int32, device=new_lens.device).split(sizes)
    cu, kv, counts, granted, positions, slots, start = parts
    lib.paged_plan(dev, stream, new_lens.data_ptr(), kv_lens.data_ptr(), page_counts.data_ptr(),
                   block_table.data_ptr(), block_table.stride(0), free_pages.data_ptr(), free_start.data_ptr(),
                   cu.data_ptr(), kv.data_ptr(), counts.data_ptr(), granted.data_ptr(), positions.data_ptr(),
                   slots.data_ptr(), start.data_ptr(), B, width, free_pages.shape[0], page_size, n_tokens)
    return Plan(cu, kv, counts, granted, positions, slots, start)


def rope_kv(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pages: torch.Tensor, positions: torch.Tensor,
            slots: torch.Tensor, hq: int, hkv: int) -> torch.Tensor:
    """qkv [n, (hq + 2 hkv) hd] -> rotated q [n, hq, hd]; the rotated k and the v of
    row t are stored into slot ``slots[t]`` of the pool. cos / sin: f32 [max_pos,
    hd / 2] (rotate-half). A row with position -1 is padding: its q is 0 and
    nothing is stored, as for a slot outside the pool; a position behind the
    tables gives NaN. Slots of one call are distinct (of two rows with one slot
    either's values may stay)."""
    _pool("rope_kv", pages, qkv)
    _, num, heads, size, hd = pages.shape
    if hkv != heads or hq < 1 or hd % 16:
        raise ValueError(f"rope_kv: {hkv} kv heads over a pool of {heads}, hd {hd} (a multiple of 16)")
    if qkv.dim() != 2 or qkv.shape[1] != (hq + 2 * hkv) * hd or qkv.stride(1) != 1 or (
            qkv.shape[0] > 1 and (qkv.stride(0) % 8 or qkv.stride(0) < 0)) or qkv.data_ptr() % 16:
        raise ValueError("rope_kv: qkv must be [n, (hq + 2 hkv) hd] with contiguous, 16-byte aligned rows")
    n = qkv.shape[0]
    _ints("rope_kv", "positions", positions, (n,))
    _ints("rope_kv", "slots", slots, (n,))
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] * 2 != hd or not t.is_contiguous() \
                or t.shape != cos.shape or t.shape[0] < 1 or t.shape[0] >= 2**31 or t.data_ptr() % 16:
            raise ValueError(f"rope_kv: {name} must be contiguous f32 [max_pos, {hd // 2}]")
    dev, stream = _where("rope_kv", qkv, cos=cos, sin=sin, pages=pages, positions=positions, slots=slots)
    q = torch.empty(n, hq, hd, dtype=qkv.dtype, device=qkv.device)
    lib.paged_rope(dev, stream, qkv.data_ptr(), qkv.stride(0), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
                   slots.data_ptr(), q.data_ptr(), pages.data_ptr(), pages.stride(0), pages.stride(1), pages.stride(2),
                   n, hq, hkv, hd, num, size, cos.shape[0], _ELEM[qkv.dtype])
    return q


def attention(q: torch.Tensor, pages: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor,
              block_table: torch.Tensor, max_q: int | None = None, max_kv: int | None = None,
              scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [n, hq, hd] (rotated), rows [cu_q[b], cu_q[b + 1]) of request b being its last
    new tokens of the ``kv_lens[b]`` cached ones -> [n, hq * hd]: row i of a request
    sees its tokens 0 .. kv_lens - rows + i. A row that sees nothing gives 0; rows
    behind cu_q[B] are left as they are in ``out``. What no row sees (the rest of a
    last page, a later token) cannot reach a result, NaN or not. Rows that would
    need a page outside the pool or beyond their table row give NaN.

    ``max_q`` / ``max_kv``: the host's bounds of rows and length per request; they
    only choose how the work is split (default: n and the table's width)."""
    _pool("attention", pages, q)
    _, num, hkv, size, hd = pages.shape
    if hd not in (64, 128):
        raise ValueError(f"attention: head dim 64 or 128, got {hd}")
    if q.dim() != 3 or q.shape[2] != hd or q.shape[1] < 1 or q.shape[1] % hkv:
        raise ValueError(f"attention: q must be [n, hq, {hd}] with hq a multiple of {hkv}")
    n, hq = q.shape[:2]
    if q.stride(2) != 1 or any(c > 1 and (s % 8 or s < 0) for c, s in zip(q.shape[:2], q.stride()[:2])) \
            or q.data_ptr() % 16 or n >= 2**31:
        raise ValueError("attention: q's heads must be contiguous and 16-byte aligned")
    B = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    _ints("attention", "kv_lens", kv_lens, (B,))
    _ints("attention", "cu_q", cu_q, (B + 1,))
    _table("attention", block_table, B)
    width = block_table.shape[1]
    if width * size > 2**30 or B > 65535 or hkv > 65535:
        raise ValueError("attention: at most 2^30 tokens per request, 65535 requests and kv heads")
    max_q = n if max_q is None else min(max(int(max_q), 1), n)
    max_kv = width * size if max_kv is None else min(max(int(max_kv), 1), width * size)
    if out is None:
        out = torch.empty(n, hq * hd, dtype=q.dtype, device=q.device)
    elif out.dtype != q.dtype or tuple(out.shape) != (n, hq * hd) or out.stride(1) != 1 or (
            n > 1 and (out.stride(0) % 8 or out.stride(0) < hq * hd)) or out.data_ptr() % 16:
        raise ValueError(f"attention: out must be {q.dtype} [{n}, {hq * hd}] with contiguous, aligned rows")
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not 1e-30 < abs(scale) < 1e30:
        raise ValueError(f"attention: scale {scale}")
    dev, stream = _where("attention", q, pages=pages, cu_q=cu_q, kv_lens=kv_lens, block_table=block_table, out=out)
    part, part_bytes = None, 0
    if q.is_cuda:
        part_bytes = lib.paged_attn_workspace(n, B, hq, hkv, hd, max_q, max_kv)
        if part_bytes:
            part = torch.empty(part_bytes // 4, dtype=torch.float32, device=q.device)
    lib.paged_attn(dev, stream, q.data_ptr(), q.stride(0), q.stride(1), pages.data_ptr(), pages.stride(0),
                   pages.stride(1), pages.stride(2), cu_q.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(),
                   block_table.stride(0), out.data_ptr(), out.stride(0), n, B, hq, hkv, hd, num, size, width,
                   scale, _ELEM[q.dtype], max_q, max_kv,
                   part.data_ptr() if part is not None else 0, part_bytes)
    return out
