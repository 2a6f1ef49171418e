"""Paged serving ops (csrc/kernels/paged_ops.hip, paged_attn.hip; CPU references
in csrc/core/paged_ref.cpp) against plain f64 forms written here: the step plan,
RoPE into pages, attention over pages; their refusals; and a run of them together
against the contiguous-cache ops."""
from __future__ import annotations

import math

import pytest
import torch

from ogkm.ops import decode as D
from ogkm.ops import fused, paged, speculative

I32 = torch.int32


def _dev(gpu):
    return "cuda" if gpu else "cpu"


def _i32(v, dev):
    return torch.tensor(v, dtype=I32).to(dev)


# ---------------------------------------------------------------- plan
def _plan_oracle(new, kv, held, table, free, start, P, n):
    """Request by request, from the definition."""
    table = [list(r) for r in table]
    width, end, asked, taken = len(table[0]) if table else 0, 0, 0, 0
    cu, kv2, held2, granted = [0], [], [], []
    pos, slot = [-1] * n, [-1] * n
    for b, (x, k, h) in enumerate(zip(new, kv, held)):
        x, k, h = max(x, 0), max(k, 0), min(max(h, 0), width)
        row, end = end, end + x
        total = -(-(k + x) // P)
        fits = total <= width and end <= n
        need = max(total - h, 0) if fits else 0
        first, asked = asked, asked + need
        ok = fits and (need == 0 or start + asked <= len(free))
        cu.append(min(end, n))
        kv2.append(k + x if ok else k)
        held2.append(max(h, total) if ok else h)
        granted.append(int(ok))
        if ok:
            taken += need
            for j in range(need):
                table[b][h + j] = free[start + first + j]
            for i in range(x):
                pos[row + i] = k + i
                page = table[b][(k + i) // P]
                slot[row + i] = -1 if page < 0 else page * P + (k + i) % P
    return dict(cu_q=cu, kv_lens=kv2, page_counts=held2, granted=granted, positions=pos, slots=slot,
                free_start=[start + taken]), table


PLANS = {
    "one-token": dict(new=[1, 1, 1], kv=[0, 16, 31], held=[0, 1, 2], n=3),
    "chunks": dict(new=[40, 1, 0, 17], kv=[5, 15, 9, 64], held=[1, 1, 1, 4], n=58),
    "padded": dict(new=[2, 3], kv=[14, 0], held=[1, 0], n=11),
    "nothing-new": dict(new=[0, 0], kv=[3, 0], held=[1, 0], n=0),
    "kept-pages-after-a-refusal": dict(new=[3, 20], kv=[15, 30], held=[2, 4], n=23),
    "free-list-runs-out": dict(new=[16, 33, 1, 1], kv=[0, 0, 7, 16], held=[0, 0, 1, 1], n=51, free=2),
    "no-free-page": dict(new=[1, 1], kv=[15, 16], held=[1, 1], n=2, free=0),
    "table-row-too-short": dict(new=[200, 4], kv=[0, 2], held=[0, 1], n=204, width=6),
    "more-rows-than-the-batch": dict(new=[4, 4, 4], kv=[0, 0, 0], held=[0, 0, 0], n=9),
    "negative-lengths": dict(new=[-3, 2], kv=[-1, -7], held=[-2, 0], n=2),
    "one-request": dict(new=[1], kv=[0], held=[0], n=1),
    "no-request": dict(new=[], kv=[], held=[], n=5),
}


def _plan_inputs(c, P, dev, start=2):
    g = torch.Generator().manual_seed(3)
    width, B = c.get("width", 16), len(c["new"])
    pool = torch.randperm(4 * width * max(B, 1) + 64, generator=g).tolist()
    table = [[pool.pop() if j < max(h, 0) else -7 for j in range(width)] for h in c["held"]]
    free = pool[:start + c.get("free", width * max(B, 1))]
    t = torch.tensor(table, dtype=I32).view(B, width).to(dev)
    return table, free, t


def _check_plan(gpu, c, P):
    dev, start = _dev(gpu), 2
    table, free, t = _plan_inputs(c, P, dev, start)
    want, want_table = _plan_oracle(c["new"], c["kv"], c["held"], table, free, start, P, c["n"])
    for _ in range(2):  # the same call again finds the same
        got = paged.plan(_i32(c["new"], dev), _i32(c["kv"], dev), _i32(c["held"], dev), t, _i32(free, dev),
                         _i32([start], dev), P, c["n"])
        for name, v in want.items():
            assert getattr(got, name).tolist() == v, name
        assert t.tolist() == want_table


@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("name", PLANS)
def test_plan_cpu(fake_rt, name, P):
    _check_plan(False, PLANS[name], P)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("name", PLANS)
def test_plan_gpu(gpu_rt, name, P):
    _check_plan(True, PLANS[name], P)


def _random_plan(B, seed, P):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randint(0, 12 * P, (B,), generator=g).tolist()
    new = [int(x) if x < 30 else 0 for x in torch.randint(0, 40, (B,), generator=g)]
    held = [-(-k // P) + int(e) for k, e in zip(kv, torch.randint(0, 2, (B,), generator=g))]
    # an odd batch size, some rows behind the last request
    return dict(new=new, kv=kv, held=held, n=sum(new) + 3, free=sum(-(-x // P) + 1 for x in new) * 2 // 3)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [63, 257, 1000, 4096])
def test_plan_many_requests_gpu(gpu_rt, B):
    """Several requests per thread of the scan, several workgroups, a free list
    that runs out in the middle of the batch."""
    _check_plan(True, _random_plan(B, B, 16), 16)


def test_plan_many_requests_cpu(fake_rt):
    _check_plan(False, _random_plan(300, 5, 16), 16)


def _plan_call(dev, **kw):
    a = dict(new_lens=_i32([1, 2], dev), kv_lens=_i32([3, 4], dev), page_counts=_i32([1, 1], dev),
             block_table=torch.zeros(2, 8, dtype=I32, device=dev), free_pages=_i32([5, 6], dev),
             free_start=_i32([0], dev), page_size=16, n_tokens=3)
    a.update(kw)
    return paged.plan(**a)


def test_plan_refuses(fake_rt):
    _plan_call("cpu")
    wide = torch.zeros(8, 2, dtype=I32)
    for bad in (dict(new_lens=torch.tensor([1, 2])), dict(kv_lens=_i32([3], "cpu")),
                dict(page_counts=torch.zeros(2, 2, dtype=I32)), dict(block_table=wide.t()),
                dict(block_table=torch.zeros(3, 8, dtype=I32)), dict(block_table=torch.zeros(2, 8)),
                dict(free_pages=torch.zeros(2, dtype=torch.int64)), dict(free_start=torch.zeros((), dtype=I32)),
                dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(n_tokens=-1),
                dict(n_tokens=1 << 31), dict(new_lens=torch.zeros(2, dtype=I32, device="meta"))):
        with pytest.raises(ValueError):
            _plan_call("cpu", **bad)
    many = torch.zeros(4097, dtype=I32)
    with pytest.raises(ValueError):
        paged.plan(many, many, many, torch.zeros(4097, 1, dtype=I32), _i32([0], "cpu"), _i32([0], "cpu"), 16, 0)


# ---------------------------------------------------------------- RoPE into pages
def _pool(num, hkv, P, hd, dt, dev, layout):
    """A pool of NaNs: contiguous, one layer of a pool over layers, or heads and
    pages exchanged in memory."""
    if layout == "layer":
        return torch.full((3, 2, num, hkv, P, hd), math.nan, dtype=dt, device=dev)[1]
    if layout == "permuted":
        return torch.full((num, hkv, 2, P, hd), math.nan, dtype=dt, device=dev).permute(2, 0, 1, 3, 4)
    return torch.full((2, num, hkv, P, hd), math.nan, dtype=dt, device=dev)


def _check_rope(gpu, dt, n, hq, hkv, hd, P, layout="contiguous", pad=0):
    dev = _dev(gpu)
    g = torch.Generator().manual_seed(n + hd)
    num, max_pos = -(-max(n, 1) // P) + 2, 4096
    wide = torch.randn(n, (hq + 2 * hkv) * hd + pad, generator=g).to(dt).to(dev)
    qkv = wide[:, :(hq + 2 * hkv) * hd]
    cos, sin = D.rope_tables(hd, max_pos, 500000.0, dev)
    pos = torch.randint(0, max_pos, (n,), generator=g).tolist()
    slots = torch.randperm(num * P, generator=g)[:n].tolist()
    if n > 4:
        pos[1], slots[2], slots[3], pos[4] = -1, -1, num * P + 5, max_pos
    pool = _pool(num, hkv, P, hd, dt, dev, layout)
    q = paged.rope_kv(qkv, cos, sin, pool, _i32(pos, dev), _i32(slots, dev), hq, hkv).cpu()
    assert q.shape == (n, hq, hd) and q.dtype == dt
    want = torch.full((2, num, hkv, P, hd), math.nan, dtype=torch.float64)
    x = qkv.cpu().double().view(n, hq + 2 * hkv, hd)
    # f32 products and a sum of two (2 * 2^-24 of the larger terms' sum), then one rounding
    eps = torch.finfo(dt).eps / 2
    tol = lambda a, b, y: eps * y.abs() + (a.abs() + b.abs()) * 2.0 ** -22 + torch.finfo(dt).tiny * torch.finfo(dt).eps  # noqa: E731
    for t in range(n):
        inside = 0 <= slots[t] < num * P and pos[t] >= 0
        if inside:
            want[1, slots[t] // P, :, slots[t] % P] = x[t, hq + hkv:]
        if pos[t] < 0:
            assert (q[t] == 0).all()
            continue
        if pos[t] >= max_pos:
            assert q[t].isnan().all()
            continue
        a, b = x[t, :hq + hkv, :hd // 2], x[t, :hq + hkv, hd // 2:]
        c, s = cos[pos[t]].double().cpu(), sin[pos[t]].double().cpu()
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
        bound = torch.cat([tol(a, b, r[:, :hd // 2]), tol(a, b, r[:, hd // 2:])], -1)
        assert ((q[t].double() - r[:hq]).abs() <= bound[:hq]).all()
        if inside:
            got = pool[0, slots[t] // P, :, slots[t] % P].cpu().double()
            assert ((got - r[hq:]).abs() <= bound[hq:]).all()
            want[0, slots[t] // P, :, slots[t] % P] = got
    # everything else is as it was
    assert torch.equal(torch.nan_to_num(pool.cpu().double(), nan=1e4), torch.nan_to_num(want, nan=1e4))


ROPES = [(1, 8, 1, 128, 16), (7, 4, 4, 64, 32), (33, 12, 2, 128, 16), (5, 3, 1, 96, 64), (130, 16, 4, 64, 256)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hq,hkv,hd,P", ROPES)
def test_rope_kv_cpu(fake_rt, dt, n, hq, hkv, hd, P):
    _check_rope(False, dt, n, hq, hkv, hd, P)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hq,hkv,hd,P", ROPES)
@pytest.mark.parametrize("layout,pad", [("contiguous", 0), ("layer", 8), ("permuted", 24)])
def test_rope_kv_gpu(gpu_rt, dt, n, hq, hkv, hd, P, layout, pad):
    _check_rope(True, dt, n, hq, hkv, hd, P, layout, pad)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_rope_kv_rounds_as_torch_cpu(fake_rt, dt):
    """Every 16-bit value times a cosine (sine 0, so one f32 product rounded once)."""
    hd, P = 64, 16
    x = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16).view(dt).view(-1, 1, hd // 2)
    n, pages = x.shape[0], torch.zeros(2, 1, 1, P, hd, dtype=dt)
    zero = torch.zeros_like(x)
    for c in (1.0, 0.3712, 2.0 ** -9, 2.0 ** -20, 1.7):
        cos, sin = torch.full((1, hd // 2), c), torch.zeros(1, hd // 2)
        q = paged.rope_kv(torch.cat([x, zero, x, zero, x, zero], 2).view(n, 3 * hd), cos, sin, pages,
                          torch.zeros(n, dtype=I32), torch.full((n,), -1, dtype=I32), 1, 1)
        want = (x.float() * cos).to(dt)
        got = q[:, :, :hd // 2]
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()].view(torch.int16), want[~want.isnan()].view(torch.int16)), c


@pytest.mark.gpu
def test_rope_kv_no_rows_gpu(gpu_rt):
    _check_rope(True, torch.bfloat16, 0, 8, 2, 128, 16)


def test_rope_kv_refuses(fake_rt):
    n, hq, hkv, hd, P = 3, 4, 2, 64, 16
    ok = dict(qkv=torch.zeros(n, (hq + 2 * hkv) * hd, dtype=torch.bfloat16), cos=torch.zeros(8, hd // 2),
              sin=torch.zeros(8, hd // 2), pages=torch.zeros(2, 4, hkv, P, hd, dtype=torch.bfloat16),
              positions=_i32([0, 1, 2], "cpu"), slots=_i32([0, 1, 2], "cpu"), hq=hq, hkv=hkv)
    paged.rope_kv(**ok)
    h = torch.float16
    for bad in (dict(qkv=ok["qkv"].half()), dict(qkv=ok["qkv"][:, :-8]), dict(qkv=ok["qkv"].float()),
                dict(qkv=torch.zeros(n, 516, dtype=torch.bfloat16)[:, 4:]), dict(cos=torch.zeros(8, hd // 2, dtype=h)),
                dict(sin=torch.zeros(9, hd // 2)), dict(cos=torch.zeros(8, hd), sin=torch.zeros(8, hd)),
                dict(positions=_i32([0, 1], "cpu")), dict(slots=torch.zeros(3)), dict(hkv=1), dict(hq=5), dict(hq=0),
                dict(pages=torch.zeros(2, 4, hkv, 24, hd, dtype=torch.bfloat16)),
                dict(pages=torch.zeros(2, 4, hkv, P, hd)), dict(pages=torch.zeros(1, 4, hkv, P, hd, dtype=h)),
                dict(pages=torch.zeros(2, 4, hkv, hd, P, dtype=torch.bfloat16).transpose(3, 4)),
                dict(slots=torch.zeros(3, dtype=I32, device="meta"))):
        with pytest.raises(ValueError):
            paged.rope_kv(**{**ok, **bad})


def test_rope_kv_refuses_overlapping_pages(fake_rt):
    """A pool whose pages share memory is refused where it is written; slices and
    permutations of a larger one are not."""
    n, hq, hkv, hd, P = 2, 2, 2, 64, 16
    ok = dict(qkv=torch.zeros(n, (hq + 2 * hkv) * hd, dtype=torch.bfloat16), cos=torch.zeros(8, hd // 2),
              sin=torch.zeros(8, hd // 2), positions=_i32([0, 1], "cpu"), slots=_i32([0, 1], "cpu"), hq=hq, hkv=hkv)
    flat = torch.zeros(2 * 4 * hkv * P * hd, dtype=torch.bfloat16)
    rows, head, page = P * hd, P * hd, hkv * P * hd
    for kv_s, page_s, head_s in ((4 * page, page, head), (page, 2 * page, head), (rows, 2 * page, 2 * rows)):
        paged.rope_kv(pages=flat.as_strided((2, 2, hkv, P, hd), (kv_s, page_s, head_s, hd, 1)), **ok)
    for kv_s, page_s, head_s in ((0, page, head), (4 * page, 0, head), (4 * page, page, 0), (page, page, head),
                                 (4 * page, page - 8, head), (4 * page, page, head - hd)):
        with pytest.raises(ValueError):
            paged.rope_kv(pages=flat.as_strided((2, 2, hkv, P, hd), (kv_s, page_s, head_s, hd, 1)), **ok)


# ---------------------------------------------------------------- attention
def _requests(ql, kl, P, extra=3, seed=1, width=None):
    """Block table of scattered pages for the lengths; entries behind a request's
    pages lie outside the pool, as does what the table has no page for."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-k // P) for k in kl]
    width = width or max(counts + [0]) + 2
    perm = torch.randperm(sum(counts) + extra, generator=g).tolist()
    table = [[perm.pop() if j < c else (-1 if j % 2 else 1 << 30) for j in range(width)] for c in counts]
    cu = [0]
    for x in ql:
        cu.append(cu[-1] + x)
    return torch.tensor(table, dtype=I32).view(len(kl), width), cu, sum(counts) + extra


def _attn_oracle(q, pool, cu, kl, table, scale):
    """Row by row in f64 -> (result, bound of the error). The bound, to first
    order, with e half a step of the type: e |o| for the output's rounding; for
    the probabilities' rounding and for errors of the scores, which move
    probabilities and their sum, (e + 2 ds + 2^-20) sum p |v|, where ds is
    (hd + 4) f32 roundings of the score's terms and of the exponent."""
    n, hq, hd = q.shape
    hkv, P = pool.shape[2], pool.shape[3]
    g, e = hq // hkv, torch.finfo(q.dtype).eps / 2
    o = torch.full((n, hq, hd), math.nan, dtype=torch.float64)
    tol = torch.zeros(n, hq, hd, dtype=torch.float64)
    for b in range(len(kl)):
        m = cu[b + 1] - cu[b]
        if not m:
            continue
        ids = table[b, :-(-kl[b] // P)].long()
        k, v = (pool[x].double()[ids].transpose(1, 2).reshape(-1, hkv, hd)[:kl[b]] for x in (0, 1))
        for i in range(m):
            see = kl[b] - m + i + 1
            t = cu[b] + i
            if see <= 0:
                o[t] = 0
                continue
            for h in range(hkv):
                qq, kk, vv = q[t, h * g:(h + 1) * g].double(), k[:see, h], v[:see, h]
                s = qq @ kk.T * scale
                p = torch.softmax(s, -1)
                r = p @ vv
                ds = (hd + 4) * 2.0 ** -24 * (qq.abs() @ kk.abs().T * abs(scale)).amax(-1, keepdim=True)
                o[t, h * g:(h + 1) * g] = r
                tol[t, h * g:(h + 1) * g] = 1.05 * (e * r.abs() + (e + 2 * ds + 2.0 ** -20) * (p @ vv.abs())) + \
                    torch.finfo(q.dtype).tiny * e * 2
    return o.view(n, -1), tol.view(n, -1)


def _check_attn(gpu, dt, ql, kl, hq, hkv, hd, P, layout="contiguous", pad=0, hints=True, sharp=1.0, extra_rows=0):
    dev = _dev(gpu)
    g = torch.Generator().manual_seed(hd + P + sum(kl))
    table, cu, num = _requests(ql, kl, P)
    n = cu[-1] + extra_rows
    q = (torch.randn(n, hq, hd + pad, generator=g) * sharp).to(dt)[:, :, :hd]
    pool = _pool(num, hkv, P, hd, dt, "cpu", layout)
    for b, k in enumerate(kl):  # what no request holds stays NaN
        for t in range(k):
            pool[:, table[b, t // P], :, t % P] = torch.randn(2, hkv, hd, generator=g).to(dt)
    want, tol = _attn_oracle(q, pool, cu, kl, table, 1 / math.sqrt(hd))
    kw = hints if isinstance(hints, dict) else dict(max_q=max(ql), max_kv=max(kl)) if hints else {}
    out = torch.full((n, hq * hd), 7.0, dtype=dt, device=dev)
    if gpu:
        q, pool = _like(q, dev), _like(pool, dev)
    got = paged.attention(q, pool, _i32(cu, dev), _i32(kl, dev), table.to(dev), out=out, **kw)
    assert got is out
    got = got.cpu().double()
    assert (got[cu[-1]:] == 7.0).all()  # rows behind the last request
    got, want, tol = got[:cu[-1]], want[:cu[-1]], tol[:cu[-1]]
    worst = ((got - want).abs() / tol.clamp(min=1e-30)).max().item() if want.numel() else 0.0
    assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all(), f"{worst:.2f} of the bound"


def _like(t, dev):
    """t on dev with its strides."""
    r = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev)
    return r.copy_(t)


BATCHES = {
    "one-token": ([1], [1]),
    "one-token-17": ([1], [17]),
    "decode": ([1, 1, 1, 1, 1], [1, 63, 64, 65, 200]),
    "drafts": ([5, 3, 2, 5], [5, 70, 33, 129]),
    "nobody-new": ([0, 1, 0], [0, 40, 12]),
    "prompt": ([100], [100]),
    "chunk-behind-cache": ([37, 61], [165, 61]),
    "mixed": ([1, 70, 1, 9, 0, 1], [90, 70, 1, 140, 3, 31]),
    "more-rows-than-keys": ([4, 6], [2, 0]),
}
SHAPES = [(8, 1, 128, 16), (4, 4, 64, 16), (12, 2, 128, 32), (16, 1, 64, 64), (6, 2, 64, 256), (32, 1, 128, 128)]


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_attention_cpu(fake_rt, name, dt):
    ql, kl = BATCHES[name]
    _check_attn(False, dt, ql, kl, 4, 2, 64, 16, extra_rows=2)


@pytest.mark.gpu
@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("hq,hkv,hd,P", SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_attention_gpu(gpu_rt, name, hq, hkv, hd, P, dt):
    ql, kl = BATCHES[name]
    _check_attn(True, dt, ql, kl, hq, hkv, hd, P, extra_rows=3)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["decode", "drafts", "mixed"])
@pytest.mark.parametrize("layout,pad", [("layer", 8), ("permuted", 64)])
@pytest.mark.parametrize("hints", [False, True])
def test_attention_strides_and_hints_gpu(gpu_rt, name, layout, pad, hints):
    """A strided q, a layer's slice of a pool and a pool with exchanged strides;
    without the host's bounds the result is the same."""
    ql, kl = BATCHES[name]
    _check_attn(True, torch.bfloat16, ql, kl, 8, 2, 128, 16, layout, pad, hints)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql,kl", [([1, 1], [5000, 3001]), ([6, 1], [2049, 4095]), ([300], [700]), ([129, 2], [1500, 2500])])
def test_attention_long_gpu(gpu_rt, dt, ql, kl):
    """Lengths that are split over workgroups, and over several tiles of rows."""
    _check_attn(True, dt, ql, kl, 8, 2, 128, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (16, 2, 64)])
@pytest.mark.parametrize("ql,kl", [([5, 5, 5], [8191, 3003, 777]), ([5, 1, 7], [4200, 4300, 1111]), ([70], [5000])])
def test_attention_split_tiles_gpu(gpu_rt, dt, hq, hkv, hd, ql, kl):
    """More rows than the few-row body takes, over keys that are split: the splits'
    shares of such lengths are not whole 64-key tiles by themselves."""
    _check_attn(True, dt, ql, kl, hq, hkv, hd, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd", [(16, 1, 128), (8, 1, 64), (12, 2, 128)])
@pytest.mark.parametrize("ql,kl,hints", [([1], [20011], True), ([1, 1, 0], [9000, 260, 17000], True),
                                         ([5], [12005], True), ([2, 9], [513, 7777], True),
                                         ([30, 4], [6000, 900], dict(max_q=5, max_kv=6000)),
                                         ([3, 1], [5000, 9000], dict(max_q=3, max_kv=4000))])
def test_attention_joins_many_splits_gpu(gpu_rt, hq, hkv, hd, ql, kl, hints):
    """Keys split so often that several threads join a row; requests that use few of
    the splits; more rows and keys than the bounds that the joining is laid out for."""
    _check_attn(True, torch.bfloat16, ql, kl, hq, hkv, hd, 16, hints=hints)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd", [(32, 32, 64), (64, 16, 128)])
@pytest.mark.parametrize("hints", [False, True])
def test_attention_sorted_tiles_gpu(gpu_rt, hq, hkv, hd, hints):
    """More tiles than CUs: they are taken in the order of their requests' keys, equal
    ones among them, beside requests without tiles."""
    _check_attn(True, torch.bfloat16, [130, 1, 0, 200, 64, 200, 33], [300, 90, 5, 450, 64, 450, 1000], hq, hkv, hd, 16,
                hints=hints, extra_rows=5)


@pytest.mark.gpu
@pytest.mark.parametrize("sharp", [0.0, 30.0])
def test_attention_flat_and_peaked_gpu(gpu_rt, sharp):
    """All scores equal; scores whose maximum moves far from tile to tile."""
    _check_attn(True, torch.float16, [1, 40], [900, 700], 8, 2, 64, 32, sharp=sharp)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(8, 1), (40, 1), (80, 2)])
@pytest.mark.parametrize("B", [70, 300])
def test_attention_many_requests_gpu(gpu_rt, B, hq, hkv):
    """More requests than a wave finds in one round, some without rows; groups of more
    heads than the few-row body takes."""
    g = torch.Generator().manual_seed(B)
    ql = [int(x) if x < 9 else 0 for x in torch.randint(0, 11, (B,), generator=g)]
    ql[B // 3], ql[-1] = 40, 33
    kl = [q + int(x) for q, x in zip(ql, torch.randint(0, 60, (B,), generator=g))]
    _check_attn(True, torch.bfloat16, ql, kl, hq, hkv, 64, 16, extra_rows=1)


def _check_scale(gpu, scale):
    dev = _dev(gpu)
    g = torch.Generator().manual_seed(6)
    for ql, kl in (([1, 3], [70, 9]), ([50], [90])):
        table, cu, num = _requests(ql, kl, 16)
        q = torch.randn(cu[-1], 4, 64, generator=g).half()
        pool = torch.randn(2, num, 2, 16, 64, generator=g).half()
        want, tol = _attn_oracle(q, pool, cu, kl, table, scale)
        # the bound's score term takes the scale's size
        got = paged.attention(q.to(dev), pool.to(dev), _i32(cu, dev), _i32(kl, dev), table.to(dev), scale=scale)
        assert ((got.cpu().double() - want).abs() <= tol.abs()).all()


@pytest.mark.parametrize("scale", [0.3, -0.125, 1e-6])
def test_attention_scale_cpu(fake_rt, scale):
    _check_scale(False, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.3, -0.125, 1e-6])
def test_attention_scale_gpu(gpu_rt, scale):
    _check_scale(True, scale)


def _check_infinite_scores(gpu, m, kv):
    """An infinite k makes a score of plus or minus infinity by the sign of q there:
    NaN, as inf - inf in the softmax, or a key that counts nothing; rows that see
    only the latter are NaN (0 / 0)."""
    dev = _dev(gpu)
    g = torch.Generator().manual_seed(m)
    hq, hd = 2, 64
    table, cu, num = _requests([m], [kv], 16)
    q = torch.randn(m, hq, hd, generator=g).bfloat16()
    q[:, 0, 7] = -1.0
    q[:, 1, 7] = 1.0
    pool = torch.randn(2, num, 1, 16, hd, generator=g).bfloat16()
    at = lambda t: (0, table[0, t // 16], 0, t % 16, 7)  # noqa: E731
    pool[at(kv - m + 1)] = math.inf
    pool[at(kv - 1)] = math.inf
    if kv == m:  # the first row sees one key
        pool[at(0)] = math.inf
    want, tol = _attn_oracle(q, pool, cu, [kv], table, 0.125)
    got = paged.attention(q.to(dev), pool.to(dev), _i32(cu, dev), _i32([kv], dev), table.to(dev)).cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    # ds of such rows is infinite: the score errors of the finite keys, |q| |k| sums of 64 terms, are below 1e-4
    bound = tol.where(torch.isfinite(tol), 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-3) * 5)
    assert ((got - want).abs()[fine] <= bound[fine]).all()


@pytest.mark.parametrize("m,kv", [(3, 3), (4, 40), (40, 70)])
def test_attention_infinite_scores_cpu(fake_rt, m, kv):
    _check_infinite_scores(False, m, kv)


@pytest.mark.gpu
@pytest.mark.parametrize("m,kv", [(3, 3), (4, 40), (40, 70), (70, 70), (3, 900)])
def test_attention_infinite_scores_gpu(gpu_rt, m, kv):
    _check_infinite_scores(True, m, kv)


def _hints_are_only_hints(dev):
    """Bounds below the true lengths cost speed, not keys or rows."""
    g = torch.Generator().manual_seed(9)
    ql, kl, hq, hkv, hd, P = [30, 1, 7], [500, 333, 90], 4, 2, 64, 16
    table, cu, num = _requests(ql, kl, P)
    q = torch.randn(cu[-1], hq, hd, generator=g).bfloat16().to(dev)
    pool = torch.randn(2, num, hkv, P, hd, generator=g).bfloat16().to(dev)
    args = (q, pool, _i32(cu, dev), _i32(kl, dev), table.to(dev))
    want, tol = _attn_oracle(q.cpu(), pool.cpu(), cu, kl, table, 0.125)
    for kw in (dict(max_q=1, max_kv=1), dict(max_q=1), dict(max_q=500, max_kv=10**6), dict(max_kv=0)):
        got = paged.attention(*args, **kw).cpu().double()
        assert ((got - want).abs() <= tol).all(), kw


def test_attention_hints_cpu(fake_rt):
    _hints_are_only_hints("cpu")


@pytest.mark.gpu
def test_attention_hints_gpu(gpu_rt):
    _hints_are_only_hints("cuda")


def _check_hidden_values(gpu, m, kv, hq, hd, dt=torch.bfloat16):
    """NaN and infinities in later tokens reach only the rows that see them."""
    dev = _dev(gpu)
    g = torch.Generator().manual_seed(kv)
    P, hkv = 16, 1
    table, cu, num = _requests([m], [kv], P)
    q = torch.randn(m, hq, hd, generator=g).to(dt)
    pool = _pool(num, hkv, P, hd, dt, "cpu", "contiguous")
    for t in range(kv):
        pool[:, table[0, t // P], :, t % P] = torch.randn(2, hkv, hd, generator=g).to(dt)
    clean, tol = _attn_oracle(q, pool, cu, [kv], table, 1 / math.sqrt(hd))
    clean, tol = clean.view(m, hq, hd), tol.view(m, hq, hd)
    first = kv - m
    # token -> what its v holds (and, for the last two, its k)
    places = {first + m // 2: [(1, 3, math.inf)], first + m // 2 + 1: [(1, 5, -math.inf), (1, 3, -math.inf)],
              kv - 2: [(1, 0, math.nan)], kv - 1: [(0, 0, math.nan)]}
    for t, what in places.items():
        for x, d, val in what:
            pool[x, table[0, t // P], 0, t % P, d] = val
    got = paged.attention(q.to(dev), pool.to(dev), _i32(cu, dev), _i32([kv], dev), table.to(dev)).cpu().double()
    got = got.view(m, hq, hd)
    for i in range(m):
        seen = set()
        nan_row = False
        special = {}
        for t, what in places.items():
            if t > first + i:
                continue
            for x, d, val in what:
                if x == 0:
                    nan_row = True
                else:
                    special.setdefault(d, []).append(val)
        if nan_row:
            assert got[i].isnan().all(), i
            continue
        for d in range(hd):
            col = got[i, :, d]
            if d in special:
                total = sum(special[d])  # inf + -inf = NaN, as in the sum
                assert col.isnan().all() if math.isnan(total) else (col == total).all(), (i, d)
            else:
                assert ((col - clean[i, :, d]).abs() <= tol[i, :, d]).all(), (i, d)


@pytest.mark.parametrize("m,kv", [(5, 40), (20, 20)])
def test_attention_hidden_values_cpu(fake_rt, m, kv):
    _check_hidden_values(False, m, kv, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq", [1, 8])
@pytest.mark.parametrize("m,kv", [(4, 4), (5, 40), (6, 600), (20, 20), (70, 150), (200, 333)])
def test_attention_hidden_values_gpu(gpu_rt, m, kv, hq, hd):
    _check_hidden_values(True, m, kv, hq, hd)


def _bad_pages(dev):
    """Rows that need a page outside the pool, or more pages than the table row
    has, are NaN; the others of the batch are right."""
    g = torch.Generator().manual_seed(2)
    ql, kl, hq, hkv, hd, P = [1, 3, 1, 2], [40, 50, 10, 33], 4, 2, 64, 16
    table, cu, num = _requests(ql, kl, P)
    q = torch.randn(cu[-1], hq, hd, generator=g).bfloat16()
    pool = torch.randn(2, num, hkv, P, hd, generator=g).bfloat16()
    want, tol = _attn_oracle(q, pool, cu, kl, table, 0.125)
    args = (q.to(dev), pool.to(dev), _i32(cu, dev))

    def rows(kl2, table2):
        return paged.attention(*args, _i32(kl2, dev), table2.to(dev)).cpu().double()

    for bad in (-1, num, 2**31 - 1, -(2**31)):
        t = table.clone()
        t[1, 1] = bad
        got = rows(kl, t)
        assert got[1:4].isnan().all()
        for r in (slice(0, 1), slice(4, 7)):
            assert ((got[r] - want[r]).abs() <= tol[r]).all()
    cap = table.shape[1] * P
    for length in (cap + 1, 2**31 - 1):
        got = rows([40, length, 10, 33], table)
        assert got[1:4].isnan().all() and ((got[0] - want[0]).abs() <= tol[0]).all()
        assert ((got[4:] - want[4:]).abs() <= tol[4:]).all()
    got = rows([40, -5, 10, 33], table)
    assert (got[1:4] == 0).all() and ((got[4:] - want[4:]).abs() <= tol[4:]).all()
    # row bounds outside q are cut to it
    got = paged.attention(args[0], args[1], _i32([-4, 1, 4, 5, 100], dev), _i32(kl, dev), table.to(dev))
    assert got.shape == (cu[-1], hq * hd)


def test_attention_bad_pages_cpu(fake_rt):
    _bad_pages("cpu")


@pytest.mark.gpu
def test_attention_bad_pages_gpu(gpu_rt):
    _bad_pages("cuda")


@pytest.mark.gpu
def test_attention_far_pages_gpu(gpu_rt):
    """Pages beyond 2^32 elements of the pool."""
    hkv, P, hd = 8, 256, 128
    num = (1 << 32) // (hkv * P * hd) + 40
    pool = torch.empty(2, num, hkv, P, hd, dtype=torch.bfloat16, device="cuda")
    ql, kl = [1, 40], [700, 300]
    ids = [num - 1, num - 7, 3, num - 2, num - 30]
    table = torch.tensor([ids[:3], ids[3:] + [0]], dtype=I32)
    pool[:, ids] = torch.randn(2, 5, hkv, P, hd, device="cuda").bfloat16()
    q = torch.randn(41, 16, hd, device="cuda").bfloat16()
    cu = [0, 1, 41]
    got = paged.attention(q, pool, _i32(cu, "cuda"), _i32(kl, "cuda"), table.cuda()).cpu().double()
    small = pool[:, ids].cpu()
    want, tol = _attn_oracle(q.cpu(), small, cu, kl, torch.tensor([[0, 1, 2], [3, 4, 0]]), 1 / math.sqrt(hd))
    assert ((got - want).abs() <= tol).all()
    # and the append finds them
    cos, sin = D.rope_tables(hd, 8, 500000.0, "cuda")
    qkv = torch.randn(2, (16 + 2 * hkv) * hd, device="cuda").bfloat16()
    paged.rope_kv(qkv, cos, sin, pool, _i32([0, 0], "cuda"), _i32([(num - 1) * P + 5, 1], "cuda"), 16, hkv)
    assert torch.equal(pool[1, num - 1, :, 5].flatten(), qkv[0, (16 + hkv) * hd:])
    assert torch.equal(pool[0, num - 1, :, 5].flatten(), qkv[0, 16 * hd:(16 + hkv) * hd])


def test_attention_refuses(fake_rt):
    hq, hkv, hd, P, dt = 4, 2, 64, 16, torch.bfloat16
    ok = dict(q=torch.zeros(3, hq, hd, dtype=dt), pages=torch.zeros(2, 4, hkv, P, hd, dtype=dt),
              cu_q=_i32([0, 1, 3], "cpu"), kv_lens=_i32([5, 7], "cpu"), block_table=torch.zeros(2, 2, dtype=I32))
    paged.attention(**ok)
    for bad in (dict(q=torch.zeros(3, 3, hd, dtype=dt)), dict(q=ok["q"].half()), dict(q=torch.zeros(3, hq * hd, dtype=dt)),
                dict(q=torch.zeros(3, hd, hq, dtype=dt).transpose(1, 2)), dict(q=torch.zeros(3, hq, 68, dtype=dt)[..., 4:]),
                dict(q=torch.zeros(3, hq, 128, dtype=dt)),
                dict(q=torch.zeros(3, hq, 32, dtype=dt), pages=torch.zeros(2, 4, hkv, P, 32, dtype=dt)),
                dict(pages=ok["pages"].float()), dict(pages=ok["pages"][:, :0]), dict(cu_q=_i32([0, 1], "cpu")),
                dict(cu_q=torch.tensor([0, 1, 3])), dict(kv_lens=torch.zeros(2)), dict(block_table=torch.zeros(2, 2)),
                dict(block_table=torch.zeros(1, 2, dtype=I32)), dict(block_table=torch.zeros(2, 0, dtype=I32)),
                dict(out=torch.zeros(3, hq * hd)), dict(out=torch.zeros(2, hq * hd, dtype=dt)),
                dict(out=torch.zeros(hq * hd, 3, dtype=dt).t()),
                dict(kv_lens=torch.zeros(2, dtype=I32, device="meta")), dict(scale=0.0), dict(scale=math.inf),
                dict(scale=math.nan)):
        with pytest.raises(ValueError):
            paged.attention(**{**ok, **bad})


@pytest.mark.gpu
def test_refuses_cpu_tensors_on_the_gpu_backend(gpu_rt):
    with pytest.raises(ValueError):
        _plan_call("cpu")
    with pytest.raises(ValueError):
        _plan_call("cuda", kv_lens=_i32([3, 4], "cpu"))


# ---------------------------------------------------------------- together
class _Server:
    """Requests over one pool: a step is plan, then rope_kv and attention per
    layer (here one), lengths and pages kept on the device."""

    def __init__(self, dev, B, hq, hkv, hd, P, pages):
        self.dev, self.P, self.hq, self.hkv = dev, P, hq, hkv
        self.pool = torch.full((2, pages, hkv, P, hd), math.nan, dtype=torch.bfloat16, device=dev)
        self.cos, self.sin = D.rope_tables(hd, 512, 500000.0, dev)
        self.table = torch.full((B, 16), -1, dtype=I32, device=dev)
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).to(I32).to(dev)
        self.kv, self.counts, self.start = (torch.zeros(n, dtype=I32, device=dev) for n in (B, B, 1))

    def step(self, new, qkv):
        p = paged.plan(new, self.kv, self.counts, self.table, self.free, self.start, self.P, qkv.shape[0])
        self.kv.copy_(p.kv_lens)
        self.counts.copy_(p.page_counts)
        self.start.copy_(p.free_start)
        q = paged.rope_kv(qkv, self.cos, self.sin, self.pool, p.positions, p.slots, self.hq, self.hkv)
        out = torch.zeros(qkv.shape[0], q.shape[1] * q.shape[2], dtype=q.dtype, device=self.dev)
        return paged.attention(q, self.pool, p.cu_q, self.kv, self.table, out=out), p


def _check_together(gpu):
    """Prompts, decodes and drafts that are taken back, against the contiguous-cache
    ops run for each request alone, token by token."""
    dev = _dev(gpu)
    g = torch.Generator().manual_seed(4)
    B, hq, hkv, hd = 3, 8, 2, 64
    srv = _Server(dev, B, hq, hkv, hd, 16, 24)
    caches = [torch.zeros(2, 1, hkv, 64, hd, dtype=torch.bfloat16, device=dev) for _ in range(B)]
    length = [0] * B
    for new, kept in (([20, 0, 3], None), ([1, 5, 1], None), ([4, 4, 4], [1, 4, 2]), ([1, 1, 1], None), ([3, 17, 2], None)):
        qkv = torch.randn(sum(new), (hq + 2 * hkv) * hd, generator=g).bfloat16().to(dev)
        got, plan = srv.step(_i32(new, dev), qkv)
        assert plan.granted.tolist() == [1] * B
        row = 0
        for b in range(B):
            for _ in range(new[b]):
                q = fused.rope_kv(qkv[row:row + 1], srv.cos[length[b]], srv.sin[length[b]], caches[b], length[b], hq, hkv)
                length[b] += 1
                want = fused.attention(q, caches[b], length[b])
                # two results of the same inputs, each within (2^-8 of itself and of sum p |v|) of the truth; |v| < 5
                torch.testing.assert_close(got[row:row + 1].float(), want.float(), rtol=2 ** -7, atol=2 ** -7 * 5)
                row += 1
        assert srv.kv.tolist() == length
        if kept:  # all but the first `kept` of the new tokens are taken back; their pages stay with the request
            length = [n - x + k for n, x, k in zip(length, new, kept)]
            srv.kv.copy_(_i32(length, dev))
    held = [t for row, c in zip(srv.table.tolist(), srv.counts.tolist()) for t in row[:c]]
    assert len(set(held)) == len(held) == srv.start.item()
    # what the pool holds is what the contiguous caches hold
    for b in range(B):
        for t in range(length[b]):
            assert torch.equal(srv.pool[:, srv.table[b, t // 16], :, t % 16], caches[b][:, 0, :, t])


def test_together_cpu(fake_rt):
    _check_together(False)


@pytest.mark.gpu
def test_together_gpu(gpu_rt):
    _check_together(True)


@pytest.mark.gpu
def test_captured_step_gpu(gpu_rt):
    """A captured step (plan, append, attention, verification) replayed over changing
    lengths, eager work between the replays, gives the eager step's results; two
    captured graphs share nothing."""
    B, hq, hkv, hd, P, K, V = 4, 8, 2, 128, 16, 2, 1000
    n = B * (K + 1)
    g = torch.Generator(device="cuda").manual_seed(5)
    probs = torch.softmax(torch.randn(B, K + 1, V, device="cuda", generator=g), -1)

    def inputs():
        return (torch.randn(n, (hq + 2 * hkv) * hd, device="cuda", generator=g).bfloat16(),
                torch.randint(0, V, (B, K), device="cuda", generator=g, dtype=I32),
                torch.rand(B, K, device="cuda", generator=g) * 0.01, torch.rand(B, device="cuda", generator=g))

    def step(srv, new, qkv, drafts, u, u_last):
        out, plan = srv.step(new, qkv)
        tokens, accepted = speculative.verify_draft(probs, None, drafts, u, u_last)
        srv.kv.sub_(new).add_(accepted + 1)
        return out, tokens, accepted, plan.slots

    new = torch.full((B,), K + 1, dtype=I32, device="cuda")
    made = []
    for _ in range(2):
        srv, held = _Server("cuda", B, hq, hkv, hd, P, 64), [t.clone() for t in inputs()]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(srv, new, *held)
        torch.cuda.current_stream().wait_stream(s)
        for t in (srv.kv, srv.counts, srv.start):
            t.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(srv, new, *held)
        made.append((graph, srv, held, outs, _Server("cuda", B, hq, hkv, hd, P, 64)))
    for turn in range(6):
        fresh = [inputs() for _ in made]
        for (graph, _, held, _, _), x in zip(made, fresh):
            for t, v in zip(held, x):
                t.copy_(v)
            graph.replay()
        for (_, srv, _, outs, eager), x in zip(made, fresh):
            want = step(eager, new, *x)
            for a, b in zip(outs, want):
                assert torch.equal(a, b), turn
            assert torch.equal(srv.kv, eager.kv) and torch.equal(srv.table, eager.table)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_captured_padded_batch_gpu(gpu_rt):
    """One captured call over a padded batch, replayed over other divisions of its rows:
    single tokens, drafts, a chunk, rows of nobody (left as they were)."""
    g = torch.Generator().manual_seed(21)
    n, hq, hkv, hd, P, dt = 200, 16, 2, 128, 16, torch.bfloat16
    q = torch.randn(n, hq, hd, generator=g).to(dt)
    batches = [([1, 1, 1, 1], [900, 3, 2000, 64]), ([100, 1, 0, 90], [1500, 17, 40, 90]), ([5, 3, 190, 2], [700, 3, 2047, 2]),
               ([0, 0, 0, 0], [5, 0, 9, 1]), ([1, 0, 1, 0], [1, 0, 2048, 7])]
    table, _, num = _requests([1] * 4, [2048] * 4, P)
    pool = torch.randn(2, num, hkv, P, hd, generator=g).to(dt)
    qd, pd, td = q.cuda(), pool.cuda(), table.cuda()
    cu, kv = _i32([0] * 5, "cuda"), _i32([0] * 4, "cuda")
    out = torch.zeros(n, hq * hd, dtype=dt, device="cuda")

    def call():
        return paged.attention(qd, pd, cu, kv, td, out=out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for ql, kl in batches + batches[::-1]:
        c = [sum(ql[:i]) for i in range(5)]
        cu.copy_(_i32(c, "cuda"))
        kv.copy_(_i32(kl, "cuda"))
        out.fill_(7.0)
        graph.replay()
        got = out.cpu().double()
        assert (got[c[-1]:] == 7.0).all()
        if c[-1]:
            want, tol = _attn_oracle(q[:c[-1]], pool, c, kl, table, 1 / math.sqrt(hd))
            assert ((got[:c[-1]] - want).abs() <= tol).all(), (ql, kl)
        out.fill_(9.0)
        call()
        assert torch.equal(out.cpu().double()[:c[-1]], got[:c[-1]])


@pytest.mark.gpu
def test_two_streams_gpu(gpu_rt):
    """Calls on two streams at once do not share a workspace."""
    g = torch.Generator().manual_seed(8)
    ql, kl, hq, hkv, hd, P = [1, 1], [6000, 5000], 8, 1, 128, 16
    table, cu, num = _requests(ql, kl, P)
    sets = []
    for _ in range(2):
        q = torch.randn(2, hq, hd, generator=g).bfloat16()
        pool = torch.randn(2, num, hkv, P, hd, generator=g).bfloat16()
        sets.append((_attn_oracle(q, pool, cu, kl, table, 1 / math.sqrt(hd)), q.cuda(), pool.cuda()))
    cud, kld, td = _i32(cu, "cuda"), _i32(kl, "cuda"), table.cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged.attention(sets[i][1], sets[i][2], cud, kld, td))
    torch.cuda.synchronize()
    for ((want, tol), _, _), outs in zip(sets, got):
        for o in outs:
            assert ((o.cpu().double() - want).abs() <= tol).all()
