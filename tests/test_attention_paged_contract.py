"""What the paged serving ops promise beyond a result within the types' rounding
(tests/test_attention_paged.py holds the forms they are compared with)."""
from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

from ogkm.ops import decode as D
from ogkm.ops import paged
from test_attention_paged import _attn_oracle, _dev, _i32, _requests


# ---------------------------------------------------------------- bits of the probabilities
def _check_probability_bits(gpu, dt, ql, kl, hq, hkv, hd, P, chunk=0):
    """Single tokens, and drafts where no request of the batch has more than 32 rows per
    kv head, keep more of a probability than the type's bits (`chunk` rows at the
    batch's start are not looked at). Every second key is 0 and has v = 1, the others score ln(1 - eps / 4) and have
    v = -1: of the type's steps below 1 (eps / 2) that probability is in the middle
    between two, and what it is rounded by is as large as the result, which is the
    difference of the two. Even lengths, so that the pairs cancel."""
    dev, eps = _dev(gpu), torch.finfo(dt).eps
    e, scale = eps / 2, -math.log(1 - eps / 4)
    table, cu, num = _requests(ql, kl, P)
    q = torch.zeros(cu[-1], hq, hd, dtype=dt)
    q[:, :, 0] = 1
    pool = torch.zeros(2, num, hkv, P, hd, dtype=dt)
    pool[0, :, :, 1::2, 0] = -1
    pool[1, :, :, ::2], pool[1, :, :, 1::2] = 1, -1
    want, _ = _attn_oracle(q, pool, cu, kl, table, scale)
    # The bound, to first order, with p of a pair below 1 and |v| = 1: e |o| for the
    # output's rounding, e^2 for a probability in two parts, (hd + 4) f32 roundings of a
    # score of at most `scale`, and 2^-20 for the exponent (f32 near the 8 that fp16's
    # probabilities are raised by: 2^-22), the exponential and the sums.
    tol = 1.05 * (e * want.abs() + e * e + 2 * (hd + 4) * 2.0 ** -24 * scale + 2.0 ** -20)
    got = paged.attention(q.to(dev), pool.to(dev), _i32(cu, dev), _i32(kl, dev), table.to(dev), max_q=max(ql),
                          max_kv=max(kl), scale=scale).cpu().double()
    got, want, tol = got[chunk:], want[chunk:], tol[chunk:]
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


BITS = [([1], [2]), ([1, 1, 1], [64, 700, 2]), ([1, 1], [2046, 900])]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql,kl", BITS)
def test_probability_bits_cpu(fake_rt, dt, ql, kl):
    _check_probability_bits(False, dt, ql, kl, 8, 2, 64, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (4, 4, 64), (24, 1, 64), (64, 2, 128)])
@pytest.mark.parametrize("ql,kl", BITS)
def test_probability_bits_gpu(gpu_rt, dt, hq, hkv, hd, ql, kl):
    """One and two column blocks, four and eight waves, keys split and not."""
    _check_probability_bits(True, dt, ql, kl, hq, hkv, hd, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql,kl,chunk", [([3, 4], [601, 88], 0), ([70, 1, 1], [70, 800, 2000], 70)])
def test_probability_bits_of_drafts_and_beside_a_chunk_gpu(gpu_rt, dt, ql, kl, chunk):
    _check_probability_bits(True, dt, ql, kl, 8, 1, 128, 16, chunk)


# ---------------------------------------------------------------- the documented step
def _documented_step():
    """The server's step as README.md gives it."""
    text = (Path(__file__).resolve().parents[1] / "README.md").read_text()
    return next(c for c in re.findall(r"```python\n(.*?)```", text, re.S) if "verify_draft" in c)


class _Layer:
    def __init__(self, pages):
        self.pages = pages

    def qkv(self, x):
        return x

    def rest(self, x, out):
        self.out = out
        return x


# Of each request: new tokens, drafts among them, how many of those the target keeps. Request 2
# wants more pages than there are until the last step, and its rows are cached all the while.
STEPS = [([4, 40, 3], [3, 0, 2], [1, 0, 2]), ([1, 3, 400], [0, 2, 0], [0, 0, 0]), ([5, 1, 400], [4, 0, 0], [4, 0, 0]),
         ([2, 5, 30], [1, 4, 0], [0, 2, 0])]
GRANTED = [[1, 1, 1], [1, 1, 0], [1, 1, 0], [1, 1, 1]]


class _Loop:
    """State that the documented step runs on, static, so that a captured step finds it again."""

    def __init__(self, dev, n):
        B, K, V, hq, hkv, hd, P = 3, 4, 50, 4, 2, 64, 16
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        self.B, self.K, self.V, self.P, self.hkv = B, K, V, P, hkv
        layer = _Layer(torch.full((2, 16, hkv, P, hd), math.nan, dtype=torch.bfloat16, device=dev))
        cos, sin = D.rope_tables(hd, 1024, 500000.0, dev)
        self.s = dict(new_lens=z(B), kv_lens=z(B), page_counts=z(B), block_table=z(B, 32) - 1,
                      free_pages=torch.arange(15, -1, -1, dtype=torch.int32).to(dev), free_start=z(1), counts=z(B),
                      x=torch.zeros(n, (hq + 2 * hkv) * hd, dtype=torch.bfloat16, device=dev), drafts=z(B, K),
                      probs=torch.zeros(B, K + 1, V, device=dev), u=torch.full((B, K), 0.5, device=dev),
                      u_last=torch.zeros(B, device=dev))
        self.fixed = dict(layers=[layer], cos=cos, sin=sin, page_size=P, n_tokens=n, hq=hq, hkv=hkv, max_q=n,
                          max_kv=512, draft_probs=None)
        self.code = compile(_documented_step(), "README.md", "exec")

    def call(self):
        env = {**self.s, **self.fixed}
        exec(self.code, env)
        for name in ("kv_lens", "page_counts", "free_start"):
            self.s[name].copy_(env[name])
        return env["plan"].granted, env["accepted"]

    def feed(self, step, g):
        """Inputs of a step: random rows; probabilities that keep the said number of drafts."""
        new, drafts, kept = step
        x = torch.randn(self.s["x"].shape, generator=g).bfloat16()
        self.s["x"].copy_(x)
        self.s["new_lens"].copy_(torch.tensor(new, dtype=torch.int32))
        self.s["counts"].copy_(torch.tensor(drafts, dtype=torch.int32))
        self.s["drafts"].copy_(torch.arange(self.B * self.K, dtype=torch.int32).view(self.B, self.K))
        p = torch.zeros(self.B, self.K + 1, self.V)
        p[:, :, -1] = 1
        for b in range(self.B):
            for j in range(kept[b]):
                p[b, j] = 0
                p[b, j, b * self.K + j] = 1
        self.s["probs"].copy_(p)
        return x

    def check(self, lens, rows):
        """Lengths, and v of every cached token, which is stored as it came."""
        assert self.s["kv_lens"].tolist() == lens
        pool, table = self.fixed["layers"][0].pages.cpu(), self.s["block_table"].tolist()
        for b, r in enumerate(rows):
            for t, v in enumerate(r):
                assert torch.equal(pool[1, table[b][t // self.P], :, t % self.P].flatten(), v), (b, t)


def _run_documented_steps(loop, call, g):
    lens, rows, width = [0] * 3, [[] for _ in range(3)], loop.s["x"].shape[1]
    for step, granted in zip(STEPS, GRANTED):
        x = loop.feed(step, g)
        got, accepted = call()
        assert got.tolist() == granted
        at = 0
        for b, (new, drafts, kept) in enumerate(zip(*step)):
            if granted[b]:
                take = new - drafts + kept
                rows[b] += list(x[at:at + take, width - loop.hkv * 64:])
                lens[b] += take
                assert accepted.tolist()[b] == kept
            at += new
        loop.check(lens, rows)


def test_documented_step_cpu(fake_rt):
    """Drafts, prompt chunks and requests without pages in one batch: a refused
    request keeps its length and its rows, a chunk keeps all of its own."""
    _run_documented_steps(loop := _Loop("cpu", 410), loop.call, torch.Generator().manual_seed(2))


@pytest.mark.gpu
def test_documented_step_captured_gpu(gpu_rt):
    """The same as one captured step, replayed."""
    loop = _Loop("cuda", 410)
    start = {k: v.clone() for k, v in loop.s.items()}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loop.call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = loop.call()
    for turn in range(3):
        for k, v in start.items():
            loop.s[k].copy_(v)

        def call():
            graph.replay()
            return outs

        _run_documented_steps(loop, call, torch.Generator().manual_seed(turn))


# ---------------------------------------------------------------- who gets pages
def _granted(gpu, new, kv, held, free, width=40):
    dev, B = _dev(gpu), len(new)
    p = paged.plan(_i32(new, dev), _i32(kv, dev), _i32(held, dev), torch.zeros(B, width, dtype=torch.int32, device=dev),
                   torch.arange(100, 100 + free, dtype=torch.int32).to(dev), _i32([0], dev), 16, sum(new))
    return p.granted.tolist(), p.page_counts.tolist(), p.free_start.tolist()


def _check_refusals(gpu):
    # 25 pages of 10: the single pages behind it are not handed out either
    assert _granted(gpu, [400, 1, 1], [0, 16, 0], [0, 1, 0], 10) == ([0, 0, 0], [0, 1, 0], [0])
    # a request that lacks none is not concerned
    assert _granted(gpu, [400, 1, 1], [0, 7, 0], [0, 1, 0], 10) == ([0, 1, 0], [0, 1, 0], [0])
    # behind the running ones, or left out, it stops nobody
    assert _granted(gpu, [1, 1, 400], [16, 0, 0], [1, 0, 0], 10) == ([1, 1, 0], [2, 1, 0], [2])
    assert _granted(gpu, [0, 1, 1], [0, 16, 0], [0, 1, 0], 10) == ([1, 1, 1], [0, 2, 1], [2])
    # nor does one that its table row has no room for
    assert _granted(gpu, [400, 1, 1], [0, 16, 0], [0, 1, 0], 10, width=4) == ([0, 1, 1], [0, 2, 1], [2])


def test_a_refused_request_keeps_its_place_cpu(fake_rt):
    _check_refusals(False)


@pytest.mark.gpu
def test_a_refused_request_keeps_its_place_gpu(gpu_rt):
    _check_refusals(True)


# ---------------------------------------------------------------- row bounds
def _check_row_bounds(gpu, n, raw, cut, kl, hq, hkv, hd):
    """Row bounds outside q are cut to it: the same results as with `cut`, and rows that
    belong to no request stay as they were."""
    dev, dt, g = _dev(gpu), torch.bfloat16, torch.Generator().manual_seed(n)
    table, _, num = _requests([1] * len(kl), kl, 16)
    q = torch.randn(n, hq, hd, generator=g).to(dt)
    pool = torch.randn(2, num, hkv, 16, hd, generator=g).to(dt)
    want, tol = torch.full((n, hq * hd), 7.0, dtype=torch.float64), torch.zeros(n, hq * hd, dtype=torch.float64)
    for b, (lo, hi) in enumerate(cut):
        if lo == hi:
            continue
        w, t = _attn_oracle(q[lo:hi], pool, [0, hi - lo], [kl[b]], table[b:b + 1], 1 / math.sqrt(hd))
        want[lo:hi], tol[lo:hi] = w, t
    for hints in ({}, dict(max_q=n, max_kv=max(kl)), dict(max_q=1, max_kv=1)):
        out = torch.full((n, hq * hd), 7.0, dtype=dt, device=dev)
        got = paged.attention(q.to(dev), pool.to(dev), _i32(raw, dev), _i32(kl, dev), table.to(dev), out=out, **hints)
        assert ((got.cpu().double() - want).abs() <= tol).all(), hints


# rows of q, bounds as given, rows of each request after the cut, lengths
BOUNDS = [
    (7, [-4, 1, 4, 5, 100], [(0, 1), (1, 4), (4, 5), (5, 7)], [40, 50, 10, 33]),
    (7, [5, 2, 7], [(5, 5), (2, 7)], [40, 50]),  # falling: the first request has no rows, rows 0 and 1 nobody
    (7, [2, 3, 3, 4], [(2, 3), (3, 3), (3, 4)], [9, 50, 64]),
    (90, [-2**31, 1, 80, 2**31 - 1], [(0, 1), (1, 80), (80, 90)], [300, 100, 700]),
    (90, [60, 50, 90], [(60, 60), (50, 90)], [40, 90]),
]


@pytest.mark.parametrize("n,raw,cut,kl", BOUNDS)
def test_row_bounds_cpu(fake_rt, n, raw, cut, kl):
    _check_row_bounds(False, n, raw, cut, kl, 4, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 64), (16, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("n,raw,cut,kl", BOUNDS)
def test_row_bounds_gpu(gpu_rt, n, raw, cut, kl, hq, hkv, hd):
    _check_row_bounds(True, n, raw, cut, kl, hq, hkv, hd)


# ---------------------------------------------------------------- infinities that every row sees
def _check_seen_infinities(gpu, dt, m, kv, hq, hkv, hd):
    """V with infinities or NaN in early tokens: each row's result is that value in its
    dim (NaN where both signs meet), and the other dims are right. Scores stay within
    a few units, so no weight is lost in f32."""
    dev, g = _dev(gpu), torch.Generator().manual_seed(m + kv)
    table, cu, num = _requests([m], [kv], 16)
    q = torch.randn(m, hq, hd, generator=g).to(dt)
    pool = torch.randn(2, num, hkv, 16, hd, generator=g).to(dt)
    want, tol = _attn_oracle(q, pool, cu, [kv], table, 1 / math.sqrt(hd))
    want = want.view(m, hq, hd)
    inf = math.inf
    for t, d, v, total in ((5, 3, inf, inf), (1, hd - 1, -inf, -inf), (0, 7, inf, math.nan), (6, 7, -inf, math.nan),
                           (2, 9, math.nan, math.nan), (3, 11, inf, inf), (4, 11, inf, inf)):
        pool[1, table[0, 0], :, t, d] = v
        want[:, :, d] = total
    want = want.view(m, hq * hd)
    got = paged.attention(q.to(dev), pool.to(dev), _i32(cu, dev), _i32([kv], dev), table.to(dev)).cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    fine = torch.isfinite(want)
    assert ((got - want).abs()[fine] <= tol[fine]).all()


SEEN = [(1, 7), (1, 300), (3, 70), (4, 1500), (40, 200), (150, 900)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,kv", SEEN[:4])
def test_seen_infinities_cpu(fake_rt, dt, m, kv):
    _check_seen_infinities(False, dt, m, kv, 4, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 4, 64), (8, 1, 128), (24, 1, 64)])
@pytest.mark.parametrize("m,kv", SEEN)
def test_seen_infinities_gpu(gpu_rt, dt, m, kv, hq, hkv, hd):
    _check_seen_infinities(True, dt, m, kv, hq, hkv, hd)
