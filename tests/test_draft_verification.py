"""verify_draft (csrc/kernels/speculative.hip; csrc/core/paged_ref.cpp) against its
definition in f64, and its refusals."""
from __future__ import annotations

import math

import pytest
import torch

from ogkm.ops import speculative

I32 = torch.int32


def _oracle(p, q, tokens, u, u_last, counts):
    """(tokens, accepted), sums exact (math.fsum) so that only a border that no
    order of f64 sums could tell would be open."""
    B, K, V = p.shape[0], p.shape[1] - 1, p.shape[2]
    out, acc = [], []
    for b in range(B):
        count = K if counts is None else min(max(counts[b], 0), K)
        m = 0
        while m < count:
            x = tokens[b][m]
            if not 0 <= x < V:
                break
            qt = 1.0 if q is None else q[b, m, x].item()
            if not u[b][m] * qt < p[b, m, x].item():
                break
            m += 1
        row = [max(x, 0.0) if x == x else 0.0 for x in p[b, m].tolist()]
        if m < count:
            qr = [float(i == tokens[b][m]) for i in range(V)] if q is None else q[b, m].tolist()
            rest = [max(x - max(y, 0.0), 0.0) if x == x and y == y else 0.0 for x, y in zip(row, qr)]
        else:
            rest = row
        if not any(rest):
            rest = row
        aim, run, pick = u_last[b] * math.fsum(rest), 0.0, -1
        total = []
        for i, w in enumerate(rest):
            if w > 0:
                total.append(w)
                pick = i
                run += w
                if run > aim:
                    break
        out.append([tokens[b][j] if j < m else pick if j == m else -1 for j in range(K + 1)])
        acc.append(m)
    return out, acc


def _check(gpu, B, K, V, dt, certain=False, ragged=False, seed=0, change=None, layout="contiguous", u_scale=1.0):
    dev = "cuda" if gpu else "cpu"
    g = torch.Generator().manual_seed(seed + V + K)
    logits = torch.randn(B, K + 1, V, generator=g) * 2
    p = torch.softmax(logits, -1).to(dt)
    q = torch.softmax(logits[:, :K] + torch.randn(B, K, V, generator=g) * 0.5, -1).to(dt)
    tokens = torch.stack([torch.multinomial(q[b].float().reshape(-1, V), 1, generator=g)[:, 0] for b in range(B)]).to(I32) \
        if B and K else torch.zeros(B, K, dtype=I32)
    u, u_last = torch.rand(B, K, generator=g) * u_scale, torch.rand(B, generator=g)
    counts = torch.randint(-1, K + 3, (B,), generator=g, dtype=I32) if ragged else None
    if change:
        change(p, q, tokens, u, u_last)
    want = _oracle(p, None if certain else q, tokens.tolist(), u.tolist(), u_last.tolist(),
                   counts.tolist() if ragged else None)
    if layout == "strided":
        p = torch.cat([p, p], -1)[..., :V]
        q = torch.stack([q, q], 2)[:, :, 1]
    to = lambda t: None if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)  # noqa: E731
    got = speculative.verify_draft(to(p), None if certain else to(q), to(tokens), to(u), to(u_last), to(counts))
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    return want


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 4, 50), (2, 0, 33), (0, 2, 9), (5, 3, 5000)])
def test_verify_cpu(fake_rt, dt, certain, B, K, V):
    _check(False, B, K, V, dt, certain, ragged=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("layout", ["contiguous", "strided"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 4, 50), (2, 0, 33), (0, 2, 9), (5, 3, 4095), (4, 2, 4096), (4, 5, 4097),
                                   (7, 8, 20001), (2, 70, 301)])
def test_verify_gpu(gpu_rt, dt, certain, layout, B, K, V):
    _check(True, B, K, V, dt, certain, ragged=True, layout=layout)
    _check(True, B, K, V, dt, certain, seed=1, layout=layout, u_scale=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_verify_whole_vocabulary_gpu(gpu_rt, dt):
    """The Llama-3 vocabulary: 32 partial sums per request, the picked chunk anywhere."""
    want = _check(True, 24, 2, 128256, dt, seed=3)
    assert len({row[m] // 4096 for row, m in zip(*want)}) > 4
    # more partial sums than lanes
    _check(True, 2, 1, 64 * 4096 * 2 + 77, dt, seed=4)


def _corners(p, q, tokens, u, u_last):
    """One request per corner."""
    V = p.shape[2]
    tokens[0, 0] = -1                       # outside the vocabulary: refused
    tokens[1, 0] = V
    p[2] = 0                                # no weight at all: -1
    p[3, 0], q[3, 0] = 1.0 / V, 1.0 / V     # refused although equal (u_q < p fails at 0): nothing remains
    p[3, 0, tokens[3, 0]] = 0
    q[3, 0, tokens[3, 0]] = 0
    p[4, 0, 0] = math.nan                   # weighs nothing
    q[4, 0, 1] = math.nan
    u[4, 0] = 0.999
    q[5, 0, tokens[5, 0]] = 0               # p > 0 = q: stays whatever u is
    u[5, 0] = 1 - 2.0 ** -24
    u_last[6] = 0                           # the first entry with weight
    u_last[7] = 1 - 2.0 ** -24              # the last numbers there are
    p[6, 0, :3] = 0
    p[8, 0] = 0                             # all weight in one entry behind the drafted one
    p[8, 0, V - 1] = 1
    tokens[8, 0] = 0
    tokens[9, 1] = tokens[9, 0]             # the same token twice
    p[10, 0, 4] = -1.0                      # a negative probability weighs nothing


def test_verify_corners_cpu(fake_rt):
    for certain in (False, True):
        _check(False, 11, 2, 300, torch.float32, certain, change=_corners)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 300, 9000])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_corners_gpu(gpu_rt, V, certain):
    _check(True, 11, 2, V, torch.float32, certain, change=_corners)


def _distribution(gpu):
    """Over many draws the tokens are distributed as the target's, whatever the
    draft proposes: 4 entries, 40000 requests, 5 standard deviations."""
    dev, n = ("cuda" if gpu else "cpu"), 40000
    g = torch.Generator().manual_seed(1)
    p = torch.tensor([0.5, 0.2, 0.05, 0.25])
    q = torch.tensor([0.1, 0.6, 0.3, 0.0])
    tokens = torch.multinomial(q, n, replacement=True, generator=g).to(I32)[:, None]
    u, u_last = torch.rand(n, 1, generator=g), torch.rand(n, generator=g)
    out, acc = speculative.verify_draft(p.expand(n, 2, 4).to(dev), q.expand(n, 1, 4).to(dev), tokens.to(dev), u.to(dev),
                                        u_last.to(dev))
    first = torch.bincount(out[:, 0].cpu().long(), minlength=4) / n
    assert ((first - p).abs() < 5 * torch.sqrt(p * (1 - p) / n)).all()
    assert abs(acc.float().mean().item() - torch.minimum(p, q).sum().item()) < 5 * 0.5 / math.sqrt(n)


def test_verify_keeps_the_distribution_cpu(fake_rt):
    _distribution(False)


@pytest.mark.gpu
def test_verify_keeps_the_distribution_gpu(gpu_rt):
    _distribution(True)


def test_verify_refuses(fake_rt):
    B, K, V = 2, 3, 10
    ok = dict(target_probs=torch.rand(B, K + 1, V), draft_probs=torch.rand(B, K, V),
              draft_tokens=torch.zeros(B, K, dtype=I32), u=torch.rand(B, K), u_last=torch.rand(B),
              counts=torch.zeros(B, dtype=I32))
    speculative.verify_draft(**ok)
    speculative.verify_draft(**{**ok, "draft_probs": None, "counts": None})
    for bad in (dict(target_probs=torch.rand(B, K, V)), dict(target_probs=torch.rand(B, V)),
                dict(target_probs=torch.rand(B, K + 1, V, dtype=torch.float64)),
                dict(target_probs=torch.rand(B, V, K + 1).transpose(1, 2)), dict(target_probs=torch.rand(B, 0, V)),
                dict(target_probs=torch.rand(B, K + 1, 0)), dict(draft_probs=torch.rand(B, K, V).half()),
                dict(draft_probs=torch.rand(B, K, V - 1)), dict(draft_tokens=torch.zeros(B, K, dtype=torch.int64)),
                dict(draft_tokens=torch.zeros(B, K + 1, dtype=I32)), dict(u=torch.rand(B, K).double()),
                dict(u=torch.rand(K, B).t()), dict(u_last=torch.rand(B, 1)), dict(counts=torch.zeros(B)),
                dict(counts=torch.zeros(B + 1, dtype=I32)), dict(u_last=torch.rand(B, device="meta"))):
        with pytest.raises(ValueError):
            speculative.verify_draft(**{**ok, **bad})
