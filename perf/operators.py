"""What the paged-serving operators are measured on: the step plan over a paged
KV cache (ops/paged.py plan), RoPE with the append into pages (rope_kv),
attention of new tokens over the pages (attention) and the verification of
drafted tokens (ops/speculative.py verify_draft) - each beside its plain form.

A case is a dict of plain values. ``run`` computes the plain form (elementary
torch operations in f32, f64 where a border decides) while ``own`` is false and
calls the framework while it is true; ``exact`` is the definition in f64.

Head counts and sizes are those of the repository's Llama-3 configurations
(8B 32:8, 70B 64:8, one rank of 70B tp8 8:1, "small" 16:4 with 64 dims; vocab
128256) at serving batch sizes, with ragged lengths drawn from the case's own
``lens`` number (so that the work of a case is known without its seed).
"""
from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 128256
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
HEADS = ((32, 8, 128), (64, 8, 128), (8, 1, 128), (16, 4, 64), (16, 1, 128), (8, 8, 64), (12, 2, 128), (24, 8, 128))
MAX_POS = 1 << 17


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 64 running requests: every one appends one token, few need a page
        dict(name="plan-64x1", op="plan", B=64, q=1, chunks=0, kv=1025, ragged=True, page=16, lens=1),
        # a step that admits prompts: 1024 requests, a quarter of them with a chunk of up to 129 tokens
        dict(name="plan-1024-mixed", op="plan", B=1024, q=129, chunks=256, kv=4097, ragged=True, page=32, lens=2),
        # one token of each of 64 requests (8B heads)
        dict(name="rope-64-8b", op="rope", n=64, hq=32, hkv=8, hd=128, page=16, dtype="bf16"),
        # a prefill chunk of 8192 tokens (70B heads)
        dict(name="rope-8192-70b", op="rope", n=8192, hq=64, hkv=8, hd=128, page=64, dtype="fp16"),
        # one request alone, one token: latency
        dict(name="attn-1x1-1025-8b", op="attn", B=1, q=1, chunks=1, kv=1025, ragged=False, hq=32, hkv=8, hd=128,
             page=16, dtype="bf16", lens=3),
        # the decode batch of the headline model: 64 requests of ragged lengths, one token each
        dict(name="attn-64x1-2048-70b", op="attn", B=64, q=1, chunks=64, kv=2048, ragged=True, hq=64, hkv=8, hd=128,
             page=16, dtype="bf16", lens=4),
        # four long contexts, one token each: the key axis has to be split
        dict(name="attn-4x1-131072-8b", op="attn", B=4, q=1, chunks=4, kv=131071, ragged=True, hq=32, hkv=8, hd=128,
             page=64, dtype="fp16", lens=5),
        # five drafted tokens of 32 requests on one tensor-parallel rank
        dict(name="attn-32x5-8192-tp8", op="attn", B=32, q=5, chunks=32, kv=8191, ragged=True, hq=8, hkv=1, hd=128,
             page=32, dtype="bf16", lens=6),
        # decodes and prompt chunks in one batch (64-wide heads)
        dict(name="attn-48-mixed-64d", op="attn", B=48, q=511, chunks=12, kv=2047, ragged=True, hq=16, hkv=4, hd=64,
             page=16, dtype="fp16", lens=7),
        # a chunk of a long prompt behind cached tokens: the matrix cores' case
        dict(name="attn-1x4096-8191-8b", op="attn", B=1, q=4096, chunks=1, kv=8191, ragged=False, hq=32, hkv=8,
             hd=128, page=128, dtype="bf16", lens=8),
        # one request's four drafted tokens
        dict(name="verify-1x4", op="verify", B=1, K=4, V=VOCAB, ragged=False, dtype="bf16", lens=9),
        # 64 requests with up to eight drafted tokens each
        dict(name="verify-64x8", op="verify", B=64, K=8, V=VOCAB, ragged=True, dtype="f32", lens=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, no dearer than the largest listed one."""
    op = rng.choice(("plan", "rope", "attn", "attn", "attn", "attn", "verify"))
    lens = rng.randrange(1 << 20)
    if op == "plan":
        B = _log(rng, 1, 2048)
        q = rng.choice((1, _log(rng, 1, 512)))
        return dict(op=op, B=B, q=q, chunks=rng.randint(0, min(B, 65536 // q)), kv=_log(rng, max(16, q), 8192),
                    ragged=rng.random() < 0.8, page=rng.choice((16, 32, 64, 128, 256)), lens=lens)
    hq, hkv, hd = rng.choice(HEADS)
    page, dtype = rng.choice((16, 32, 64, 128, 256)), rng.choice(("bf16", "fp16"))
    if op == "rope":
        return dict(op=op, n=_log(rng, 1, 8192), hq=hq, hkv=hkv, hd=hd, page=page, dtype=dtype)
    if op == "verify":
        return dict(op=op, B=_log(rng, 1, 64), K=rng.randint(1, 8), V=rng.choice((VOCAB, _log(rng, 4096, 131071))),
                    ragged=rng.random() < 0.5, dtype=rng.choice(("f32", "bf16", "fp16")), lens=lens)
    kind = rng.choice(("decode", "draft", "chunk", "mixed"))
    if kind == "decode":
        B = _log(rng, 1, 128)
        q, kv = 1, _log(rng, 1, min(131071, (1 << 21) // (B * hkv)))
    elif kind == "draft":
        B, q = _log(rng, 1, 64), rng.randint(2, 9)
        kv = _log(rng, q, min(65535, (1 << 20) // (B * hkv)))
    elif kind == "chunk":
        B = rng.randint(1, 4)
        q = _log(rng, 17, 2048 // B)
        kv = _log(rng, q, 16383 // B)
    else:
        B = rng.randint(2, 48)
        q = _log(rng, 17, 511)
        kv = _log(rng, q, 2047)
    if q > 9:  # as many score products as the largest listed case has, at most
        B = max(1, min(B, int(8e8 / (hq * q * kv))))
        q = min(q, max(1, int(8e8 / (hq * kv))))
    return dict(op="attn", B=B, q=q, chunks=rng.randint(1, B) if kind == "mixed" else B, kv=kv,
                ragged=rng.random() < 0.8, hq=hq, hkv=hkv, hd=hd, page=page, dtype=dtype, lens=lens)


def _lengths(case):
    """New tokens and cached-plus-new tokens of every request. ``chunks``
    requests bring up to ``q`` tokens (exactly q where the batch is a uniform
    step of a few tokens), the others one."""
    r = random.Random(case["lens"])
    B, q, kv = case["B"], case["q"], case["kv"]
    many = set(r.sample(range(B), case["chunks"]))
    ql, kl = [], []
    for b in range(B):
        n = 1 if b not in many else q if q <= 16 or not case["ragged"] else r.randint((q + 1) // 2, q)
        n = min(n, kv)
        ql.append(n)
        kl.append(max(n, r.randint((kv + 3) // 4, kv)) if case["ragged"] else kv)
    kl[0] = kv
    return ql, kl


def _drafts(case):
    r = random.Random(case["lens"])
    return [r.randint(0, case["K"]) if case["ragged"] else case["K"] for _ in range(case["B"])]


# ---------------------------------------------------------------- inputs
def _ints(v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32).to(device)


def _table(counts, width, spare, g):
    """Block table of requests that hold ``counts`` pages each, scattered over
    the pool; entries behind a request's pages are -1; and the spare pages."""
    perm = torch.randperm(sum(counts) + spare, generator=g, dtype=torch.int64).to(torch.int32)
    c = torch.tensor(counts)
    first = torch.cumsum(c, 0) - c
    col = torch.arange(width)
    at = (first[:, None] + col).clamp(max=max(perm.numel() - 1, 0))
    table = torch.where(col < c[:, None], perm[at], torch.tensor(-1, dtype=torch.int32))
    return table.cuda(), perm[sum(counts):].cuda()


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gg = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "plan":
        P = case["page"]
        ql, kl = _lengths(case)
        old = [k - n for k, n in zip(kl, ql)]
        counts = [-(-o // P) for o in old]
        width = -(-case["kv"] // P) + 2
        need = sum(-(-k // P) - c for k, c in zip(kl, counts))
        s["table"], s["free"] = _table(counts, width, need + 7, g)
        s |= dict(new=_ints(ql), kv=_ints(old), counts=_ints(counts), start=_ints([0]), page=P, n=sum(ql))
        return s
    if case["op"] == "verify":
        B, K, V, dt = case["B"], case["K"], case["V"], DTYPES[case["dtype"]]
        logits = torch.empty(B, K + 1, V, device="cuda").normal_(0, 2.5, generator=gg)
        p = torch.softmax(logits, -1)
        q = torch.softmax(logits[:, :K] + torch.empty(B, K, V, device="cuda").normal_(0, 0.6, generator=gg), -1)
        s["tokens"] = torch.multinomial(q.view(B * K, V), 1, generator=gg).view(B, K).to(torch.int32)
        s |= dict(p=p.to(dt), q=q.to(dt), counts=_ints(_drafts(case)),
                  u=torch.rand(B, K, device="cuda", generator=gg), u_last=torch.rand(B, device="cuda", generator=gg))
        return s
    hq, hkv, hd, P, dt = case["hq"], case["hkv"], case["hd"], case["page"], DTYPES[case["dtype"]]
    if case["op"] == "rope":
        n = case["n"]
        used = -(-n // P) + 3
        inv = 1.0 / (500000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd))
        ang = torch.outer(torch.arange(MAX_POS, dtype=torch.float64, device="cuda"), inv)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["qkv"] = torch.empty(n, (hq + 2 * hkv) * hd, device="cuda").normal_(0, 1, generator=gg).to(dt)
        s["pages"] = torch.empty(2, used, hkv, P, hd, device="cuda").normal_(0, 1, generator=gg).to(dt)
        s["slots"] = torch.randperm(used * P, generator=g)[:n].to(torch.int32).cuda()
        s["positions"] = torch.randint(0, MAX_POS, (n,), generator=g, dtype=torch.int32).cuda()
        return s
    ql, kl = _lengths(case)
    counts = [-(-k // P) for k in kl]
    s["table"], _ = _table(counts, -(-case["kv"] // P) + 1, 5, g)
    n = sum(ql)
    s["q"] = torch.empty(n, hq, hd, device="cuda").normal_(0, 1, generator=gg).to(dt)
    s["pages"] = torch.empty(2, sum(counts) + 5, hkv, P, hd, device="cuda", dtype=dt).normal_(0, 1, generator=gg)
    cu = [0]
    for x in ql:
        cu.append(cu[-1] + x)
    s |= dict(cu=_ints(cu), kv=_ints(kl), max_q=max(ql), max_kv=max(kl))
    return s


# ---------------------------------------------------------------- plain forms
def _plain_plan(s):
    P, n = s["page"], s["n"]
    new, kv, have = s["new"].long(), s["kv"].long(), s["counts"].long()
    table, free, width = s["table"], s["free"], s["table"].shape[1]
    end = torch.cumsum(new, 0)
    cu = torch.cat([end.new_zeros(1), end]).clamp(max=n)
    total = (kv + new + P - 1) // P
    fits = (total <= width) & (end <= n)
    need = torch.where(fits, (total - have).clamp(min=0), 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (s["start"] + upto <= free.numel()))
    take = torch.where(granted, need, 0)
    col = torch.arange(width, device=table.device)
    j = col - have[:, None]  # which of its new pages a column is
    at = (s["start"] + (upto - need)[:, None] + j).clamp(0, max(free.numel() - 1, 0))
    table.copy_(torch.where((j >= 0) & (j < take[:, None]), free[at], table))
    t = torch.arange(n, device=table.device)
    b = torch.searchsorted(end, t, right=True).clamp(max=new.numel() - 1)
    pos = kv[b] + t - cu[b]
    page = table[b, (pos // P).clamp(max=width - 1)].long()
    live = (t < cu[-1]) & granted[b]
    slots = torch.where(live & (page >= 0), page * P + pos % P, -1)
    return {"cu_q": cu.int(), "kv_lens": torch.where(granted, kv + new, kv).int(),
            "page_counts": torch.where(granted, torch.maximum(have, total), have).int(),
            "positions": torch.where(live, pos, -1).int(), "slots": slots.int(), "granted": granted.int(),
            "free_start": (s["start"] + take.sum()).int(), "block_table": table}


def _plain_rope(s):
    c = s["case"]
    hq, hkv, hd, P = c["hq"], c["hkv"], c["hd"], c["page"]
    x = s["qkv"].view(-1, hq + 2 * hkv, hd)
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    a, b = x[:, :hq + hkv].float().chunk(2, -1)
    r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
    at = s["slots"].long()
    s["pages"][0][at // P, :, at % P] = r[:, hq:]
    s["pages"][1][at // P, :, at % P] = x[:, hq + hkv:]
    return {"q": r[:, :hq], "pages": s["pages"]}


def _plain_attn(s):
    c = s["case"]
    hq, hkv, hd, P, B = c["hq"], c["hkv"], c["hd"], c["page"], c["B"]
    g, mq, mk, n = hq // hkv, s["max_q"], s["max_kv"], s["q"].shape[0]
    cu, kv = s["cu"].long(), s["kv"].long()
    ql = cu[1:] - cu[:-1]
    i = torch.arange(mq, device="cuda")
    q = s["q"][(cu[:-1, None] + i).clamp(max=n - 1)].float()  # [B, mq, hq, hd]
    q = q.view(B, mq, hkv, g, hd).permute(0, 2, 1, 3, 4).reshape(B, hkv, mq * g, hd)
    t = torch.arange(mk, device="cuda")
    page = s["table"][:, t // P].long().clamp(min=0)
    k = s["pages"][0][page, :, t % P].float().permute(0, 2, 3, 1).contiguous()  # [B, hkv, hd, mk]
    v = s["pages"][1][page, :, t % P].float().permute(0, 2, 1, 3).contiguous()
    pos = kv[:, None] - ql[:, None] + i  # of the query rows
    seen = (t <= pos[:, :, None]) & (t < kv[:, None, None])  # [B, mq, mk]
    sc = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).view(B, hkv, mq, g, mk)
    sc.masked_fill_(~seen[:, None, :, None], float("-inf"))
    p = sc.sub_(sc.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, mq * g, mk), v).view(B, hkv, mq, g, hd)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(B, mq, hq * hd)
    row = torch.arange(n, device="cuda")
    b = torch.searchsorted(cu[1:], row, right=True).clamp(max=B - 1)
    return o[b, row - cu[b]].to(s["q"].dtype)


def _plain_verify(s):
    p, q, tok, count = s["p"], s["q"], s["tokens"].long(), s["counts"].long()
    B, K = tok.shape
    pt = p[:, :K].gather(-1, tok[..., None])[..., 0].double()
    qt = q.gather(-1, tok[..., None])[..., 0].double()
    j = torch.arange(K, device=p.device)
    ok = (s["u"].double() * qt < pt) & (j < count[:, None])
    m = torch.cumprod(ok.long(), 1).sum(1)  # accepted drafts
    row = torch.arange(B, device=p.device)
    target = p[row, m].double()
    rest = torch.where((m < count)[:, None], target - q[row, m.clamp(max=K - 1)].double(), target).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, target)
    c = torch.cumsum(rest, -1)
    new = (c <= s["u_last"].double()[:, None] * c[:, -1:]).sum(-1)
    col = torch.arange(K + 1, device=p.device)
    pad = torch.cat([tok, tok.new_zeros(B, 1)], 1)
    out = torch.where(col < m[:, None], pad, torch.where(col == m[:, None], new[:, None], -1))
    return {"tokens": out.int(), "accepted": m.int()}


_loaded = []


def _framework():
    if not _loaded:
        from ogkm import rt
        from ogkm.ops import paged, speculative

        if not rt.is_initialized():
            rt.init("hip")
        _loaded.extend((paged, speculative))
    return _loaded


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        paged, speculative = _framework()
        c = s["case"]
        if op == "plan":
            r = paged.plan(s["new"], s["kv"], s["counts"], s["table"], s["free"], s["start"], s["page"], s["n"])
            return {"cu_q": r.cu_q, "kv_lens": r.kv_lens, "page_counts": r.page_counts, "positions": r.positions,
                    "slots": r.slots, "granted": r.granted, "free_start": r.free_start, "block_table": s["table"]}
        if op == "rope":
            q = paged.rope_kv(s["qkv"], s["cos"], s["sin"], s["pages"], s["positions"], s["slots"], c["hq"], c["hkv"])
            return {"q": q, "pages": s["pages"]}
        if op == "attn":
            return paged.attention(s["q"], s["pages"], s["cu"], s["kv"], s["table"], max_q=s["max_q"],
                                   max_kv=s["max_kv"])
        tokens, accepted = speculative.verify_draft(s["p"], s["q"], s["tokens"], s["u"], s["u_last"], s["counts"])
        return {"tokens": tokens, "accepted": accepted}
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "verify": _plain_verify}[op](s)


# ---------------------------------------------------------------- floors and definitions
def work(case):
    if case["op"] == "plan":
        ql, kl = _lengths(case)
        B, n, P = case["B"], sum(ql), case["page"]
        # lengths and counts in and out, a table entry and a free page for each new page, one table entry for each
        # (request, page) that a new token falls into, positions and slots out
        pages = sum(-(-k // P) - (k - x) // P for k, x in zip(kl, ql))
        return {"bytes": 4.0 * (3 * B + 4 * B + 2 * n + 2 * pages), "flops": 2.0 * n}
    if case["op"] == "rope":
        n, hq, hkv, hd = case["n"], case["hq"], case["hkv"], case["hd"]
        return {"bytes": 2.0 * 2 * n * (hq + 2 * hkv) * hd + n * (4.0 * hd + 8), "flops": 3.0 * n * (hq + hkv) * hd}
    if case["op"] == "attn":
        ql, kl = _lengths(case)
        hq, hkv, hd, P = case["hq"], case["hkv"], case["hd"], case["page"]
        pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(ql, kl))
        return {"bytes": 2.0 * (2 * sum(kl) * hkv * hd + 2 * sum(ql) * hq * hd) + 4.0 * sum(-(-k // P) for k in kl),
                "flops": 4.0 * hd * hq * pairs}
    # two rows of every request (one where all drafts stay), and two values of each draft
    B, V, size = case["B"], case["V"], 4 if case["dtype"] == "f32" else 2
    return {"bytes": 2.0 * B * V * size + sum(_drafts(case)) * (2 * size + 8) + 4.0 * B * (case["K"] + 4), "flops": 3.0 * B * V}


def exact(case, seed):
    if case["op"] in ("plan", "verify"):
        return None  # whole numbers: held to equality
    s = prepare(case, seed)
    hq, hkv, hd, P = case["hq"], case["hkv"], case["hd"], case["page"]
    if case["op"] == "rope":
        z = s["qkv"].double().view(-1, hq + 2 * hkv, hd)
        at, slot = s["positions"].tolist(), s["slots"].long()
        turn = torch.polar(torch.ones(len(at), hd // 2, dtype=torch.float64, device="cuda"),
                           torch.atan2(s["sin"].double(), s["cos"].double())[at])
        size = torch.hypot(s["sin"].double(), s["cos"].double())[at]
        w = torch.complex(z[:, :hq + hkv, :hd // 2].contiguous(), z[:, :hq + hkv, hd // 2:].contiguous())
        w = w * (turn * size)[:, None]
        r = torch.cat([w.real, w.imag], -1)
        pages = s["pages"].double().transpose(2, 3).reshape(2, -1, hkv, hd)
        pages[0, slot], pages[1, slot] = r[:, hq:], z[:, hq + hkv:]
        return {"q": r[:, :hq], "pages": pages.view(2, -1, P, hkv, hd).transpose(2, 3).contiguous()}
    g = hq // hkv
    ql, kl = _lengths(case)
    out = torch.empty(sum(ql), hq * hd, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, length) in enumerate(zip(ql, kl)):
        ids = s["table"][b, : -(-length // P)].long()
        hidden = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        for h in range(hkv):
            k, v = (s["pages"][x, ids, h].reshape(-1, hd)[:length].double() for x in (0, 1))
            for j in range(h * g, (h + 1) * g):
                w = (s["q"][at:at + n, j].double() @ k.T) / math.sqrt(hd)
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                out[at:at + n, j * hd:(j + 1) * hd] = w @ v
        at += n
    return out
