"""What the paged serving ops promise beyond a result within the types' rounding
(tests/test_attention_paged.py holds the forms they are compared with)."""
from __future__ import annotations

import math

import pytest
import torch

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
