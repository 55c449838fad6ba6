"""GPU: attention over pages at the ends of fp16: scores as large as they come, values of the greatest number."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R
from momij_amd.paged import PagedCache
from test_gpu_paged_attn import D, batch_of, ctx, cuda, make  # noqa: F401

pytestmark = pytest.mark.gpu
TOP = 65504.0
FORMS = [(1, 16), (9, 16), (64, 16)]


@pytest.mark.parametrize("M,nq", FORMS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_greatest_scores(ctx, M, nq, sign):  # noqa: F811
    """All dims of queries and keys at fp16's greatest number: scores of 2^39, 2^36 in units of log2.  Equal ones
    weigh the same; of 2^28 more (2^25 in log2) one key has everything."""
    L = 300
    cache, gen, _ = make(ctx, [L], [M], 64, 4, seed=M)
    every = torch.arange(L + M, device="cuda")
    k, v = R.rows_of(cache, 0, 0, every)
    k = torch.full_like(k, sign * TOP)
    R.put(cache, 0, 0, every, k, v)
    q = torch.full((M, nq * D), sign * TOP, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of([M]), q, nq, out)
    got = out.double().reshape(M, nq, D)
    for r in range(M):
        n = L + r + 1
        x = v[:n].repeat_interleave(nq // 4, 1)
        want, size = x.mean(0), x.abs().mean(0)
        # weights are equal powers of two, so exact up to the sums in fp32 and the output's rounding
        tol = want.abs() * 2.0 ** -11 + size * (n + 8) * 2.0 ** -24 + 2.0 ** -25
        assert bool(((got[r] - want).abs() <= tol).all()), r
    # a step of fp16 less in all keys but one
    k[:] = sign * 65472.0
    k[137] = sign * TOP
    R.put(cache, 0, 0, every, k, v)
    ctx.paged_attn(cache, 0, batch_of([M]), q, nq, out)
    want = v[137].repeat_interleave(nq // 4, 0).expand(M, nq, D)
    assert torch.equal(out.double().reshape(M, nq, D), want)


@pytest.mark.parametrize("M,nq", FORMS)
def test_the_greatest_values(ctx, M, nq):  # noqa: F811
    """V of 65504 everywhere: so is the output, though weights are rounded upwards.  Units of 32 keys of score 0 and,
    four of 32, of one whose weight lies just above the middle of two fp16 numbers when the reference is the others'
    score: the rounded weights' sum is up to 2^-11 more than the sum of the weights, and from 65520 on a number
    would round to an infinity."""
    L = 131000
    at, k = (np.arange(64) / 1024.0 + 1.0)[:, None], np.arange(1, 6000) / 128.0
    k = k.astype(np.float16).astype(np.float64)
    w = np.exp2(at * k / math.sqrt(D) * math.log2(math.e))  # scores q k / sqrt(128)
    off = (w.astype(np.float16).astype(np.float64) / w - 1.0) * ((w > 24) & (w < 60))
    i, j = np.unravel_index(off.argmax(), off.shape)
    assert off.max() > 1.9 * 2.0 ** -12
    cache, gen, _ = make(ctx, [L], [M], 64, 4, seed=M)
    every = torch.arange(L + M, device="cuda")
    kk = torch.zeros((L + M, 4, D), device="cuda")
    kk[:, :, 5] = torch.where(every // 128 % 8 == 7, float(k[j]), 0.0)[:, None]
    v = torch.full((L + M, 4, D), TOP, device="cuda")
    v[:, :, 1::2] = -TOP
    R.put(cache, 0, 0, every, kk, v)
    q = torch.zeros((M, nq, D), dtype=torch.float16, device="cuda")
    q[:, :, 5] = float(at[i, 0])
    out = torch.full((M, nq * D), 7.0, dtype=torch.float16, device="cuda")
    ctx.paged_attn(cache, 0, batch_of([M]), q.reshape(M, -1), nq, out)
    got = out.reshape(M, nq, D)
    # half a step of fp16 for every weight and for the output
    for x in (got[:, :, ::2], -got[:, :, 1::2]):
        assert bool(((x.double() - TOP).abs() <= TOP * 2.0 ** -10).all())


@pytest.mark.parametrize("M,nq", FORMS)
@pytest.mark.parametrize("L", [0, 40, 4000])
def test_infinite_values_stay_infinite(ctx, M, nq, L):  # noqa: F811
    """A row that gives an infinity to itself: it is one, of its sign; beside it the greatest numbers are kept."""
    cache, gen, _ = make(ctx, [L], [M], 64, 4, seed=L + M)
    every = torch.arange(L + M, device="cuda")
    k, v = R.rows_of(cache, 0, 0, every)
    v = torch.full_like(v, TOP)
    v[L + M - 1, :, 0::3], v[L + M - 1, :, 1::3] = math.inf, -math.inf
    R.put(cache, 0, 0, every, torch.zeros_like(k), v)
    q = torch.zeros((M, nq * D), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of([M]), q, nq, out)
    got = out.reshape(M, nq, D)
    assert bool((got[:M - 1] == TOP).all()) and bool((got[M - 1, :, 2::3] == TOP).all())
    assert bool((got[M - 1, :, 0::3] == math.inf).all()) and bool((got[M - 1, :, 1::3] == -math.inf).all())
