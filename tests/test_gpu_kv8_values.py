"""GPU: attention over 8-bit pages at the ends of the numbers' ranges: V values far apart in size, and
scores past the steps of fp32."""
import math

import pytest

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
D, B = 128, 64


@pytest.fixture(scope="module")
def ctx():
    from momij_amd.ops import Context

    c = Context(0)
    yield c
    c.close()


# M, nQ, nKV, blocks: each form of the page kernels, several pages to a state
FORMS = [(1, 32, 32, 200), (5, 128, 32, 200), (9, 128, 32, 200), (20, 16, 4, 400), (64, 16, 4, 360)]


@pytest.mark.parametrize("M,nQ,nKV,n", FORMS)
def test_small_values_beside_great_ones(ctx, M, nQ, nKV, n):
    """Blocks that hold V of 2^14 in the upper dims or 2^-12 in the lower ones, both among those of every
    wave (pages in a row, or four or eight apart): scales 2^26 apart under like weights.

    The weights carry the V scale into fp16: 2^-11 of a weight, or below fp16's normal range half its
    least step, 2^-25.  The greatest weight times scale of a part lies between 2^9 and 2^15 there, so
    that step is at most 2^-34 of it, a code."""
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda")

    G, open_ = nQ // nKV, 20
    kk = rnd(nKV, n, B, D).half()
    vv = 0.5 + 0.5 * torch.rand((nKV, n, B, D), generator=gen, device="cuda")
    i = torch.arange(n, device="cuda")
    great = (((i + i // 8) % 2 == 0)[:, None] == (torch.arange(D, device="cuda") >= D // 2)).float()
    vv = torch.where(((i + i // 8) % 2 == 0)[:, None, None], 2.0 ** 14 * vv, 2.0 ** -12 * vv)
    vv = (vv * great[:, None]).half()
    cap = open_ + M
    rk, rv = rnd(nKV, cap, D).half(), torch.zeros((nKV, cap, D), device="cuda").half()
    q = (0.7 * rnd(M, nQ * D)).half()
    cache, out = Kv8Cache(ctx, nKV, n), torch.empty_like(q)
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(kk.reshape(nKV, -1, D), vv.reshape(nKV, -1, D)), 0, n, 0)
    ctx.kv8_attn(cache, KvRing(rk, rv), q, M, nQ, n, n * B, n * B + open_, None, out)
    ctx.sync()
    at = [(n * B + i) % cap for i in range(cap)]
    ok = torch.cat([torch.ones((M, n * B + open_), dtype=torch.bool), ref.sees(None, M)[0]], 1).cuda()
    for g in range(nKV):
        (kc, ks), (vc, vs) = ref.seal(kk[g]), ref.seal(vv[g])
        k = torch.cat([(kc * ks.double()[:, None, None]).reshape(-1, D), rk[g, at].double()])
        scale = torch.cat([vs.double().repeat_interleave(B), torch.ones(cap, device="cuda").double()])
        code = torch.cat([vc.reshape(-1, D), rv[g, at].double()])
        qg = q.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D)
        want, p, _, rel = ref.attention(qg, k, code * scale[:, None], ok.repeat_interleave(G, 0))
        unit = (p * scale).amax(1, keepdim=True)
        tol = (p @ (code * scale[:, None]).abs()) * (ref.E16 + rel + 2.0 ** -20) + want.abs() * ref.E16
        tol += 2.0 ** -25 + 2.0 ** -34 * unit * code.abs().sum(0)
        err = (out.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D) - want).abs()
        assert (err <= tol).all(), (g, float((err / tol).max()), float((err / want.abs()).max()))


def randoms(seed):
    import torch

    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return lambda *s: torch.rand(s, generator=gen, device="cuda")


def attend(ctx, kk, vv, rk, rv, q, M, nQ, n):
    """Outputs [M, nKV, G, D] and masses of rows q over the sealed blocks of kk, vv [nKV][n * B][D] and 20
    open rows of the ring."""
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    nKV = kk.shape[0]
    cache, out = Kv8Cache(ctx, nKV, n), torch.empty_like(q)
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(kk, vv), 0, n, 0)
    ctx.kv8_attn(cache, KvRing(rk, rv), q, M, nQ, n, n * B, n * B + 20, None, out, mass_out=cache.mass)
    ctx.sync()
    return out.double().reshape(M, nKV, nQ // nKV, D), cache.mass.double()


def check_winners(out, mass, vv, at, n):
    """Each row's weight lies on the keys at [x, M, nKV, G], in equal parts: the mean of their values.

    The error: a weight's and the output's rounding to fp16, and exponentials."""
    import torch

    nKV, M, G = vv.shape[0], at.shape[1], at.shape[3]
    for g in range(nKV):
        vc, vs = ref.seal(vv[g].reshape(n, B, D))
        v = (vc * vs.double()[:, None, None]).reshape(-1, D)[at[:, :, g]]
        err, size = (out[:, g] - v.mean(0)).abs(), v.abs().mean(0)
        assert (err <= size * (2 * ref.E16 + 2.0 ** -19) + 2.0 ** -25).all(), (g, float((err / size).max()))
        part = torch.full((at[:, :, g].numel(),), 1.0 / at.shape[0], device="cuda", dtype=torch.float64)
        want = torch.zeros(n, device="cuda").double().index_add_(0, (at[:, :, g] // B).reshape(-1), part)
        assert ((mass[g] - want).abs() <= want * (2.0 ** -19 + (M * G + 4) * ref.E32)).all(), g


def values(rand, nKV, n):
    """V of blocks whose scales lie up to 2^9 apart."""
    return ((0.5 + 0.5 * rand(nKV, n, B, D)) * 2.0 ** (1.0 - 9.0 * rand(nKV, n, 1, 1))).half().reshape(nKV, -1, D)


@pytest.mark.parametrize("M,nQ,nKV,n", FORMS)
def test_scores_past_the_steps_of_fp32(ctx, M, nQ, nKV, n):
    """Queries and keys near fp16's greatest: scores to 2^35, whose steps in fp32 are thousands.  Each
    query is a key's pattern of signs, so every other score is lower by a third or more; the keys of the
    first and the second block are the same, and share a query's weight whatever their V scales."""
    import torch

    rand, G, T = randoms(n + M), nQ // nKV, n * B
    sign = torch.where(rand(nKV, T, D) < 0.5, -1.0, 1.0)
    sign[:, B:2 * B] = sign[:, :B]
    vv = values(rand, nKV, n)
    rk, rv = ((rand(nKV, 20 + M, D) - 0.5).half() for _ in range(2))
    for tie in (False, True):
        lo, hi = (B, 2 * B) if tie else (2 * B, T)
        at = lo + (rand(M, nKV, G) * (hi - lo)).long().clamp(max=hi - lo - 1)
        q = 60000.0 * sign[torch.arange(nKV, device="cuda")[None, :, None], at].reshape(M, nQ * D)
        out, mass = attend(ctx, (50000.0 * sign).half(), vv, rk, rv, q.half(), M, nQ, n)
        check_winners(out, mass, vv, torch.stack([at, at - B]) if tie else at[None], n)


@pytest.mark.parametrize("M,nQ,nKV,n", FORMS)
def test_scores_far_below_zero(ctx, M, nQ, nKV, n):
    """Keys along one direction and queries against it: the shortest key has the greatest score."""
    import torch

    rand, G, T = randoms(n + M + 1), nQ // nKV, n * B
    sign = torch.where(rand(D) < 0.5, -1.0, 1.0)
    size, at = 30000.0 + 30000.0 * rand(nKV, T, 1), T // 2 + 3
    size[:, at] = 10000.0
    vv = values(rand, nKV, n)
    rk, rv = (50000.0 * sign).expand(nKV, 20 + M, D).half().contiguous(), rand(nKV, 20 + M, D).half()
    q = (-60000.0 * sign).expand(M, nQ, D).reshape(M, nQ * D).half()
    out, mass = attend(ctx, (size * sign).half(), vv, rk, rv, q, M, nQ, n)
    check_winners(out, mass, vv, torch.full((1, M, nKV, G), at, device="cuda"), n)
