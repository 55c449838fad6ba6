"""GPU: attention over 8-bit pages whose V values are far apart in size: the small ones are not lost
beside the great ones."""
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
