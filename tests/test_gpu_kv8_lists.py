"""GPU: choosing and evicting at the ends of their ranges: nothing kept, everything kept or listed, more
listed than there is, wide passes over long lists, and the attention block over a long list."""
import math

import numpy as np
import pytest

from momij_amd import synth
from tests import kv8_ref as ref
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu
D, B = 128, 64


@pytest.fixture(scope="module")
def ctx():
    from momij_amd.ops import Context

    c = Context(0)
    yield c
    c.close()


def generator(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("n", [1, 256, 257, 1024, 1025, 4096, 4097, 16384, 16385, 20000])
def test_evict_none_all_and_only_the_held(ctx, n):
    import torch

    from momij_amd.kv8 import Kv8Cache

    gen, stride = generator(n), n + 3
    cache = Kv8Cache(ctx, 2, stride)
    cache.table.copy_(torch.stack([torch.randperm(stride, generator=gen, device="cuda") for _ in range(2)]))
    mass = torch.rand((2, stride), generator=gen, device="cuda")
    mass[0, ::3], mass[1, 1::5] = math.nan, math.inf
    a, b = min(n, 3) // 2, min(n, 3) - min(n, 3) // 2
    for keep, first, last in ((0, 0, 0), (n, 0, 0), (n, a, b), (a + b, a, b), (a + b, 0, a + b), (a + b, a + b, 0)):
        table, m1 = torch.full_like(cache.table, -7), torch.full_like(mass, -7.0)
        torch.cuda.synchronize()
        ctx.kv8_evict(cache, n, keep, first, last, mass, table, m1)
        ctx.sync()
        for g in range(2):
            kept = ref.choose(mass[g, :n].tolist(), first, last, keep)
            held = set(kept)
            order = kept + [i for i in range(stride) if i not in held]
            assert table[g].tolist() == cache.table[g, order].tolist(), (keep, first, last, g)
            assert m1[g, :keep].nan_to_num(-1.0).tolist() == mass[g, kept].nan_to_num(-1.0).tolist()
            assert not m1[g, keep:].any()


def pool(ctx, gen, nKV, n, pages):
    """A cache whose lists name random pages (again and again) of random bounds."""
    import torch

    from momij_amd.kv8 import Kv8Cache

    cache = Kv8Cache(ctx, nKV, n)
    b = torch.randint(-127, 128, (pages, 2, D), generator=gen, device="cuda")
    cache.k_bounds[:pages] = torch.stack([b.amax(1), b.amin(1)], 1).to(torch.int8)
    cache.k_scale[:pages] = torch.rand(pages, generator=gen, device="cuda") + 0.1
    cache.table.copy_(torch.randint(0, pages, (nKV, n), generator=gen, device="cuda"))
    return cache


@pytest.mark.parametrize("M,nQ,nKV,n,n_sel,first,last", [
    (2, 8, 2, 513, 513, 1, 1), (2, 8, 2, 513, 600, 300, 300), (1, 4, 1, 1025, 1100, 0, 0), (2, 8, 2, 600, 2, 1, 1),
    (1, 4, 1, 16385, 16385, 2, 2), (1, 4, 1, 16385, 16400, 0, 9000), (1, 4, 1, 16385, 4, 1, 3),
    (64, 16, 4, 600, 9, 1, 2), (64, 20, 4, 1500, 33, 0, 1), (33, 64, 1, 700, 5, 1, 0), (64, 16, 16, 520, 70, 2, 2),
    (64, 16, 4, 512, 20, 1, 1)])
def test_select_ends(ctx, M, nQ, nKV, n, n_sel, first, last):
    import torch

    gen = generator(M + n)
    cache = pool(ctx, gen, nKV, n, min(400, nKV * n))
    q = torch.randn((M, nQ * D), generator=gen, device="cuda").half()
    sel = torch.full((M, nKV, n_sel), -9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_select(cache, q, M, nQ, n, n_sel, first, last, sel)
    ctx.sync()
    at = cache.table.long()
    sc = ref.scores(q.reshape(M, nKV, nQ // nKV, D), cache.k_bounds[at, 0].double(), cache.k_bounds[at, 1].double(),
                    cache.k_scale[at])
    sc[:, :, :first], sc[:, :, n - min(last, n):] = math.inf, math.inf
    # the first of equal scores: a stable descending order
    order = sc.sort(dim=-1, descending=True, stable=True).indices[..., :n_sel].sort(-1).values
    want = torch.full_like(sel, -1)
    want[..., :min(n, n_sel)] = order.int()
    assert torch.equal(sel, want)


@pytest.mark.parametrize("M,tree", [(1, False), (9, True)])
def test_block_over_a_long_list(ctx, M, tree):
    """The same pages in a short list, and far apart in one of 700 whose other entries name none: the
    same blocks are chosen (by the other kernels) and give the same bits."""
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    nQ, nKV, H, n, far, n_sel, cap = 16, 4, 2048, 20, 700, 6, 60
    rng, gen = np.random.default_rng(M), generator(M)
    cfg = dict(H=H, nQ=nQ, nKV=nKV, D=D, rope_dim=64, rope_base=1e6, eps=1e-6, window=0, C=0, gs=64)
    aw = {k: dev(v) for k, v in synth.attn_weights(rng, H, nQ, nKV, D, 64).items()}
    h0 = dev(synth.normal_f16(rng, (M, H)))
    parents = ref.tree(M, rng) if tree else None
    cache, src = Kv8Cache(ctx, nKV, far), [torch.randn((nKV, n * B, D), generator=gen, device="cuda").half()
                                           for _ in range(2)]
    kv = [torch.randn((nKV, cap, D), generator=gen, device="cuda").half() for _ in range(2)]
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(*src), 0, n, 0)
    ctx.sync()
    got = []
    for blocks in (n, far):
        if blocks == far:
            pages = cache.table[:, :n].clone()
            cache.table.fill_(-1)
            cache.table[:, torch.from_numpy(np.sort(rng.permutation(far)[:n])).cuda()] = pages
        h, rows = h0.clone(), [t.clone() for t in kv]
        torch.cuda.synchronize()
        ctx.attn_block_kv8(cfg, aw, cache, KvRing(*rows), h, blocks, n * B, n * B + 30, parents, M, n_sel=n_sel)
        ctx.sync()
        assert not torch.equal(h, h0)
        got.append([h] + rows)
    assert all(torch.equal(a, b) for a, b in zip(*got))
