"""GPU: attention over 8-bit pages where a block's pages come in several batches, and where a call has
more parts than one round of the join takes.  Sizes are chosen by the restated split (kv8_plan)."""
import numpy as np
import pytest

from tests import kv8_ref as ref
from tests.kv8_plan import plan

pytestmark = pytest.mark.gpu
D, B = 128, 64


@pytest.fixture(scope="module")
def ctx():
    from momij_amd.ops import Context

    c = Context(0)
    yield c
    c.close()


def check(ctx, M, nQ, nKV, n, open_, tree, lost=()):
    """Outputs and masses against 64 bits; lost: blocks that name no page in every second head."""
    import torch

    from tests.test_gpu_kv8 import Ctx8, gen, run_attn
    from tests.test_gpu_kv8_flow import attend

    rnd, G = gen(M + n), nQ // nKV
    c = Ctx8(ctx, rnd, nKV, n, open_, M)
    parents = ref.tree(M, np.random.default_rng(n)) if tree else None
    gone = [list(lost) if g % 2 == 0 else [] for g in range(nKV)]
    for g in range(nKV):
        if gone[g]:
            c.cache.table[g, gone[g]] = torch.tensor([-1, nKV * (n + 2)], dtype=torch.int32, device="cuda")[
                torch.arange(len(gone[g]), device="cuda") % 2]
    q = rnd(M, nQ * D).half()
    m0 = torch.rand((nKV, n + 2), device="cuda")
    for mass in (None, m0):
        out, m1 = run_attn(ctx, c, q, nQ, nKV, parents, mass=mass)
        again, m2 = run_attn(ctx, c, q, nQ, nKV, parents, mass=mass)
        assert torch.equal(out, again) and (mass is None or torch.equal(m1, m2))
        for g in range(nKV):
            ok = c.mask(parents)
            for i in gone[g]:
                ok[:, i * B:(i + 1) * B] = False
            want, p, tol, rel = attend(q.reshape(M, nKV, G, D)[:, g], *c.keys(g), ok, G)
            err = (out.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D) - want).abs()
            assert (err <= tol).all(), (g, float((err / tol).max()))
            if mass is not None:
                add = p[:, :n * B].reshape(M * G, n, B).sum(2)
                want = m0[g, :n].double() + add.sum(0)
                tol = (add * (rel + 2.0 ** -20)).sum(0) + want * (M * G + 4) * ref.E32 + 1e-30
                assert ((m1[g, :n].double() - want).abs() <= tol).all(), g
                assert all(m1[g, i] == m0[g, i] for i in gone[g])


BATCHES = [
    # M, nQ, nKV, blocks, open rows, tree; shared, tiles a wave, waves a page
    (20, 256, 64, 200, 5, False, True, 1, 1), (20, 256, 64, 130, 70, True, True, 1, 1),
    (64, 256, 64, 300, 10, True, True, 2, 1), (1, 128, 128, 520, 9, False, False, 1, 1),
    (20, 128, 128, 530, 3, True, False, 2, 1), (40, 128, 128, 300, 20, False, False, 2, 2)]


@pytest.mark.parametrize("M,nQ,nKV,n,open_,tree,shared,tiles,pair", BATCHES)
@pytest.mark.parametrize("lost", [False, True])
def test_batches(ctx, M, nQ, nKV, n, open_, tree, shared, tiles, pair, lost):
    """Two batches of pages and more; lost: the first batch without a page, and the last block."""
    p = plan(nQ, nKV, M, n, 0, open_ + M, False)
    assert (p["shared"], p["tiles"], p["pair"]) == (shared, tiles, pair) and p["upp"] > p["batch"]
    check(ctx, M, nQ, nKV, n, open_, tree, list(range(p["batch"])) + [n - 1] if lost else ())


@pytest.mark.parametrize("M,nQ,nKV,n,n_sel", [(64, 16, 4, 700, 600), (40, 32, 8, 560, 540), (64, 192, 4, 300, 290)])
def test_batches_of_listed_blocks(ctx, M, nQ, nKV, n, n_sel):
    import torch

    from tests.test_gpu_kv8 import Ctx8, check_rows, gen, run_attn

    p = plan(nQ, nKV, M, n, n_sel, 20 + M, False)
    assert not p["shared"] and p["upp"] > p["batch"]
    rnd = gen(nQ)
    c = Ctx8(ctx, rnd, nKV, n, 20, M)
    rng = np.random.default_rng(n)
    sel = np.stack([[np.sort(rng.permutation(n)[:n_sel]) for _ in range(nKV)] for _ in range(M)])
    blocks = torch.zeros((M, nKV, n), dtype=torch.bool).scatter_(2, torch.from_numpy(sel), True)
    q = rnd(M, nQ * D).half()
    out, _ = run_attn(ctx, c, q, nQ, nKV, None, sel=torch.from_numpy(sel.astype(np.int32)).cuda())
    check_rows(c, q, out, nQ, nKV, torch.stack([c.mask(None, blocks[:, g]) for g in range(nKV)]))


@pytest.mark.parametrize("M,nQ,nKV,n,open_", [(1, 16, 1, 200, 16000), (2, 16, 1, 2000, 16300)])
def test_more_parts_than_a_round(ctx, M, nQ, nKV, n, open_):
    """More than 256 parts: a second round of the join's groups, and of the masses'."""
    assert plan(nQ, nKV, M, n, 0, open_ + M, True)["parts"] > 256
    check(ctx, M, nQ, nKV, n, open_, False)


@pytest.mark.parametrize("M,nQ,nKV,n,open_", [(1, 16, 4, 40, 5000), (9, 16, 4, 300, 4200), (3, 64, 64, 9, 700),
                                              (64, 16, 4, 2, 2100), (2, 8, 1, 5, 20000)])
def test_masses_beside_long_rings(ctx, M, nQ, nKV, n, open_):
    check(ctx, M, nQ, nKV, n, open_, M > 2)
