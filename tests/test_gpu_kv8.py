"""GPU: the KV cache in 8 bits (appending, sealing, attention over pages and ring, chosen blocks,
eviction) against 64-bit statements of the same."""
import math

import numpy as np
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


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s: torch.randn(s, generator=g, device="cuda")


def cfg_of(nQ, nKV, rope=64, base=1e6):
    return dict(H=2048, nQ=nQ, nKV=nKV, D=D, rope_dim=rope, rope_base=base, eps=1e-6, window=0, C=0,
                gs=64)


# ------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("M,nQ,nKV,rope,L,C,kind", [
    (1, 16, 4, 64, 0, 1, "chain"), (1, 16, 4, 64, 131071, 128, "chain"),
    (64, 16, 4, 128, 1 << 40, 64, "tree"), (9, 12, 4, 32, 77, 13, "tree"), (5, 8, 8, 0, 1000, 6, "chain"),
    (17, 16, 1, 64, 3, 40, "tree"), (3, 3, 3, 128, 5, 3, "chain"), (33, 64, 1, 64, 99, 50, "chain")])
def test_append(ctx, M, nQ, nKV, rope, L, C, kind):
    import torch

    from momij_amd.kv8 import KvRing

    rnd = gen(M + nQ)
    rng = np.random.default_rng(M)
    parents = None if kind == "chain" else ref.tree(M, rng)
    wide = rnd(M, (nQ + 2 * nKV) * D + 64).half()
    qkv = wide[:, : (nQ + 2 * nKV) * D]  # rows of a wider matrix
    qw, kw = (1 + 0.2 * rnd(D)).half(), (1 + 0.2 * rnd(D)).half()
    k0, v0 = rnd(nKV, C, D).half(), rnd(nKV, C, D).half()
    k, v = k0.clone(), v0.clone()
    q = torch.full((M, nQ * D), 7.0, device="cuda").half()
    torch.cuda.synchronize()
    ctx.qkv_append(cfg_of(nQ, nKV, rope), qkv, qw, kw, KvRing(k, v), L, parents, M, q)
    ctx.sync()
    x = qkv.double().reshape(M, -1, D)
    depth = ref.sees(parents, M)[1]
    w = torch.cat([qw.double().expand(nQ, D), kw.double().expand(nKV, D)])
    y = x[:, : nQ + nKV]
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w
    z = y.clone()
    if rope:
        half = rope // 2
        f = 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
        # the reference's angles reduced in extended precision: position * turns, exactly enough
        pos = np.array([L + d for d in depth], dtype=np.longdouble)
        turns = pos[:, None] * (f.numpy().astype(np.longdouble) / (2 * np.longdouble(np.pi)))[None]
        th = torch.from_numpy(((turns - np.rint(turns)) * 2 * np.pi).astype(np.float64)).cuda()[:, None]
        a, b = y[..., :half], y[..., half:rope]
        z[..., :half] = a * th.cos() - b * th.sin()
        z[..., half:rope] = b * th.cos() + a * th.sin()
    # fp16 result; the norm in fp32 (a sum of 128 squares, a root, two products); the angle: position
    # * frequency within 2^-52 of itself, in turns, then sine and cosine within 2^-22
    ang = 2 * math.pi * (L + 64) * 0.16 * 2.0 ** -51 + 2.0 ** -21
    mag = y.abs().amax(-1, keepdim=True)
    tol = z.abs() * (ref.E16 + 140 * ref.E32) + 2 * mag * ang + 2.0 ** -24
    got = q.double().reshape(M, nQ, D)
    assert ((got - z[:, :nQ]).abs() <= tol[:, :nQ]).all()
    slots = [(L + r) % C for r in range(M)]
    gk = k.double()[:, slots].transpose(0, 1)
    assert ((gk - z[:, nQ:]).abs() <= tol[:, nQ:]).all()
    assert torch.equal(v[:, slots].transpose(0, 1), qkv.reshape(M, -1, D)[:, nQ + nKV:])
    other = [s for s in range(C) if s not in slots]
    assert torch.equal(k[:, other], k0[:, other]) and torch.equal(v[:, other], v0[:, other])


# -------------------------------------------------------------------------------------- seal
@pytest.mark.parametrize("nKV,count,at,pos,C", [(4, 1, 0, 0, 64), (4, 3, 2, 1000, 200), (1, 7, 0, 63, 449),
                                                (8, 2, 5, 1 << 40, 128)])
def test_seal_unseal(ctx, nKV, count, at, pos, C):
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    rnd = gen(C)
    k, v = (rnd(nKV, C, D) * 3).half(), (rnd(nKV, C, D) * 1e-3).half()
    k[0, pos % C, 5], k[0, (pos + 1) % C, 6], v[0, pos % C, 9] = math.inf, math.nan, -math.inf
    if count > 1:  # a block of zeros, and one whose greatest value is the least fp16 number
        k[nKV - 1, [(pos + 64 + i) % C for i in range(64)]] = 0.0
        v[nKV - 1, [(pos + 64 + i) % C for i in range(64)]] = 0.0
        v[nKV - 1, (pos + 64) % C, 3] = 2.0 ** -24
    cache = Kv8Cache(ctx, nKV, at + count + 1)
    pages = nKV * (at + count + 1)
    perm = torch.randperm(pages, device="cuda").to(torch.int32)
    cache.table.copy_(perm.reshape(nKV, -1))
    bad = int(cache.table[0, at].item())
    cache.table[0, at] = pages if count % 2 else -1  # names no page: neither written nor read back
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(77)
    cache.k_scale.fill_(-1.0)
    cache.v_scale.fill_(-1.0)
    back = [torch.full((nKV, C, D), 5.0, device="cuda").half() for _ in range(2)]
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(k, v), pos, count, at)
    ctx.kv8_unseal(cache, at, count, KvRing(*back), pos)
    ctx.sync()
    seen = set()
    for g in range(nKV):
        for i in range(count):
            slots = [(pos + 64 * i + j) % C for j in range(64)]
            pg = int(cache.table[g, at + i].item())
            if not 0 <= pg < pages:
                assert (back[0][g, slots] == 5.0).all() and (back[1][g, slots] == 5.0).all()
                continue
            seen.add(pg)
            for x, src in ((0, k), (1, v)):
                c, s = ref.seal(src[g, slots])
                codes, scale = ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale))[x]
                assert torch.equal(codes[pg], ref.page_bytes(c, x == 0)), (g, i, x)
                assert float(scale[pg]) == float(s)
                want = (c * s.double()).float().half()
                assert torch.equal(back[x][g, slots], want)
                if x == 0:
                    assert torch.equal(cache.k_bounds[pg].double(),
                                       torch.stack([c.amax(0), c.amin(0)]))
    for pg in range(pages):  # pages of other entries keep what they held
        if pg not in seen:
            assert (cache.k_codes[pg] == 77).all() and float(cache.v_scale[pg]) == -1.0, (pg, bad)


# --------------------------------------------------------------------------------- attention
class Ctx8:
    """A filled cache and ring with the float64 values they stand for."""

    def __init__(self, ctx, rnd, nKV, n, open_, M, start=None, extra=3, spread=1.0):
        import torch

        from momij_amd.kv8 import Kv8Cache, KvRing

        self.n, self.start = n, n * B if start is None else start
        self.L, self.M = self.start + open_, M
        self.C = C = open_ + M + extra
        self.cache = Kv8Cache(ctx, nKV, n + 2)
        pages = nKV * (n + 2)
        self.cache.table.copy_(torch.randperm(pages, device="cuda").to(torch.int32).reshape(nKV, -1))
        # pages nobody lists hold what must not be seen
        self.cache.k_codes.fill_(255)
        self.cache.v_codes.fill_(255)
        self.cache.k_scale.fill_(math.nan)
        self.cache.v_scale.fill_(math.inf)
        size = torch.exp(0.5 * rnd(nKV, 1, D))
        kk, vv = (rnd(nKV, max(n, 1) * B, D) * size * spread).half(), rnd(nKV, max(n, 1) * B, D).half()
        torch.cuda.synchronize()
        ctx.kv8_seal(self.cache, KvRing(kk, vv), 0, n, 0)
        ctx.sync()
        self.kc, ks = ref.seal(kk.reshape(nKV, -1, B, D)[:, :n])
        vc, vs = ref.seal(vv.reshape(nKV, -1, B, D)[:, :n])
        self.ks = ks
        self.k = (self.kc * ks.double()[..., None, None]).reshape(nKV, n * B, D)
        self.v = (vc * vs.double()[..., None, None]).reshape(nKV, n * B, D)
        rk, rv = (rnd(nKV, C, D) * size * spread).half(), rnd(nKV, C, D).half()
        self.slots = [(self.start + i) % C for i in range(open_ + M)]
        free = [s for s in range(C) if s not in self.slots]
        rk[:, free], rv[:, free] = math.nan, math.inf
        self.rk, self.rv, self.ring = rk, rv, KvRing(rk, rv)
        self.open = open_

    def keys(self, g):
        import torch

        return (torch.cat([self.k[g], self.rk[g, self.slots].double()]),
                torch.cat([self.v[g], self.rv[g, self.slots].double()]))

    def mask(self, parents, blocks=None):
        """[M, keys]: what each row may see; blocks [M][n] bool: the blocks a row reads."""
        import torch

        own = ref.sees(parents, self.M)[0]
        b = torch.ones((self.M, self.n), dtype=torch.bool) if blocks is None else blocks
        return torch.cat([b.repeat_interleave(B, 1), torch.ones((self.M, self.open), dtype=torch.bool),
                          own], 1).cuda()


def run_attn(ctx, c, q, nQ, nKV, parents, sel=None, mass=None, ws=None, ld_out=None):
    import torch

    M = c.M
    out = torch.full((M, ld_out or nQ * D), 9.0, device="cuda").half()
    mass_out = None if mass is None else torch.full_like(mass, -3.0)
    torch.cuda.synchronize()
    ctx.kv8_attn(c.cache, c.ring, q, M, nQ, c.n, c.start, c.L, parents, out, sel=sel, mass_in=mass,
                 mass_out=mass_out, ws=ws)
    ctx.sync()
    return out, mass_out


ATTN = [
    # M, nQ, nKV, blocks, open rows, tree
    (1, 16, 4, 0, 0, False),       # a first token: its own row alone
    (1, 16, 4, 1, 0, False), (1, 16, 4, 30, 80, False), (1, 8, 8, 5, 63, False),
    (2, 16, 1, 3, 64, False), (3, 12, 4, 7, 1, True), (4, 20, 4, 9, 5, True),
    (9, 16, 4, 17, 50, False), (17, 16, 4, 65, 17, True), (13, 6, 2, 33, 128, True),
    (33, 16, 2, 12, 0, True), (64, 16, 4, 20, 1, False), (64, 32, 4, 3, 130, True),
    (64, 64, 1, 2, 10, True), (5, 7, 1, 300, 77, False), (1, 64, 1, 40, 3, False),
    (16, 16, 4, 40, 0, False), (12, 16, 4, 41, 3, True), (64, 4, 4, 1, 0, True)]


@pytest.mark.parametrize("M,nQ,nKV,n,open_,tree", ATTN)
@pytest.mark.parametrize("mass", [False, True])
def test_attention(ctx, M, nQ, nKV, n, open_, tree, mass):
    import torch

    rnd = gen(M * 100 + n)
    c = Ctx8(ctx, rnd, nKV, n, open_, M)
    parents = ref.tree(M, np.random.default_rng(n)) if tree else None
    wide = rnd(M, nQ * D + 128).half()
    q = wide[:, 64:64 + nQ * D]
    m0 = torch.rand((nKV, n + 2), device="cuda") if mass else None
    out, m1 = run_attn(ctx, c, q, nQ, nKV, parents, mass=m0, ld_out=nQ * D + 8)
    G, ok = nQ // nKV, c.mask(parents)
    assert (out[:, nQ * D:] == 9.0).all()
    got = out[:, :nQ * D].double().reshape(M, nKV, G, D)
    for g in range(nKV):
        k, v = c.keys(g)
        qg = q.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D)
        want, p, tol, rel = ref.attention(qg, k, v, ok.repeat_interleave(G, 0))
        err = (got[:, g].reshape(M * G, D) - want).abs()
        assert (err <= tol).all(), float((err / tol).max())
        if mass:
            add = p[:, :n * B].reshape(M * G, n, B).sum(2)
            want = m0[g, :n].double() + add.sum(0)
            # weights within rel and two exponentials' last places; a sum over the rows' heads
            tol = (add * (rel + 2.0 ** -20)).sum(0) + want * (M * G + 4) * ref.E32 + 1e-30
            assert ((m1[g, :n].double() - want).abs() <= tol).all()
            assert (m1[g, n:] == -3.0).all()  # entries past the blocks are left as they were


@pytest.mark.parametrize("nQ,nKV,M,open_,start", [(16, 4, 9, 100, 1 << 33), (16, 4, 1, 63, 12345)])
def test_attention_far_positions(ctx, nQ, nKV, M, open_, start):
    """The ring's slots at positions past 32 bits, in a ring that wraps."""
    rnd = gen(3)
    c = Ctx8(ctx, rnd, nKV, 4, open_, M, start=start, extra=0)
    q = rnd(M, nQ * D).half()
    out, _ = run_attn(ctx, c, q, nQ, nKV, None)
    check_rows(c, q, out, nQ, nKV, c.mask(None))


def check_rows(c, q, out, nQ, nKV, ok, rows=None):
    G, M = nQ // nKV, c.M
    for g in range(nKV):
        k, v = c.keys(g)
        qg = q.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D)
        want, _, tol, _ = ref.attention(qg, k, v, (ok if ok.dim() == 2 else ok[g]).repeat_interleave(G, 0))
        err = (out.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D) - want).abs()
        bad = ~(err <= tol)
        if rows is not None:
            bad = bad.reshape(M, G, D)[rows]
        assert not bad.any(), float((err / tol).max())


def test_large_scores(ctx):
    """Scores of several hundred, the running maximum moving from block to block."""
    rnd = gen(8)
    for M, n in ((1, 40), (9, 40), (64, 12)):
        c = Ctx8(ctx, rnd, 4, n, 30, M, spread=12.0)
        q = (rnd(M, 16 * D) * 6).half()
        out, _ = run_attn(ctx, c, q, 16, 4, None)
        check_rows(c, q, out, 16, 4, c.mask(None))


@pytest.mark.parametrize("M", [3, 17, 64])
def test_values_out_of_sight(ctx, M):
    """Infinities and NaN in K and V of pass rows: the rows that do not descend from them are as if
    they were not there, those that do show them."""
    import torch

    rnd = gen(M)
    c = Ctx8(ctx, rnd, 4, 6, 20, M)
    parents = [-1] + [0] * (M - 1)  # siblings
    bad = [1, M - 1]
    c.rk[:, [c.slots[c.open + b] for b in bad]] = math.nan
    c.rv[0, c.slots[c.open + 1], 3:9] = math.inf
    c.rv[1:, c.slots[c.open + M - 1]] = math.nan
    q = rnd(M, 16 * D).half()
    out, _ = run_attn(ctx, c, q, 16, 4, parents)
    keep = [r for r in range(M) if r not in bad]
    assert not out[keep].isnan().any()
    clean = c.rk.clone(), c.rv.clone()
    for t in (c.rk, c.rv):
        t[:, [c.slots[c.open + b] for b in bad]] = 0.0
    check_rows(c, q, out, 16, 4, c.mask(parents), rows=keep)
    assert out[bad].isnan().all()
    # finite keys, an infinity in one value: it shows in its dims alone
    c.rk.copy_(torch.where(clean[0].isnan(), torch.zeros_like(clean[0]), clean[0]))
    c.rv[0, c.slots[c.open + 1], 3:9] = math.inf
    out, _ = run_attn(ctx, c, q, 16, 4, parents)
    o = out.reshape(M, 16, D)
    assert (o[1, :4, 3:9] == math.inf).all() and o[1, :4, 9:].isfinite().all() and o[1, 4:].isfinite().all()
    assert o[keep].isfinite().all()
    # every row sees an infinity among the committed ones
    c.rv[2, c.slots[0], 7] = -math.inf
    out, _ = run_attn(ctx, c, q, 16, 4, parents)
    assert (out.reshape(M, 16, D)[:, 8:12, 7] == -math.inf).all()


def test_nan_query(ctx):
    rnd = gen(4)
    for M in (1, 9, 64):
        c = Ctx8(ctx, rnd, 4, 9, 10, M)
        q = rnd(M, 16 * D).half()
        q[M - 1, :D] = math.nan
        out, _ = run_attn(ctx, c, q, 16, 4, None)
        o = out.reshape(M, 16, D)
        assert o[M - 1, 0].isnan().all() and o[M - 1, 1:].isfinite().all() and o[:M - 1].isfinite().all()


@pytest.mark.parametrize("M", [1, 9, 40])
def test_bad_pages(ctx, M):
    """Table entries outside the pool name no block: the rest is attended, masses stay."""
    import torch

    rnd = gen(11)
    n, nQ, nKV = 12, 16, 4
    c = Ctx8(ctx, rnd, nKV, n, 7, M)
    pages = nKV * (n + 2)
    gone = {0: [0, 5], 1: [11], 2: list(range(n)), 3: []}
    for g, ids in gone.items():
        for j, i in enumerate(ids):
            c.cache.table[g, i] = [pages, -1, 2 ** 31 - 1, -2 ** 31][j % 4]
    q = rnd(M, nQ * D).half()
    m0 = torch.rand((nKV, n + 2), device="cuda")
    out, m1 = run_attn(ctx, c, q, nQ, nKV, None, mass=m0)
    ok = c.mask(None)[None].repeat(nKV, 1, 1)
    for g, ids in gone.items():
        for i in ids:
            ok[g, :, i * B:(i + 1) * B] = False
            assert m1[g, i] == m0[g, i]
    check_rows(c, q, out, nQ, nKV, ok)


# -------------------------------------------------------------------------------- selection
SEL = [
    # M, nQ, nKV, blocks, n_sel, first, last, open
    (1, 16, 4, 40, 8, 1, 2, 30), (9, 16, 4, 130, 16, 1, 2, 50), (3, 12, 4, 7, 7, 0, 0, 0),
    (2, 16, 1, 65, 1, 0, 0, 5), (5, 64, 1, 20, 3, 1, 1, 5), (1, 8, 8, 3, 9, 1, 1, 9),
    (17, 20, 4, 33, 12, 2, 3, 17), (64, 16, 4, 50, 5, 0, 1, 1), (1, 16, 4, 2047, 64, 1, 2, 3),
    (4, 16, 4, 0, 3, 1, 1, 5), (7, 28, 4, 9, 4, 2, 2, 2)]


@pytest.mark.parametrize("M,nQ,nKV,n,n_sel,first,last,open_", SEL)
def test_select_and_attend(ctx, M, nQ, nKV, n, n_sel, first, last, open_):
    import torch

    rnd = gen(n + M)
    c = Ctx8(ctx, rnd, nKV, n, open_, M)
    G = nQ // nKV
    wide = rnd(M, nQ * D + 64).half()
    q = wide[:, :nQ * D]
    sel = torch.full((M, nKV, n_sel), -9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_select(c.cache, q, M, nQ, n, n_sel, first, last, sel)
    ctx.sync()
    sc = ref.scores(q.reshape(M, nKV, G, D), c.kc.amax(2), c.kc.amin(2), c.ks).cpu() if n else None
    blocks = torch.zeros((nKV, M, n), dtype=torch.bool)
    for r in range(M):
        for g in range(nKV):
            want = ref.choose(sc[r, g].tolist(), first, last, min(n_sel, n)) if n else []
            assert sel[r, g].tolist() == want + [-1] * (n_sel - len(want)), (r, g)
            blocks[g, r, want] = True
    parents = ref.tree(M, np.random.default_rng(M))
    out, _ = run_attn(ctx, c, q, nQ, nKV, parents, sel=sel)
    ok = torch.stack([c.mask(parents, blocks[g]) for g in range(nKV)])
    check_rows(c, q, out, nQ, nKV, ok)


def test_select_ties_and_nan(ctx):
    """Equal blocks: the lowest indices; zero queries: every score 0; NaN scales and pages outside the
    pool count as the least; infinite and NaN query values have the codes a sealed one has."""
    import torch

    rnd = gen(5)
    M, n, n_sel = 6, 90, 10
    c = Ctx8(ctx, rnd, 1, n, 4, M)
    for i in range(n):  # three kinds of block
        c.cache.table[0, i] = c.cache.table[0, i % 3]
    c.kc, c.ks = c.kc[:, [i % 3 for i in range(n)]], c.ks[:, [i % 3 for i in range(n)]]
    q = rnd(M, 4 * D).half()
    q[1] = 0.0
    q[2, 5], q[2, 7], q[3, :] = math.inf, math.nan, math.nan
    sel = torch.empty((M, 1, n_sel), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_select(c.cache, q, M, 4, n, n_sel, 0, 0, sel)
    ctx.sync()
    sc = ref.scores(q.reshape(M, 1, 4, D), c.kc.amax(2), c.kc.amin(2), c.ks).cpu()
    for r in range(M):
        assert sel[r, 0].tolist() == ref.choose(sc[r, 0].tolist(), 0, 0, n_sel)
    assert sel[1, 0].tolist() == list(range(n_sel))
    c.cache.k_scale[c.cache.table[0, 1].long()] = math.nan
    c.cache.table[0, 0] = -1
    torch.cuda.synchronize()
    ctx.kv8_select(c.cache, q, M, 4, n, n_sel, 0, 0, sel)
    ctx.sync()
    sc[:, :, 1::3] = -math.inf
    sc[:, :, 0] = -math.inf
    for r in range(M):
        assert sel[r, 0].tolist() == ref.choose(sc[r, 0].tolist(), 0, 0, n_sel)


def test_lists_of_the_caller(ctx):
    """Lists with gaps, indices outside the blocks, and one block twice (it counts twice)."""
    import torch

    rnd = gen(6)
    M, nQ, nKV, n = 3, 16, 4, 10
    c = Ctx8(ctx, rnd, nKV, n, 5, M)
    lists = [[3, -1, 7, n, 2 ** 31 - 1], [-5, -1, -1, -1, -1], [0, 9, 9, -1, 4]]
    sel = torch.tensor(lists, dtype=torch.int32, device="cuda")[:, None].repeat(1, nKV, 1).contiguous()
    q = rnd(M, nQ * D).half()
    out, _ = run_attn(ctx, c, q, nQ, nKV, None, sel=sel)
    G = nQ // nKV
    own = ref.sees(None, M)[0]
    for g in range(nKV):
        for r in range(M):
            rows = [i * B + j for i in lists[r] if 0 <= i < n for j in range(B)]
            k, v = c.keys(g)
            tail = [n * B + j for j in range(c.open)] + [n * B + c.open + j for j in range(M) if own[r, j]]
            at = torch.tensor(rows + tail, device="cuda")
            qg = q.double().reshape(M, nKV, G, D)[r, g]
            want, _, tol, _ = ref.attention(qg, k[at], v[at], torch.ones((G, len(at)), dtype=torch.bool,
                                                                          device="cuda"))
            assert ((out.double().reshape(M, nKV, G, D)[r, g] - want).abs() <= tol).all()


# --------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("nKV,n,keep,first,last,stride", [
    (4, 65, 64, 1, 4, 65), (1, 1, 0, 0, 0, 3), (4, 0, 0, 0, 0, 2), (2, 10, 10, 3, 3, 12),
    (8, 300, 7, 2, 5, 301), (3, 2047, 1024, 1, 16, 2050), (1, 5000, 4999, 0, 0, 5000),
    (4, 64, 1, 0, 0, 64)])
def test_evict(ctx, nKV, n, keep, first, last, stride):
    import torch

    from momij_amd.kv8 import Kv8Cache

    rnd = gen(n + keep)
    cache = Kv8Cache(ctx, nKV, stride)
    cache.table.copy_(torch.stack([torch.randperm(stride, device="cuda") + g * stride
                                   for g in range(nKV)]).to(torch.int32))
    mass = rnd(nKV, stride).abs()
    mass[:, ::3] = 0.25  # ties
    mass[:, 1::11] = math.nan
    mass[:, 2::13] = math.inf
    mass[:, 5::17] = -0.0
    mass[:, 6::17] = 0.0
    table, m1 = torch.empty_like(cache.table), torch.empty_like(mass)
    torch.cuda.synchronize()
    ctx.kv8_evict(cache, n, keep, first, last, mass, table, m1)
    ctx.sync()
    for g in range(nKV):
        kept = ref.choose([float(x) for x in mass[g, :n]], first, last, keep)
        order = kept + [i for i in range(n) if i not in set(kept)] + list(range(n, stride))
        assert table[g].tolist() == cache.table[g, order].tolist()
        want = torch.zeros(stride)
        want[:keep] = mass[g, kept].cpu()
        assert torch.equal(m1[g].cpu().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("n", [1, 64, 1023, 1024, 1025, 2048, 2049, 4096, 4097, 16384, 16385])
@pytest.mark.parametrize("pages,nQ", [(40, 4), (1000, 16), (300, 48)])
def test_select_long_lists(ctx, n, pages, nQ):
    """Lists of every length class; blocks listed again and again tie."""
    import torch

    from momij_amd.kv8 import Kv8Cache

    rnd = gen(n + pages)
    M, n_sel, first, last = 3, min(n, 57), 1, 0
    cache = Kv8Cache(ctx, 1, max(n, pages))
    hi = (rnd(pages, D) * 30 + 40).round().clamp(-127, 127)
    lo = torch.minimum(hi, (rnd(pages, D) * 30 - 40).round().clamp(-127, 127))
    cache.k_bounds[:pages] = torch.stack([hi, lo], 1).to(torch.int8)
    cache.k_scale[:pages] = torch.exp(0.5 * rnd(pages)) * 0.01
    at = torch.randint(0, pages, (n,), device="cuda", dtype=torch.int32)
    cache.table[0, :n] = at
    q = rnd(M, nQ * D).half()
    sel = torch.empty((M, 1, n_sel), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_select(cache, q, M, nQ, n, n_sel, first, last, sel)
    ctx.sync()
    sc = ref.scores(q.reshape(M, 1, nQ, D), hi[None].double(), lo[None].double(),
                    cache.k_scale[None, :pages])[:, 0, at.long()].cpu()
    for r in range(M):
        assert sel[r, 0].tolist() == ref.choose(sc[r].tolist(), first, last, n_sel)


@pytest.mark.parametrize("n", [1024, 1025, 4096, 4097, 16384, 16385])
@pytest.mark.parametrize("kind", ["wide", "equal", "two", "near", "negative"])
def test_evict_long_lists(ctx, n, kind):
    import torch

    from momij_amd.kv8 import Kv8Cache

    rnd = gen(n)
    cache = Kv8Cache(ctx, 2, n)
    x = rnd(2, n)
    mass = dict(wide=torch.exp(20 * x), equal=torch.full_like(x, 3.0), two=(x > 0.5).float(),
                near=1.0 + x.abs() * 1e-6, negative=x * torch.exp(30 * rnd(2, n)))[kind]
    for keep in (1, n // 3, n - 1):
        table, m1 = torch.empty_like(cache.table), torch.empty_like(mass)
        torch.cuda.synchronize()
        ctx.kv8_evict(cache, n, keep, 0, 1, mass, table, m1)
        ctx.sync()
        for g in range(2):
            kept = ref.choose(mass[g].tolist(), 0, 1, keep)
            order = kept + sorted(set(range(n)) - set(kept))
            assert table[g].tolist() == cache.table[g, order].tolist(), (keep, g)
            assert torch.equal(m1[g, :keep], mass[g, kept]) and not m1[g, keep:].any()
