"""GPU: attention of a batch's rows over the pages of their sequences, and the rows' append, against plain
forms in 64 bits (tests/paged_ref.py)."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R
from momij_amd.ops import Context
from momij_amd.paged import PagedCache, RowBatch, tree_masks

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    with torch.cuda.stream(c.stream):
        yield c
    c.close()


def cuda(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def make(ctx, lens, rows, page=64, nkv=4, layers=1, seed=0, spare=1, extra=3, scale=1.0):
    """A cache whose sequences hold `lens` tokens and have pages for `rows` more; every place of the pool that
    no token has is a NaN.  Pages lie anywhere."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    blocks = [-(-(x + m) // page) for x, m in zip(lens, rows)]
    n_pages, width = sum(blocks) + extra, max(blocks + [1]) + spare
    shape = (layers, n_pages, nkv, page // 32, 4096)
    k, v = (torch.full(shape, math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    table = np.full((len(lens), width), -1, np.int64)
    perm = rng.permutation(n_pages)
    for s, b in enumerate(blocks):
        table[s, :b] = perm[sum(blocks[:s]):sum(blocks[:s + 1])]
    refs = np.zeros(n_pages, np.int64)
    refs[table[table >= 0]] = 1
    cache = PagedCache.over(ctx, k, v, cuda(table), cuda(lens), cuda(refs))
    for layer in range(layers):
        for s, (x, m) in enumerate(zip(lens, rows)):
            if x + m:
                kk, vv = (torch.randn((x + m, nkv, D), generator=gen, device="cuda") * scale for _ in range(2))
                R.put(cache, layer, s, torch.arange(x + m, device="cuda"), kk, vv)
    return cache, gen, rng


def batch_of(rows, parents=None, max_rows=None, pad=0):
    start = np.concatenate([[0], np.cumsum(rows)])
    anc = None
    if parents is not None:
        anc = cuda([a for p in parents for a in tree_masks(p)] + [-1] * pad, torch.int64)
    return RowBatch(cuda(start), int(start[-1]) + pad, max_rows or max(max(rows), 1), anc)


def check(cache, rows, sees, q, out, nq, window=0, layer=0, holes=()):
    """sees[s][r]: the rows that row r of sequence s sees."""
    nkv, G, at = cache.n_kv_heads, nq // cache.n_kv_heads, 0
    lens = cache.lens.tolist()
    worst = 0.0
    for s, m in enumerate(rows):
        if m == 0:
            continue
        L = lens[s]
        k, v = R.rows_of(cache, layer, s, torch.arange(L + m, device="cuda"))
        gone = torch.zeros(L + m, dtype=torch.bool, device="cuda")
        for j in [j for t, j in holes if t == s]:
            gone[j * cache.page_tokens:(j + 1) * cache.page_tokens] = True
        ok = torch.zeros((m, L + m), dtype=torch.bool, device="cuda")
        for r in range(m):
            ok[r, torch.tensor(R.seen(L, sees[s][r], window) if sees[s][r] else list(range(L)), device="cuda",
                               dtype=torch.long)] = True
        ok &= ~gone
        qs = q[at:at + m].double().reshape(m, nkv, G, D)
        got = out[at:at + m].double().reshape(m, nkv, G, D)
        for g in range(nkv):
            ref, _, tol, _ = R.attention(qs[:, g].reshape(m * G, D), k[:, g], v[:, g],
                                         ok.repeat_interleave(G, 0))
            err = (got[:, g].reshape(m * G, D) - ref).abs()
            assert not bool(err.isnan().any()), (s, g)
            worst = max(worst, float((err / tol).max()))
        at += m
    assert worst <= 1.0, worst


def chains(rows):
    return [R.ways(R.tree(m)) if m else [] for m in rows]


HEADS = [(16, 4), (8, 8), (16, 1), (12, 4), (64, 1), (4, 4), (32, 4)]
LENS = [[0], [1], [31, 32, 33], [63, 0, 64, 65, 200], [700, 3, 129, 1, 256, 95, 40]]


@pytest.mark.parametrize("nq,nkv", HEADS)
@pytest.mark.parametrize("page", [32, 64, 128, 256])
def test_decode(ctx, nq, nkv, page):
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 500, 1000]
    rows = [1] * len(lens)
    cache, gen, _ = make(ctx, lens, rows, page, nkv, seed=nq + page)
    q = (torch.randn((len(lens), nq * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of(rows), q, nq, out)
    check(cache, rows, chains(rows), q, out, nq)


@pytest.mark.parametrize("M", [2, 4, 5, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("nq,nkv", [(16, 4), (8, 8), (16, 1), (12, 4)])
@pytest.mark.parametrize("lens", LENS[2:], ids=str)
def test_trees_and_chains(ctx, M, nq, nkv, lens):
    rows = [max(1, M - 3 * i) if i != 1 else M for i in range(len(lens))]
    cache, gen, rng = make(ctx, lens, rows, 32, nkv, seed=M)
    parents = [R.tree(m, rng) for m in rows]
    q = (torch.randn((sum(rows), nq * D), generator=gen, device="cuda") * 2).half()
    for par in (parents, None):
        out = torch.full_like(q, 7.0)
        ctx.paged_attn(cache, 0, batch_of(rows, par), q, nq, out)
        check(cache, rows, [R.ways(p) for p in parents] if par else chains(rows), q, out, nq)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 512, 5000])
@pytest.mark.parametrize("M", [1, 9, 40])
def test_window(ctx, window, M):
    lens, rows = [0, 5, 64, 333, 1200], [M, M, 1, M, M]
    cache, gen, rng = make(ctx, lens, rows, 64, 4, seed=window)
    parents = [R.tree(m, rng) for m in rows]
    q = (torch.randn((sum(rows), 16 * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    # blocks behind every row's window may be gone
    for s, L in enumerate(lens):
        gone = max(0, L - window + 1) // 64
        cache.table[s, :gone] = -1
    ctx.paged_attn(cache, 0, batch_of(rows, parents), q, 16, out, window=window)
    check(cache, rows, [R.ways(p) for p in parents], q, out, 16, window)


@pytest.mark.parametrize("L,M,nq", [(131000, 1, 16), (131001, 9, 16), (40000, 17, 16), (20000, 64, 16),
                                    (9000, 64, 64)])
def test_long(ctx, L, M, nq):
    cache, gen, _ = make(ctx, [L, 70], [M, 1], 64, 4, seed=L)
    q = (torch.randn((M + 1, nq * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of([M, 1]), q, nq, out)
    check(cache, [M, 1], chains([M, 1]), q, out, nq)
    again = torch.full_like(q, 5.0)
    ctx.paged_attn(cache, 0, batch_of([M, 1]), q, nq, again)
    assert torch.equal(out, again)


@pytest.mark.parametrize("M,nq", [(1, 16), (3, 16), (9, 16), (64, 16)])
def test_uneven_batch(ctx, M, nq):
    """One sequence of most of the work among many of little, some of no rows."""
    lens = [20 * (i % 7) for i in range(61)] + [30000]
    rows = [0 if i % 5 == 2 else 1 + i % M for i in range(61)] + [M]
    cache, gen, _ = make(ctx, lens, rows, 64, 4, seed=M)
    q = (torch.randn((sum(rows), nq * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of(rows), q, nq, out)
    check(cache, rows, chains(rows), q, out, nq)


@pytest.mark.parametrize("M,hole", [(1, None), (3, None), (5, 1300), (9, None), (17, 1301), (64, None), (64, 2040)])
def test_runs_of_many_units(ctx, M, hole):
    """So much work that a block's run is longer than the page numbers it holds at once; 24 sequences with the
    pages of one.  hole: a block of the table that names no page (units are missing in the middle of a run)."""
    L, n = 131000 - M, 24
    one, gen, _ = make(ctx, [L], [M], 64, 4, seed=M)
    table = one.table.repeat(n, 1).contiguous()
    if hole is not None:
        table[:, hole] = -1
    cache = PagedCache.over(ctx, one.k, one.v, table, one.lens.repeat(n), one.refs)
    q = (torch.randn((n * M, 16 * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of([M] * n), q, 16, out)
    src = one  # (its own table still names every page: the reference leaves the hole out itself)
    for s in (0, 1, 11, n - 1):
        check(src, [M], chains([M]), q[s * M:(s + 1) * M], out[s * M:(s + 1) * M], 16,
              holes=[] if hole is None else [(0, hole)])


def test_1024_sequences(ctx):
    lens = [(37 * i) % 90 for i in range(1024)]
    rows = [1 + (i % 3 == 0) for i in range(1024)]
    cache, gen, _ = make(ctx, lens, rows, 32, 1, seed=3)
    q = (torch.randn((sum(rows), 4 * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of(rows), q, 4, out)
    check(cache, rows, chains(rows), q, out, 4)


@pytest.mark.parametrize("M,nq", [(1, 16), (5, 16), (12, 16), (64, 16)])
def test_layers_strides_and_rows_left_alone(ctx, M, nq):
    lens, rows = [100, 0, 33], [M, 1, M]
    cache, gen, _ = make(ctx, lens, rows, 64, 4, layers=3, seed=9)
    n = sum(rows)
    wide = (torch.randn((n + 2, nq * D + 40), generator=gen, device="cuda") * 2).half()
    dest = torch.full((n + 2, nq * D + 24), 7.0, dtype=torch.float16, device="cuda")
    q, out = wide[:, 16:16 + nq * D], dest[:, 8:8 + nq * D]
    ctx.paged_attn(cache, 2, batch_of(rows, pad=2), q, nq, out)
    check(cache, rows, chains(rows), q, out, nq, layer=2)
    assert bool((dest[n:] == 7).all()) and bool((dest[:, :8] == 7).all()) and bool((dest[:, 8 + nq * D:] == 7).all())
    # rows past max_rows
    if M > 1:
        dest.fill_(7.0)
        ctx.paged_attn(cache, 2, batch_of(rows, max_rows=M - 1), q[:n], nq, out[:n])
        assert bool((dest[M - 1] == 7).all()) and not bool((out[M - 2] == 7).any())
        assert bool((dest[n - 1] == 7).all())


@pytest.mark.parametrize("M,nq", [(1, 16), (9, 16), (40, 16)])
def test_pages_that_are_not_there(ctx, M, nq):
    lens, rows = [500, 64, 300], [M, M, M]
    cache, gen, _ = make(ctx, lens, rows, 64, 4, seed=5)
    q = (torch.randn((3 * M, nq * D), generator=gen, device="cuda") * 2).half()
    out = torch.full_like(q, 7.0)
    cache.table[0, 2], cache.table[0, 3], cache.table[2, 0] = -1, cache.n_pages, 2 ** 31 - 1
    cache.table[1, :] = -5
    ctx.paged_attn(cache, 0, batch_of(rows), q, nq, out)
    check(cache, rows, chains(rows), q, out, nq, holes=[(0, 2), (0, 3), (2, 0)] + [(1, j) for j in range(3)])
    assert bool((out[M:2 * M] == 0).all())


def test_rows_that_see_nothing(ctx):
    lens, rows = [0, 40], [4, 3]
    cache, gen, _ = make(ctx, lens, rows, 32, 4, seed=6)
    q = torch.randn((7, 16 * D), generator=gen, device="cuda").half()
    out = torch.full_like(q, 7.0)
    # row 1 of the first: nothing; row 2: rows 0 and 2; row 3: a row that there is not, and itself
    masks = [1, 0, 0b101, 1 << 20 | 0b1000, 0, 0b11, 0b100]
    b = RowBatch(cuda([0, 4, 7]), 7, 4, cuda(masks, torch.int64))
    ctx.paged_attn(cache, 0, b, q, 16, out)
    assert bool((out[1] == 0).all())
    k, v = R.rows_of(cache, 0, 0, torch.arange(4, device="cuda"))
    ok = torch.tensor([[1, 0, 0, 0], [0, 0, 0, 0], [1, 0, 1, 0], [0, 0, 0, 1]], dtype=torch.bool, device="cuda")
    for g in range(4):
        ref, _, tol, _ = R.attention(q[:4].double().reshape(4, 4, 4, D)[:, g].reshape(16, D), k[:, g], v[:, g],
                                     ok.repeat_interleave(4, 0))
        got = out[:4].double().reshape(4, 4, 4, D)[:, g].reshape(16, D)
        assert bool(((got - ref).abs() <= tol).all())
    k, v = R.rows_of(cache, 0, 1, torch.arange(43, device="cuda"))
    ok = torch.ones((3, 43), dtype=torch.bool, device="cuda")
    ok[:, 40:] = torch.tensor([[0, 0, 0], [1, 1, 0], [0, 0, 1]], dtype=torch.bool, device="cuda")
    for g in range(4):
        ref, _, tol, _ = R.attention(q[4:].double().reshape(3, 4, 4, D)[:, g].reshape(12, D), k[:, g], v[:, g],
                                     ok.repeat_interleave(4, 0))
        got = out[4:].double().reshape(3, 4, 4, D)[:, g].reshape(12, D)
        assert bool(((got - ref).abs() <= tol).all())


@pytest.mark.parametrize("L", [0, 30, 64, 500])
@pytest.mark.parametrize("nq", [4, 16, 64])
def test_infinities_out_of_sight_and_in_sight(ctx, L, nq):
    """K and V of rows that others do not see hold NaN and infinities: these rows' results are as if they
    did not, and rows that see an infinity of V give one."""
    M = 9
    cache, gen, rng = make(ctx, [L], [M], 64, 4, seed=L)
    parents = [-1, 0, 0, 1, 2, 2, 4, 3, 0]
    ways = R.ways(parents)
    bad_v, bad_k = 2, 5  # rows whose V, whose K and V are bad
    k, v = R.rows_of(cache, 0, 0, torch.arange(L, L + M, device="cuda"))
    k, v = k.clone(), v.clone()
    v[bad_v, :, ::2], v[bad_v, :, 1::4] = math.inf, -math.inf
    k[bad_k], v[bad_k] = math.nan, math.nan
    R.put(cache, 0, 0, torch.arange(L, L + M, device="cuda"), k, v)
    q = torch.randn((M, nq * D), generator=gen, device="cuda").half()
    out = torch.full_like(q, 7.0)
    ctx.paged_attn(cache, 0, batch_of([M], [parents]), q, nq, out)
    got = out.double().reshape(M, nq, D)
    for r in range(M):
        if bad_k in ways[r]:
            assert bool(got[r].isnan().all())
        elif bad_v in ways[r]:
            assert bool((got[r, :, ::2] == math.inf).all()) and bool((got[r, :, 1::4] == -math.inf).all())
            assert bool(got[r, :, 3::4].isfinite().all())
    fine = [r for r in range(M) if bad_k not in ways[r] and bad_v not in ways[r]]
    G = nq // 4
    ks, vs = R.rows_of(cache, 0, 0, torch.arange(L + M, device="cuda"))
    ok = torch.zeros((len(fine), L + M), dtype=torch.bool, device="cuda")
    for i, r in enumerate(fine):
        ok[i, R.seen(L, ways[r], 0)] = True
    for g in range(4):
        ref, _, tol, _ = R.attention(q[fine].double().reshape(-1, 4, G, D)[:, g].reshape(-1, D), ks[:, g],
                                     vs[:, g], ok.repeat_interleave(G, 0))
        err = (got[fine].reshape(-1, 4, G, D)[:, g].reshape(-1, D) - ref).abs()
        assert bool((err <= tol).all())


@pytest.mark.parametrize("size", [30.0, 3000.0, 60000.0])
@pytest.mark.parametrize("M,nq", [(1, 16), (9, 16), (64, 16)])
def test_great_scores(ctx, size, M, nq):
    """Scores up to 2^38: the greatest key wins and nothing overflows.  (The weights' exponents are differences of
    such scores, whose own rounding is the tolerance: one key a row stands far above the others.)"""
    L = 400
    cache, gen, _ = make(ctx, [L], [M], 64, 4, seed=2)
    k, v = R.rows_of(cache, 0, 0, torch.arange(L + M, device="cuda"))
    k = torch.zeros_like(k)
    k[:, :, 0] = -1.0
    k[137, :, 0] = size
    R.put(cache, 0, 0, torch.arange(L + M, device="cuda"), k, v)
    q = torch.zeros((M, nq, D), dtype=torch.float16, device="cuda")
    q[:, :, 0] = size
    out = torch.full((M, nq * D), 7.0, dtype=torch.float16, device="cuda")
    ctx.paged_attn(cache, 0, batch_of([M]), q.reshape(M, nq * D), nq, out)
    want = v[137].repeat_interleave(nq // 4, 0).expand(M, nq, D)
    assert torch.equal(out.double().reshape(M, nq, D), want.half().double())


def test_far_scores_keep_their_softmax(ctx):
    """Equal scores of 2^30 weigh the same."""
    L, nq = 100, 16
    cache, gen, _ = make(ctx, [L], [1], 64, 4, seed=2)
    k, v = R.rows_of(cache, 0, 0, torch.arange(L + 1, device="cuda"))
    k = torch.zeros_like(k)
    k[:, :, 0] = 32768.0
    R.put(cache, 0, 0, torch.arange(L + 1, device="cuda"), k, v)
    q = torch.zeros((1, nq, D), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 65504.0
    out = torch.full((1, nq * D), 7.0, dtype=torch.float16, device="cuda")
    ctx.paged_attn(cache, 0, batch_of([1]), q.reshape(1, -1), nq, out)
    want = v.mean(0).repeat_interleave(4, 0)
    # weights are equal, so exact up to the sums in fp32 and the output's rounding
    tol = want.abs() * 2.0 ** -11 + v.abs().mean(0).repeat_interleave(4, 0) * (L + 8) * 2.0 ** -24 + 2.0 ** -25
    assert bool(((out.double().reshape(nq, D) - want).abs() <= tol).all())


def test_small_weights_add_up(ctx):
    """131072 keys of 2^-26 of the greatest weight each make a 512th of the whole."""
    L = 1 << 17
    cache, gen, _ = make(ctx, [L], [1], 256, 1, seed=2)
    pos = torch.arange(L + 1, device="cuda")
    k = torch.zeros((L + 1, 1, D), device="cuda", dtype=torch.float64)
    v = torch.ones_like(k)
    k[77, 0, 0] = 26 * math.log(2) * math.sqrt(D) / 8
    v[77] = 0.0
    R.put(cache, 0, 0, pos, k, v)
    q = torch.zeros((1, D), dtype=torch.float16, device="cuda")
    q[0, 0] = 8.0
    out = torch.zeros((1, D), dtype=torch.float16, device="cuda")
    ctx.paged_attn(cache, 0, batch_of([1]), q, 1, out)
    s = float(k[77, 0, 0].half()) * 8 / math.sqrt(D)
    want = L / (math.exp(s) + L)
    # each weight half a step of fp16, scores 2^-22 of 18 (and so the ratio), the output's rounding
    assert float((out.double() - want).abs().max()) <= want * (2.0 ** -11 + 2.0 ** -11 + 18 * 2.0 ** -22)


def test_pool_past_4_gib(ctx):
    """Pages whose halves lie past 2^32."""
    n_pages, nkv = 34000, 8
    shape = (1, n_pages, nkv, 2, 4096)
    k, v = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2))
    table = cuda([[n_pages - 1, 0, n_pages - 2, -1]])
    cache = PagedCache.over(ctx, k, v, table, cuda([150]), torch.zeros(n_pages, dtype=torch.int32, device="cuda"))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    kk, vv = (torch.randn((159, nkv, D), generator=gen, device="cuda") for _ in range(2))
    R.put(cache, 0, 0, torch.arange(159, device="cuda"), kk, vv)
    q = torch.randn((9, 16 * D), generator=gen, device="cuda").half()
    out = torch.zeros_like(q)
    ctx.paged_attn(cache, 0, batch_of([9]), q, 16, out)
    check(cache, [9], chains([9]), q, out, 16)


def norm_rope(x, w, pos, rope, eps, base):
    """[T, H, 128] normed and rotated in 64 bits, and the bound of what 32 bits and fp16 add: about 19 roundings
    of the sum of squares (halved by the root), six more, and 2^-22 of the angle's sine: below 64 half
    steps of fp32 of both terms; half a step of fp16."""
    y = x.double()
    if w is not None:
        y = y / ((y * y).sum(-1, keepdim=True) / D + eps).sqrt() * w.double()
    z = y.clone()
    size = y.abs()
    h = rope // 2
    if h:
        f = base ** (-torch.arange(h, dtype=torch.float64, device=x.device) / h)
        th = pos.double()[:, None, None] * f
        a, b = y[..., :h], y[..., h:rope]
        z[..., :h], z[..., h:rope] = a * th.cos() - b * th.sin(), b * th.cos() + a * th.sin()
        size = size.clone()
        size[..., :h] = size[..., h:rope] = a.abs() + b.abs()
    return z, z.abs() * 2.0 ** -11 + size * 2.0 ** -18 + 2.0 ** -25


def cfg(nq, nkv, rope, eps=1e-6):
    return dict(H=2048, nQ=nq, nKV=nkv, D=D, rope_dim=rope, rope_base=1e6, eps=eps, window=0, C=0, gs=64)


@pytest.mark.parametrize("nq,nkv", HEADS)
@pytest.mark.parametrize("rope", [0, 32, 64, 128])
@pytest.mark.parametrize("page", [32, 256])
@pytest.mark.parametrize("norm", [True, False])
def test_append(ctx, nq, nkv, rope, page, norm):
    lens, rows = [0, 31, 64, 1000, 131000 if nkv == 1 else 77], [3, 9, 0, 1, 17]
    cache, gen, rng = make(ctx, lens, rows, page, nkv, layers=2, seed=rope)
    parents = [R.tree(m, rng) if m else [] for m in rows]
    n, width = sum(rows), (nq + 2 * nkv) * D
    wide = (torch.randn((n + 1, width + 8), generator=gen, device="cuda") * 1.5).half()
    qkv = wide[:, 8:]
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).half() if norm else None for _ in range(2))
    twin = PagedCache.over(ctx, cache.k.clone(), cache.v.clone(), cache.table, cache.lens, cache.refs)
    q = torch.full((n + 1, nq * D), 7.0, dtype=torch.float16, device="cuda")
    ctx.paged_append(cfg(nq, nkv, rope), cache, 1, batch_of(rows, parents, pad=1), qkv, qw, kw, q)
    assert bool((q[n:] == 7).all())
    x, at = qkv[:n].reshape(n, nq + 2 * nkv, D), 0
    for s, m in enumerate(rows):
        if not m:
            continue
        pos = torch.tensor([lens[s] + len(w) - 1 for w in R.ways(parents[s])], device="cuda")
        ref, tol = norm_rope(x[at:at + m, :nq], qw, pos, rope, 1e-6, 1e6)
        assert bool(((q[at:at + m].double().reshape(m, nq, D) - ref).abs() <= tol).all())
        slots = torch.arange(lens[s], lens[s] + m, device="cuda")
        k, v = R.rows_of(cache, 1, s, slots)
        ref, tol = norm_rope(x[at:at + m, nq:nq + nkv], kw, pos, rope, 1e-6, 1e6)
        assert bool(((k - ref).abs() <= tol).all())
        assert torch.equal(v, x[at:at + m, nq + nkv:].double())
        R.put(twin, 1, s, slots, k, v)
        at += m
    # nothing else was written
    for a, b in ((cache.k, twin.k), (cache.v, twin.v)):
        assert torch.equal(torch.nan_to_num(a, nan=9.0), torch.nan_to_num(b, nan=9.0))


def test_append_where_there_is_no_room(ctx):
    """Rows past the table's end or without a page are not written; queries come all the same."""
    lens, rows, nq, nkv = [60, 10], [9, 3], 16, 4
    cache, gen, _ = make(ctx, lens, rows, 32, nkv, seed=1, spare=0)
    cache.table[0, 2], cache.table[1, 0] = -1, cache.n_pages + 5  # tokens 64 and on of the first, all of the second
    n = sum(rows)
    qkv = torch.randn((n, (nq + 2 * nkv) * D), generator=gen, device="cuda").half()
    before = cache.k.clone()
    q = torch.zeros((n, nq * D), dtype=torch.float16, device="cuda")
    w = torch.ones(D, dtype=torch.float16, device="cuda")
    ctx.paged_append(cfg(nq, nkv, 64), cache, 0, batch_of(rows), qkv, w, w, q)
    assert bool((q.abs().sum(1) > 0).all())
    same = torch.nan_to_num(before, nan=9.0) == torch.nan_to_num(cache.k, nan=9.0)
    written = torch.zeros(cache.n_pages, dtype=torch.bool)
    written[cache.table[0, 1].item()] = True  # tokens 60 .. 63
    assert [bool(x.all()) for x in same[0]] == [not w for w in written.tolist()]
    # a length past what the table can hold
    cache.lens[0] = 2 ** 31 - 1
    cache.lens[1] = -7
    mid = cache.k.clone()
    ctx.paged_append(cfg(nq, nkv, 64), cache, 0, batch_of(rows), qkv, w, w, q)
    out = torch.zeros((n, nq * D), dtype=torch.float16, device="cuda")
    ctx.paged_attn(cache, 0, batch_of(rows), q, nq, out)
    ctx.paged_attn(cache, 0, batch_of(rows), q, nq, out, window=8)
    ctx.sync()
    assert torch.equal(torch.nan_to_num(mid, nan=9.0), torch.nan_to_num(cache.k, nan=9.0))
