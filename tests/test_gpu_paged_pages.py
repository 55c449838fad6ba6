"""GPU: the pages of many sequences (room, branches, giving back, moving accepted rows) against the rules
restated in tests/paged_ref.py, and whole steps of a batch, run and replayed."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R
from momij_amd._lib import MomijError
from momij_amd.ops import Context
from momij_amd.paged import PagedCache, RowBatch
from test_gpu_paged_attn import batch_of, cfg, chains, check, cuda, make, norm_rope

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    with torch.cuda.stream(c.stream):
        yield c
    c.close()


def filled(ctx, n_seqs, n_pages, nkv=2, blocks=6, layers=2, page=32, seed=0):
    """An empty cache whose pool holds numbers that tell the places apart."""
    cache = PagedCache(ctx, n_seqs, n_pages, nkv, blocks, layers, page)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    for x in (cache.k, cache.v):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
    return cache


def book_of(cache):
    return R.Book(cache.table.tolist(), cache.lens.tolist(), cache.refs.tolist(), cache.page_tokens)


def same(cache, book):
    assert cache.table.tolist() == book.table
    assert cache.lens.tolist() == book.lens
    assert cache.refs.tolist() == book.refs


def starts(rows):
    return RowBatch(cuda(np.concatenate([[0], np.cumsum(rows)])), int(sum(rows)), 64)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("n,n_pages,page", [(1, 3, 32), (7, 20, 32), (40, 70, 64), (300, 17000, 32), (1024, 2500, 128)])
def test_many_calls_in_turn(ctx, n, n_pages, page, seed):
    """Room, branches, lengths and giving back at random, also where the pool runs out; after every call the
    tables, lengths and counts are those of the rules, and no page is named without being counted."""
    rng = np.random.default_rng(seed)
    cache = filled(ctx, n, n_pages, nkv=1, blocks=5, layers=1, page=page, seed=seed)
    book = book_of(cache)
    out = torch.zeros((n, 4), dtype=torch.int32, device="cuda")
    for step in range(14):
        rows = [int(x) for x in np.where(rng.random(n) < 0.7, rng.integers(0, 65, n), 0)]
        if step == 5:
            rows = [0] * n
        before_k, before_v = cache.k.clone(), cache.v.clone()
        ctx.pages_reserve(cache, starts(rows), out)
        want, copies = book.reserve(rows)
        assert out.tolist() == want
        same(cache, book)
        assert book.named() == book.refs
        for s, o, p, fill in copies:
            ik, iv = R.unit_at(torch.arange(-(-fill // 8) * 8, device="cuda"))
            for x, i in ((before_k, ik), (before_v, iv)):
                x.view(1, n_pages, -1)[0, p, i] = x.view(1, n_pages, -1)[0, o, i]
        assert torch.equal(before_k, cache.k) and torch.equal(before_v, cache.v)
        # the rows of those who were served are kept in part
        acc = [int(rng.integers(-1, m + 2)) if w[0] else -1 for m, w in zip(rows, want)]
        ctx.pages_commit(cache, starts(rows), cuda(acc))
        for s, m in enumerate(rows):
            if m:
                book.lens[s] += max(0, min(acc[s], m - 1) + 1)
        same(cache, book)
        src = [int(x) for x in np.where(rng.random(n) < 0.3, rng.integers(-2, n + 2, n), -1)]
        ctx.pages_fork(cache, cuda(src))
        book.fork(src)
        same(cache, book)
        cut = [int(x) for x in np.where(rng.random(n) < 0.4, rng.integers(0, 4 * page, n), -1)]
        ctx.pages_truncate(cache, cuda(cut))
        book.truncate(cut)
        same(cache, book)
        assert book.named() == book.refs
    ctx.pages_truncate(cache, torch.zeros_like(cache.lens))
    ctx.sync()
    assert not cache.refs.any() and bool((cache.table == -1).all())


@pytest.mark.parametrize("n,layers,nkv", [(100, 24, 8), (1024, 1024, 1)])
def test_few_copies_of_many_sequences(ctx, n, layers, nkv):
    """More sequences, layers and heads than a launch has blocks: branches here and there, each of which
    gets a page of its own with the committed tokens of every layer and head."""
    page, L, n_pages = 32, 20, 16
    shape = (layers, n_pages, nkv, 1, 4096)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    k, v = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16) for _ in range(2))
    table, lens, refs = np.full((n, 2), -1), np.zeros(n, int), np.zeros(n_pages, int)
    table[3, 0], lens[3], refs[9] = 9, L, 1
    cache = PagedCache.over(ctx, k, v, cuda(table), cuda(lens), cuda(refs))
    to = [0, 5, 63, 64, n // 2 - 1, n // 2, n - 2, n - 1]
    src = np.full(n, -1)
    src[to] = 3
    ctx.pages_fork(cache, cuda(src))
    before = [x.clone() for x in (k, v)]
    out = torch.zeros((n, 4), dtype=torch.int32, device="cuda")
    ctx.pages_reserve(cache, starts([1 if s in to or s == 3 else 0 for s in range(n)]), out)
    ctx.sync()
    got = out.tolist()
    new = [p for p in range(n_pages) if p != 9]
    at = 0
    for s in range(n):  # (all leave the shared page, also the source: its count is that before the call)
        if s in to or s == 3:
            assert got[s] == [1, 1, 9, new[at]], s
            at += 1
        else:
            assert got[s] == [0, 0, -1, -1], s
    i = [x.cuda() for x in R.unit_at(torch.arange(24))]
    for x, b, j in zip((k, v), before, i):
        b = b.view(layers, n_pages, nkv, 4096)
        for p in new[:at]:
            b[:, p, :, j.reshape(-1)] = b[:, 9, :, j.reshape(-1)]
        assert torch.equal(x.view(layers, n_pages, nkv, 4096), b)


def test_lengths_themselves_give_back_what_was_reserved(ctx):
    cache = filled(ctx, 3, 12)
    out = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    ctx.pages_reserve(cache, starts([64, 10, 33]), out)
    ctx.pages_commit(cache, starts([64, 10, 33]), cuda([39, 9, -1]))
    ctx.pages_truncate(cache, cache.lens)
    ctx.sync()
    assert cache.lens.tolist() == [40, 10, 0]
    assert (cache.table >= 0).sum(1).tolist() == [2, 1, 0] and int(cache.refs.sum()) == 3


def test_tables_that_hold_nonsense(ctx):
    """Entries outside the pool are nobody's; lengths past the table count as what it holds."""
    cache = filled(ctx, 4, 9, blocks=3)
    cache.table.copy_(cuda([[9, -3, 5], [2 ** 31 - 1, 1, -(2 ** 31)], [0, 0, 0], [-1, -1, -1]]))
    cache.lens.copy_(cuda([64, 2 ** 31 - 1, -5, 96]))
    cache.refs.copy_(cuda([3, 1, 0, 0, 0, 1, 0, 0, 0]))
    out = torch.zeros((4, 4), dtype=torch.int32, device="cuda")
    ctx.pages_reserve(cache, starts([5, 5, 40, 1]), out)
    ctx.sync()
    assert out.tolist() == [[1, 0, -1, -1], [0, 0, -1, -1], [1, 2, -1, -1], [0, 0, -1, -1]]
    assert cache.table[2].tolist() == [2, 3, 0] and cache.refs.tolist() == [1, 1, 1, 1, 0, 1, 0, 0, 0]
    ctx.pages_fork(cache, cuda([-1, -1, -1, 1]))
    ctx.sync()
    assert cache.table[3].tolist() == [-1, 1, -1] and cache.refs[1].item() == 2 and cache.lens[3].item() == 96
    ctx.pages_truncate(cache, cuda([0, 0, 0, 0]))
    ctx.sync()
    assert bool((cache.table == -1).all()) and cache.refs.tolist() == [0] * 9


def test_a_batch_that_decreases_or_leaves_its_arrays(ctx):
    """row_start that is no list of starts: the calls stay inside the arrays."""
    cache = filled(ctx, 4, 40, nkv=4)
    cache.table.copy_(torch.arange(24, dtype=torch.int32, device="cuda").reshape(4, 6))
    cache.lens.fill_(50)
    cache.refs[:24] = 1
    q = torch.randn((6, 16 * D), device="cuda").half()
    out = torch.zeros_like(q)
    qkv = torch.randn((6, 24 * D), device="cuda").half()
    w = torch.ones(D, dtype=torch.float16, device="cuda")
    res = torch.zeros((4, 4), dtype=torch.int32, device="cuda")
    for start in ([0, 100, -5, 3, 6], [5, 4, 3, 2, 1], [-9, -8, 2 ** 31 - 1, 7, 0], [2 ** 31 - 1] * 5):
        b = RowBatch(cuda(start), 6, 3, cuda([-1] * 6, torch.int64))
        ctx.pages_reserve(cache, b, res)
        ctx.paged_append(cfg(16, 4, 64), cache, 1, b, qkv, w, w, out)
        ctx.paged_attn(cache, 1, b, q, 16, out)
        ctx.pages_commit(cache, b, cuda([99, -99, 2, 2 ** 31 - 1]), cuda([0, 2, 1, -7, 2 ** 31 - 1, 5]))
    ctx.sync()


@pytest.mark.parametrize("page,nkv,layers", [(32, 4, 3), (64, 1, 2), (256, 8, 1)])
@pytest.mark.parametrize("m", [1, 2, 9, 17, 64])
def test_commit_moves_the_path(ctx, page, nkv, layers, m):
    """Paths into trees, with sequences of no rows and no kept rows beside; lens_out apart and in place."""
    rng = np.random.default_rng(m)
    lens, rows = [0, page - 1, 40, 70, 5], [m, m, 0, max(1, m - 1), m]
    n = len(lens)
    cache = filled(ctx, n, 40, nkv, 300 // page + 2, layers, page, seed=m)
    perm = rng.permutation(40)
    at = 0
    table = np.full((n, cache.blocks), -1)
    for s in range(n):
        b = -(-(lens[s] + rows[s]) // page)
        table[s, :b] = perm[at:at + b]
        at += b
    cache.table.copy_(cuda(table))
    cache.lens.copy_(cuda(lens))
    accepted, path = [], []
    for s, k in enumerate(rows):
        par = R.tree(k, rng) if k else []
        way = R.ways(par)[-1] if k else []
        if s == 4:
            way = way[:1]
        accepted.append(len(way) - 1 if s != 3 else -1)
        path += way + [-1] * (k - len(way))
    keep = [(R.rows_of(cache, l, s, lens[s] + torch.arange(rows[s], device="cuda")) if rows[s] else None)
            for l in range(layers) for s in range(n)]
    twin = PagedCache.over(ctx, cache.k.clone(), cache.v.clone(), cache.table, cache.lens, cache.refs)
    start = np.concatenate([[0], np.cumsum(rows)])
    for l in range(layers):
        for s in range(n):
            a = accepted[s] + 1
            if rows[s] and a > 0:
                k, v = keep[l * n + s]
                way = path[start[s]:start[s] + a]
                R.put(twin, l, s, lens[s] + torch.arange(a, device="cuda"), k[way], v[way])
    want = [x + (a + 1 if k else 0) for x, a, k in zip(lens, accepted, rows)]
    apart = torch.full_like(cache.lens, 77)
    ctx.pages_commit(cache, starts(rows), cuda(accepted), cuda(path), apart)
    ctx.sync()
    assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)
    assert apart.tolist() == want and cache.lens.tolist() == lens
    ctx.pages_commit(cache, starts(rows), cuda(accepted))
    ctx.sync()
    assert torch.equal(cache.k, twin.k) and cache.lens.tolist() == want


def step(ctx, cache, batch, qkv, weights, q, out, c, window, reserved):
    ctx.pages_reserve(cache, batch, reserved)
    for l in range(cache.n_layers):
        ctx.paged_append(c, cache, l, batch, qkv[l], *weights, q)
        ctx.paged_attn(cache, l, batch, q, 16, out[l], window=window)


@pytest.mark.parametrize("window", [0, 48])
def test_a_batch_goes_on(ctx, window):
    """Several passes of a batch: prompts, branches of them, drafts of which some are kept, requests that end and
    others that take their place.  Every pass attends what the sequence's own history says."""
    rng = np.random.default_rng(8)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(8)
    nq, nkv, n, layers = 16, 4, 6, 2
    c = cfg(nq, nkv, 64)
    cache = filled(ctx, n, 60, nkv, 8, layers, 32)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    weights = [(1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).half() for _ in range(2)]
    reserved = torch.zeros((n, 4), dtype=torch.int32, device="cuda")
    history = [[([], []) for _ in range(layers)] for _ in range(n)]  # K and V rows as they were written
    tokens = [0] * n
    for i in range(9):
        if i == 0:
            rows, parents = [40, 25, 0, 0, 0, 1], None
        else:
            rows = [int(x) for x in rng.integers(0 if i % 2 else 1, 12, n)]
            parents = [R.tree(m, rng) if m else [] for m in rows]
        if i == 2:  # three samples of the first prompt, one of the second
            src = [-1, -1, 0, 0, 1, -1]
            ctx.pages_fork(cache, cuda(src))
            for s, f in enumerate(src):
                if f >= 0:
                    history[s] = [([*k], [*v]) for k, v in history[f]]
                    tokens[s] = tokens[f]
        if i == 5:  # one request ends, one goes back to its first 20 tokens
            ctx.pages_truncate(cache, cuda([-1, 20, -1, 0, -1, -1]))
            for s, t in ((1, min(20, tokens[1])), (3, 0)):
                history[s] = [(k[:t], v[:t]) for k, v in history[s]]
                tokens[s] = t
        R_ = sum(rows)
        batch = batch_of(rows, parents)
        qkv = [(torch.randn((R_, (nq + 2 * nkv) * D), generator=gen, device="cuda") * 1.5).half() for _ in range(layers)]
        q = torch.zeros((R_, nq * D), dtype=torch.float16, device="cuda")
        out = [torch.full((R_, nq * D), 7.0, dtype=torch.float16, device="cuda") for _ in range(layers)]
        step(ctx, cache, batch, qkv, weights, q, out, c, window, reserved)
        ctx.sync()
        assert [x[0] for x in reserved.tolist()] == [int(m > 0) for m in rows]
        sees = [R.ways(p) for p in parents] if parents else chains(rows)
        at, path, accepted = 0, [], []
        for s, m in enumerate(rows):
            way = (sees[s][int(rng.integers(0, m))] if parents else list(range(m))) if m else []
            for l in range(layers):
                if m == 0:
                    continue
                x = qkv[l][at:at + m].reshape(m, nq + 2 * nkv, D)
                pos = torch.tensor([tokens[s] + len(w) - 1 for w in sees[s]], device="cuda")
                # keys are what the cache holds (checked against 64 bits), values what was given
                k, v = R.rows_of(cache, l, s, tokens[s] + torch.arange(m, device="cuda"))
                ref, tol = norm_rope(x[:, nq:nq + nkv], weights[1], pos, 64, 1e-6, 1e6)
                assert bool(((k - ref).abs() <= tol).all())
                assert torch.equal(v, x[:, nq + nkv:].double())
                if tokens[s]:
                    hk, hv = R.rows_of(cache, l, s, torch.arange(tokens[s], device="cuda"))
                    assert torch.equal(hk, torch.stack(history[s][l][0])) and torch.equal(hv, torch.stack(history[s][l][1]))
                for r in way:
                    history[s][l][0].append(k[r])
                    history[s][l][1].append(v[r])
            accepted.append(len(way) - 1)
            path += way + [-1] * (m - len(way))
            at += m
        check(cache, rows, sees, q, out[layers - 1], nq, window, layers - 1)
        ctx.pages_commit(cache, batch, cuda(accepted), cuda(path) if parents else None)
        tokens = [t + a + 1 for t, a in zip(tokens, accepted)]
        ctx.sync()
        assert cache.lens.tolist() == tokens
        b = book_of(cache)
        assert b.named() == b.refs


def test_a_captured_step_goes_by_the_arrays(ctx):
    """A whole step of a batch in one graph, replayed with other lengths, rows, masks and tables; each replay equals
    the same step run eagerly, with eager work between the replays."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    nq, nkv, n, layers, V, most = 16, 4, 5, 2, 1000, 40
    c = cfg(nq, nkv, 64)
    f16 = dict(dtype=torch.float16, device="cuda")
    weights = [torch.ones(D, **f16) for _ in range(2)]
    ws = [torch.zeros(ctx.paged_workspace(nq, nkv, 9), dtype=torch.uint8, device="cuda"),
          torch.zeros(ctx.accept_workspace(n, most, V), dtype=torch.uint8, device="cuda")]

    def state():
        cache = filled(ctx, n, 50, nkv, 8, layers, 32)
        return dict(cache=cache, start=cuda([0] * (n + 1)), anc=cuda([0] * most, torch.int64),
                    qkv=torch.zeros((layers, most, (nq + 2 * nkv) * D), **f16), q=torch.zeros((most, nq * D), **f16),
                    out=torch.zeros((layers, most, nq * D), **f16), reserved=cuda([[0] * 4] * n),
                    logits=torch.zeros((most, V), device="cuda"), tokens=cuda([0] * most),
                    T=torch.ones(n, device="cuda"), ua=torch.zeros(most, device="cuda"), us=torch.zeros(n, device="cuda"),
                    accepted=cuda([0] * n), path=cuda([0] * most), token=cuda([0] * n))

    def go(d):
        b = RowBatch(d["start"], most, 9, d["anc"])
        ctx.pages_reserve(d["cache"], b, d["reserved"])
        for l in range(layers):
            ctx.paged_append(c, d["cache"], l, b, d["qkv"][l], *weights, d["q"])
            ctx.paged_attn(d["cache"], l, b, d["q"], nq, d["out"][l], ws=ws[0])
        ctx.accept_rows(b, d["logits"], d["tokens"], d["T"], d["ua"], d["us"], d["accepted"], d["path"], d["token"],
                        ws=ws[1])
        ctx.pages_commit(d["cache"], b, d["accepted"], d["path"])

    a, b = state(), state()
    go(a)  # (with no rows: nothing happens)
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.stream):
        go(a)
    rng = np.random.default_rng(0)
    for i in range(6):
        rows = [int(x) for x in rng.integers(0, 9, n)] if i else [8, 3, 0, 1, 8]
        parents = [R.tree(m, rng) if m else [] for m in rows]
        fresh = dict(start=cuda(np.concatenate([[0], np.cumsum(rows)])),
                     qkv=torch.randn(a["qkv"].shape, generator=gen, device="cuda").half(),
                     logits=torch.randn((most, V), generator=gen, device="cuda") * 3,
                     ua=torch.rand(most, generator=gen, device="cuda") * 0.01,
                     us=torch.rand(n, generator=gen, device="cuda"))
        fresh["tokens"] = fresh["logits"].argmax(-1).roll(1).int()
        bt = batch_of(rows, parents)
        fresh["anc"] = torch.cat([bt.anc, torch.zeros(most - bt.rows, dtype=torch.int64, device="cuda")])
        for d in (a, b):
            for k, v in fresh.items():
                d[k].copy_(v)
        if i == 3:
            for d in (a, b):
                ctx.pages_fork(d["cache"], cuda([-1, -1, 0, 0, -1]))
        graph.replay()
        torch.cuda.synchronize()
        go(b)
        ctx.sync()
        for k in ("q", "out", "reserved", "accepted", "path", "token"):
            m = sum(rows)
            x, y = (d[k][:, :m] if k == "out" else d[k][:m] if k in ("q", "path") else d[k] for d in (a, b))
            assert torch.equal(x, y), (i, k)
        for x, y in zip(*((d["cache"].table, d["cache"].lens, d["cache"].refs, d["cache"].k, d["cache"].v) for d in (a, b))):
            assert torch.equal(x, y), i


def test_capture_needs_a_workspace(ctx):
    cache = filled(ctx, 1, 8, 4)
    q = torch.zeros((1, 16 * D), dtype=torch.float16, device="cuda")
    out, b = torch.zeros_like(q), RowBatch(cuda([0, 1]), 1, 1)
    f = torch.zeros(1, device="cuda")
    i = [cuda([0]) for _ in range(4)]
    x = torch.zeros((1, 50), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.stream):
        f.add_(1.0)
        with pytest.raises(MomijError, match="cannot be captured"):
            ctx.paged_attn(cache, 0, b, q, 16, out)
        with pytest.raises(MomijError, match="cannot be captured"):
            ctx.accept_rows(b, x, i[0], f, f, f, i[1], i[2], i[3])
    ctx.sync()


def test_on_another_stream_and_two_contexts(ctx):
    """Two contexts on streams of their own attend one pool at the same time."""
    other = Context(0)
    cache = filled(ctx, 2, 64, 4, 30, 1, 64)
    cache.table.copy_(cuda(np.arange(60).reshape(2, 30)))
    cache.lens.copy_(cuda([1800, 900]))
    twin = PagedCache.over(other, cache.k, cache.v, cache.table, cache.lens, cache.refs)
    q = torch.randn((10, 16 * D), device="cuda").half()
    outs = [torch.zeros_like(q) for _ in range(3)]
    ctx.paged_attn(cache, 0, batch_of([5, 5]), q, 16, outs[2])
    torch.cuda.synchronize()
    for _ in range(5):
        ctx.paged_attn(cache, 0, batch_of([5, 5]), q, 16, outs[0])
        other.paged_attn(twin, 0, batch_of([5, 5]), q, 16, outs[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2])
    other.close()


def test_an_abort_serves_nobody(ctx):
    cache = filled(ctx, 2, 8, 4)
    cache.table[0, 0], cache.lens[0], cache.refs[0] = 0, 9, 2
    out = torch.full((2, 4), 5, dtype=torch.int32, device="cuda")
    before = cache.table.clone(), cache.refs.clone(), cache.k.clone()
    torch.cuda.synchronize()
    ctx.set_abort(True)
    ctx.pages_reserve(cache, starts([3, 3]), out)
    torch.cuda.synchronize()
    ctx.set_abort(False)
    with pytest.raises(MomijError):
        ctx.sync()
    assert out.tolist() == [[0, 0, -1, -1]] * 2
    for x, y in zip(before, (cache.table, cache.refs, cache.k)):
        assert torch.equal(x, y)
    ctx.pages_reserve(cache, starts([3, 3]), out)
    ctx.sync()
    assert out[:, 0].tolist() == [1, 1]


@pytest.mark.parametrize("M", [1, 9, 64])
def test_an_aborted_step_leaves_its_arrays(ctx, M):
    """The word set: nothing is attended, accepted or kept; cleared, the same calls on the same workspaces are
    right."""
    nq, nkv, V = 16, 4, 5000
    lens, rows = [700, 90], [M, M]
    cache, gen, _ = make(ctx, lens, rows, 64, nkv, seed=M)
    q = torch.randn((2 * M, nq * D), generator=gen, device="cuda").half()
    logits = torch.randn((2 * M, V), generator=gen, device="cuda")
    tokens = torch.randint(0, V, (2 * M,), generator=gen, device="cuda").int()
    T, u, us = (torch.full((k,), 0.5, device="cuda") for k in (2, 2 * M, 2))
    out, acc, path, tok = torch.full_like(q, 7.0), cuda([55] * 2), cuda([55] * (2 * M)), cuda([55] * 2)
    ws = [torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda")
          for size in (ctx.paged_workspace(nq, nkv, M), ctx.accept_workspace(2, 2 * M, V))]
    batch = batch_of(rows)

    def step():
        ctx.paged_attn(cache, 0, batch, q, nq, out, ws=ws[0])
        ctx.accept_rows(batch, logits, tokens, T, u, us, acc, path, tok, ws=ws[1])
        ctx.pages_commit(cache, batch, acc)

    torch.cuda.synchronize()
    ctx.set_abort(True)
    step()
    torch.cuda.synchronize()
    ctx.set_abort(False)
    with pytest.raises(MomijError):
        ctx.sync()
    assert bool((out == 7.0).all()) and cache.lens.tolist() == lens
    assert acc.tolist() + path.tolist() + tok.tolist() == [55] * (4 + 2 * M)
    acc.fill_(-1)
    ctx.paged_attn(cache, 0, batch, q, nq, out, ws=ws[0])
    check(cache, rows, chains(rows), q, out, nq)
    ctx.accept_rows(batch, logits, tokens, T, u, us, acc, path, tok, ws=ws[1])
    ctx.sync()
    assert all(0 <= t < V for t in tok.tolist())
