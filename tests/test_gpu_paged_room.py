"""GPU: steps in which somebody has no room.  What other requests hold stays as it is bit for bit, and a length
advances over tokens that were written, or not at all."""
import numpy as np
import pytest
import torch

import paged_ref as R
from momij_amd.paged import PagedCache, RowBatch
from test_gpu_paged_attn import D, batch_of, cfg, cuda
from test_gpu_paged_pages import book_of, ctx, filled, same, starts  # noqa: F401

pytestmark = pytest.mark.gpu
NQ, NKV, V = 16, 4, 600


class Step:
    """A step as the documentation has it: room, append and attention in every layer, acceptance, commit."""

    def __init__(self, ctx, cache, rows, parents=None, seed=0, window=0):  # noqa: F811
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        n, total = len(rows), sum(rows)
        self.ctx, self.cache, self.rows = ctx, cache, rows
        self.batch = batch_of(rows, parents)
        self.qkv = [torch.randn((total, (NQ + 2 * NKV) * D), generator=gen, device="cuda").half()
                    for _ in range(cache.n_layers)]
        self.w = torch.ones(D, dtype=torch.float16, device="cuda")
        self.q = torch.zeros((total, NQ * D), dtype=torch.float16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.reserved, self.accepted, self.token = cuda([[0] * 4] * n), cuda([0] * n), cuda([0] * n)
        self.path = cuda([0] * total)
        self.logits = torch.randn((total, V), generator=gen, device="cuda")
        # (drafts that are certain and accepted whatever they are: their uniform is 0)
        self.tokens = torch.randint(0, V, (total,), generator=gen, device="cuda").int()
        self.T, self.us = torch.ones(n, device="cuda"), torch.rand(n, generator=gen, device="cuda")
        self.ua = torch.zeros(total, device="cuda")
        self.ws = [torch.zeros(size, dtype=torch.uint8, device="cuda")
                   for size in (ctx.paged_workspace(NQ, NKV, max(rows)), ctx.accept_workspace(n, total, V))]

    def reserve(self):
        self.ctx.pages_reserve(self.cache, self.batch, self.reserved)

    def append(self, cache=None):
        for l in range(self.cache.n_layers):
            self.ctx.paged_append(cfg(NQ, NKV, 64), cache or self.cache, l, self.batch, self.qkv[l], self.w, self.w,
                                  self.q)
            self.ctx.paged_attn(cache or self.cache, l, self.batch, self.q, NQ, self.out, ws=self.ws[0])

    def accept(self):
        self.ctx.accept_rows(self.batch, self.logits, self.tokens, self.T, self.ua, self.us, self.accepted, self.path,
                             self.token, ws=self.ws[1])

    def commit(self, how="path", cache=None):
        lens = torch.full_like(self.cache.lens, 77) if how == "apart" else None
        self.ctx.pages_commit(cache or self.cache, self.batch, self.accepted, None if how == "chain" else self.path, lens)
        return self.cache.lens if lens is None else lens

    def __call__(self, how="path"):
        self.reserve()
        self.append()
        self.accept()
        return self.commit(how)


def history(cache):
    """K and V of every sequence's committed tokens, in all layers."""
    return [[[x.clone() for x in R.rows_of(cache, l, s, torch.arange(n, device="cuda"))] for l in range(cache.n_layers)]
            for s, n in enumerate(cache.lens.tolist())]


def kept(cache, before, but=()):
    """Committed tokens of before are what they were."""
    for s, layers in enumerate(before):
        if s not in but:
            for l, (k, v) in enumerate(layers):
                kk, vv = R.rows_of(cache, l, s, torch.arange(len(k), device="cuda"))
                assert torch.equal(k, kk) and torch.equal(v, vv), (s, l)


def parent_and_branch(ctx, cut, n_pages=2, page=64, forks=1, seed=0):  # noqa: F811
    """Sequence 0 of 100 tokens and branches of it cut to `cut` tokens; nothing is free."""
    cache = filled(ctx, 1 + forks, n_pages, NKV, 6, 2, page, seed)
    n = -(-100 // page)
    cache.table[0, :n] = cuda(list(range(n)))
    cache.lens[0] = 100
    cache.refs[:n] = 1
    ctx.pages_fork(cache, cuda([-1] + [0] * forks))
    ctx.pages_truncate(cache, cuda([-1] + [cut] * forks))
    return cache


HOW = ["path", "chain", "apart"]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("cut", [100, 80, 70, 65])
@pytest.mark.parametrize("m", [1, 5, 9])
def test_a_branch_without_room_beside_its_parent(ctx, how, cut, m):  # noqa: F811
    """The branch's last page is its parent's too, and there is none for it: the parent's tokens stay, the branch
    stays as long as it was."""
    cache = parent_and_branch(ctx, cut)
    step = Step(ctx, cache, [0, m], seed=m)
    before, table, refs = history(cache), cache.table.clone(), cache.refs.clone()
    k, v = cache.k.clone(), cache.v.clone()
    lens = step(how)
    ctx.sync()
    assert step.reserved.tolist()[1] == [0, 0, -1, -1]
    kept(cache, before)
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    assert lens.tolist() == [100, cut]
    assert torch.equal(cache.table, table) and torch.equal(cache.refs, refs)
    # a page is found: the same step goes through
    more = PagedCache.over(ctx, *(torch.cat([x, x], 1) for x in (cache.k, cache.v)), cache.table, cache.lens,
                           torch.cat([cache.refs, torch.zeros_like(cache.refs)]))
    again = Step(ctx, more, [0, m], seed=m)
    before = history(more)
    lens = again(how)
    ctx.sync()
    assert again.reserved[1, 0].item() == 1 and lens.tolist() == [100, cut + m]
    kept(more, before)


@pytest.mark.parametrize("how", HOW)
def test_two_branches_without_room(ctx, how):  # noqa: F811
    """Neither writes where the other would."""
    cache = parent_and_branch(ctx, 80, forks=2)
    step = Step(ctx, cache, [1, 3, 3], seed=2)
    k, v = cache.k.clone(), cache.v.clone()
    lens = step(how)
    ctx.sync()
    # (the parent's own page is shared as well)
    assert step.reserved[:, 0].tolist() == [0, 0, 0] and lens.tolist() == [100, 80, 80]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("L,m", [(64, 1), (64, 9), (60, 9), (63, 2), (0, 5), (32, 64)])
def test_rows_that_have_no_page(ctx, how, L, m):  # noqa: F811
    """A sequence at the end of its pages, or with space for some of its rows only, beside one that has room."""
    cache = filled(ctx, 2, 4, NKV, 6, 2, 32, seed=L)
    n = -(-L // 32)
    cache.table[0, :n] = cuda(list(range(n)))
    cache.table[1, 0] = 3
    cache.lens.copy_(cuda([L, 7]))
    cache.refs.copy_(cuda([1] * 4))  # (nothing is free)
    step = Step(ctx, cache, [m, 2], seed=m)
    before = history(cache)
    lens = step(how)
    ctx.sync()
    assert step.reserved[:, 0].tolist() == [0, 1]
    assert lens.tolist() == [L, 9]
    kept(cache, before)


@pytest.mark.parametrize("how", HOW)
def test_a_table_that_is_full(ctx, how):  # noqa: F811
    """Rows past the table's last entry."""
    cache = filled(ctx, 1, 9, NKV, 2, 2, 32)
    first = Step(ctx, cache, [60])
    first()
    ctx.sync()
    assert cache.lens.tolist() == [60]
    step = Step(ctx, cache, [9], seed=3)
    lens = step(how)
    ctx.sync()
    assert step.reserved[0].tolist() == [0, 0, -1, -1] and lens.tolist() == [60]
    step = Step(ctx, cache, [4], seed=3)
    assert step(how).tolist() == [64]


@pytest.mark.parametrize("how", ["path", "chain"])
def test_the_one_that_is_left_alone_on_its_page(ctx, how):  # noqa: F811
    """Two branches of one page and one page free: the first takes it, and by that the second is alone on its own.
    The record says that the second had no room, so its length stays; the next step finds it room."""
    cache = filled(ctx, 3, 2, NKV, 4, 2, 32)
    cache.table[0, 0], cache.lens[0], cache.refs[0] = 0, 20, 1
    ctx.pages_fork(cache, cuda([-1, 0, -1]))
    step = Step(ctx, cache, [3, 4, 0], seed=5)
    before = history(cache)
    step(how)
    ctx.sync()
    assert step.reserved.tolist() == [[1, 1, 0, 1], [0, 0, -1, -1], [0, 0, -1, -1]]
    assert cache.lens.tolist() == [23, 20, 0] and cache.refs.tolist() == [1, 1]
    kept(cache, before)
    step = Step(ctx, cache, [0, 4, 0], seed=6)
    before = history(cache)
    step(how)
    ctx.sync()
    assert step.reserved[1].tolist() == [1, 0, -1, -1] and cache.lens.tolist() == [23, 24, 0]
    kept(cache, before)


@pytest.mark.parametrize("give_back", [False, True])
@pytest.mark.parametrize("when", ["before append", "before commit"])
def test_a_branch_in_the_middle_of_a_step(ctx, when, give_back):  # noqa: F811
    """A sequence that has room keeps its step, though a branch of its committed tokens is made meanwhile (and pages
    behind the lengths are given back: the rows' is not one); the branch is the committed tokens, also after it has
    gone on itself."""
    cache = filled(ctx, 2, 6, NKV, 6, 2, 32)
    Step(ctx, cache, [45, 0])()
    step = Step(ctx, cache, [6, 0], seed=1)
    before = history(cache)
    step.reserve()
    if when == "before append":
        ctx.pages_fork(cache, cuda([-1, 0]))
    step.append()
    step.accept()
    if when == "before commit":
        ctx.pages_fork(cache, cuda([-1, 0]))
    if give_back:
        ctx.pages_truncate(cache, cache.lens)
    step.commit()
    ctx.sync()
    assert cache.lens.tolist() == [51, 45]
    kept(cache, [before[0], before[0]])
    v = [R.rows_of(cache, l, 0, torch.arange(45, 51, device="cuda"))[1] for l in range(2)]
    for l in range(2):
        assert torch.equal(v[l], step.qkv[l].reshape(6, -1, D)[:, NQ + NKV:].double())
    other = Step(ctx, cache, [0, 5], seed=2)
    whole = history(cache)
    other()
    ctx.sync()
    assert other.reserved[1, 0].item() == 1 and cache.lens.tolist() == [51, 50]
    kept(cache, whole)


def test_branches_and_cuts_need_room_again(ctx):  # noqa: F811
    """Rows appended without a call for room: a new branch, and a sequence cut to fewer tokens while a branch has
    the rest, write nothing that is another's and keep nothing."""
    cache = parent_and_branch(ctx, 80, n_pages=6)
    Step(ctx, cache, [3, 3])()  # (both have had room before)
    ctx.pages_fork(cache, cuda([-1, 0]))
    ctx.pages_truncate(cache, cuda([90, -1]))
    ctx.sync()
    assert cache.lens.tolist() == [90, 103]
    step = Step(ctx, cache, [4, 4], seed=4)
    k, v = cache.k.clone(), cache.v.clone()
    step.append()
    step.accept()
    step.commit()
    ctx.sync()
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v) and cache.lens.tolist() == [90, 103]
    assert Step(ctx, cache, [4, 4], seed=4)().tolist() == [94, 107]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("served", ["its own", "shared", "none"])
def test_another_view_of_the_pages(ctx, served, how):  # noqa: F811
    """Room asked for by one view, rows appended and kept by another, which knows of it or not."""
    cache = parent_and_branch(ctx, 80)
    view = PagedCache.over(ctx, cache.k, cache.v, cache.table, cache.lens, cache.refs,
                           cache.served if served == "shared" else None)
    if served == "none":
        view._ref._obj.served = None
    step = Step(ctx, cache, [0, 3], seed=7)
    k = cache.k.clone()
    step.reserve()
    step.append(view)
    step.accept()
    assert step.commit(how, cache=view).tolist() == [100, 80]
    assert torch.equal(cache.k, k)
    # its parent gone, the branch is alone on the page
    ctx.pages_truncate(cache, cuda([0, -1]))
    step.reserve()
    step.append(view)
    step.accept()
    assert step.reserved[1].tolist() == [1, 0, -1, -1] and step.commit(how, cache=view).tolist() == [0, 83]


def test_a_captured_step_without_room(ctx):  # noqa: F811
    """The whole step in one graph: replayed while the branch has no room, and after a page was given back."""
    cache = parent_and_branch(ctx, 80, n_pages=3, forks=2)
    cache.table[2].fill_(-1)
    cache.table[2, 0] = 2
    cache.lens[2] = 9
    cache.refs.copy_(cuda([2, 2, 1]))
    # (sequence 0 takes no part; 2 holds the last page)
    step = Step(ctx, cache, [0, 2, 1], seed=8)
    ctx.paged_attn(cache, 0, step.batch, step.q, NQ, step.out, ws=step.ws[0])
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.stream):
        step()
    before = history(cache)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert step.reserved[:, 0].tolist() == [0, 0, 1]
        assert cache.lens.tolist() == [100, 80, 10 + i]
        kept(cache, before, but=[2])
        assert bool((cache.k.float() * 0 == 0).all())  # (the program's own work between replays)
    ctx.pages_truncate(cache, cuda([-1, -1, 0]))
    step.batch.row_start.copy_(cuda([0, 0, 2, 2]))
    graph.replay()
    torch.cuda.synchronize()
    assert step.reserved[:, 0].tolist() == [0, 1, 0] and cache.lens.tolist() == [100, 82, 0]
    kept(cache, before[:2])


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("n,n_pages,page", [(7, 7, 32), (40, 30, 64)])
def test_many_steps_of_a_pool_that_runs_out(ctx, n, n_pages, page, seed):  # noqa: F811
    """Steps at random as the documentation has them, branches, cuts and ends between them: lengths go by the
    record, and every sequence's tokens are those that it was given."""
    rng = np.random.default_rng(seed)
    cache = filled(ctx, n, n_pages, NKV, 5, 1, page, seed)
    book = book_of(cache)
    told = [torch.zeros((0, NKV, D), dtype=torch.float64, device="cuda") for _ in range(n)]
    refusals = 0
    for i in range(12):
        rows = [int(x) for x in np.where(rng.random(n) < 0.6, rng.integers(1, 20, n), 0)]
        rows[0] = max(rows[0], 1)
        parents = [R.tree(m, rng) if m else [] for m in rows]
        step = Step(ctx, cache, rows, parents, seed=100 * seed + i)
        step.reserve()
        want, _ = book.reserve(rows)
        assert step.reserved.tolist() == want
        step.append()
        accepted, path, at = [], [], 0
        for s, m in enumerate(rows):
            way = R.ways(parents[s])[int(rng.integers(0, m))] if m else []
            x = step.qkv[0][at:at + m].reshape(m, NQ + 2 * NKV, D)[:, NQ + NKV:].double()
            accepted.append(len(way) - 1)
            path += way + [-1] * (m - len(way))
            if want[s][0]:
                book.lens[s] += len(way)
                told[s] = torch.cat([told[s], x[way]])
            refusals += m > 0 and not want[s][0]
            at += m
        step.accepted.copy_(cuda(accepted))
        step.path.copy_(cuda(path))
        step.commit()
        same(cache, book)
        for s in range(n):
            assert torch.equal(R.rows_of(cache, 0, s, torch.arange(book.lens[s], device="cuda"))[1], told[s]), s
        src = [int(x) for x in np.where(rng.random(n) < 0.2, rng.integers(0, n, n), -1)]
        old = list(told)
        for s, f in enumerate(src):
            if f >= 0 and f != s and not (src[f] >= 0 and src[f] != f):
                told[s] = old[f]
        ctx.pages_fork(cache, cuda(src))
        book.fork(src)
        cut = [int(x) for x in np.where(rng.random(n) < 0.2, rng.integers(0, 3 * page, n), -1)]
        ctx.pages_truncate(cache, cuda(cut))
        book.truncate(cut)
        told = [t[:book.lens[s]] for s, t in enumerate(told)]
    assert refusals > 0


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("n,n_pages,page", [(9, 14, 32), (40, 60, 64)])
def test_branches_in_the_middle_of_steps(ctx, n, n_pages, page, seed):  # noqa: F811
    """Branches made before a step's append or before its commit: the source's step goes on, a branch that had rows
    in it has lost them, and nobody's tokens are another's."""
    rng = np.random.default_rng(50 + seed)
    cache = filled(ctx, n, n_pages, NKV, 5, 1, page, seed)
    book = book_of(cache)
    told = [torch.zeros((0, NKV, D), dtype=torch.float64, device="cuda") for _ in range(n)]
    made = 0
    for i in range(14):
        rows = [int(x) for x in np.where(rng.random(n) < 0.5, rng.integers(1, 12, n), 0)]
        rows[0] = max(rows[0], 1)
        step = Step(ctx, cache, rows, seed=100 * seed + i)
        step.reserve()
        want, _ = book.reserve(rows)
        assert step.reserved.tolist() == want
        src = [int(x) for x in np.where(rng.random(n) < 0.15, rng.integers(0, n, n), -1)]
        goes = [src[s] >= 0 and src[s] != s and not (src[src[s]] >= 0 and src[src[s]] != src[s]) for s in range(n)]
        when = i % 2
        for phase in range(2):
            if phase == when:
                ctx.pages_fork(cache, cuda(src))
                book.fork(src)
                told = [told[src[s]] if goes[s] else told[s] for s in range(n)]
                made += sum(goes)
            if phase == 0:
                step.append()
        step.accepted.copy_(cuda([int(rng.integers(0, m)) if m else -1 for m in rows]))
        step.commit("chain")
        at = 0
        for s, m in enumerate(rows):
            k = step.accepted[s].item() + 1
            if m and want[s][0] and not goes[s]:
                book.lens[s] += k
                told[s] = torch.cat([told[s], step.qkv[0][at:at + k].reshape(k, -1, D)[:, NQ + NKV:].double()])
            at += m
        same(cache, book)
        assert book.named() == book.refs
        for s in range(n):
            assert torch.equal(R.rows_of(cache, 0, s, torch.arange(book.lens[s], device="cuda"))[1], told[s]), (i, s)
        cut = [0 if rng.random() < 0.15 else -1 for _ in range(n)]
        ctx.pages_truncate(cache, cuda(cut))
        book.truncate(cut)
        told = [t[:book.lens[s]] for s, t in enumerate(told)]
    assert made > 5


def test_an_aborted_call_for_room(ctx):  # noqa: F811
    """Nobody has room after a call that was aborted, also where the word is cleared before the rest of the step."""
    cache = parent_and_branch(ctx, 80, n_pages=6)
    step = Step(ctx, cache, [0, 3], seed=9)
    step()
    ctx.sync()
    assert cache.lens.tolist() == [100, 83]
    k = cache.k.clone()
    torch.cuda.synchronize()
    ctx.set_abort(True)
    step.reserve()
    torch.cuda.synchronize()
    ctx.set_abort(False)
    with pytest.raises(Exception):
        ctx.sync()
    step.append()
    step.accept()
    step.commit()
    ctx.sync()
    assert torch.equal(cache.k, k) and cache.lens.tolist() == [100, 83]
