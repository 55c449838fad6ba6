"""GPU: the drafts of a batch checked from given random numbers, against the rules in 64 bits
(tests/paged_ref.py); whole numbers, compared exactly."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R
from momij_amd.ops import Context
from momij_amd.paged import RowBatch, tree_masks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    with torch.cuda.stream(c.stream):
        yield c
    c.close()


def cuda(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def go(ctx, rows, logits, tokens, T, ua, us, parents=None, q=None, pad=0, max_rows=None):
    """The call; accepted, path and token as lists.  Rows of no sequence stay as they are."""
    start = np.concatenate([[0], np.cumsum(rows)])
    total, n = int(start[-1]), len(rows)
    anc = None if parents is None else cuda([m for p in parents for m in tree_masks(p)] + [-1] * pad, torch.int64)
    b = RowBatch(cuda(start), total + pad, max_rows or max(max(rows), 1), anc)
    accepted, token = cuda([55] * n), cuda([55] * n)
    path = cuda([55] * (total + pad))
    ctx.accept_rows(b, logits, tokens, T, ua, us, accepted, path, token, q=q)
    ctx.sync()
    assert path[total:].tolist() == [55] * pad
    return accepted.tolist(), path[:total].tolist(), token.tolist()


def want(rows, logits, tokens, T, ua, us, parents=None, q=None):
    acc, path, token, at = [], [], [], 0
    x, t, Ts, a, u = (y.cpu() for y in (logits, tokens, T, ua, us))
    q = q.cpu() if q is not None else None
    for s, m in enumerate(rows):
        if m == 0:
            acc.append(0)
            token.append(-1)
            continue
        par = parents[s] if parents else R.tree(m)
        r = R.accept(x[at:at + m], par, t[at:at + m], float(Ts[s]), a[at:at + m], u[s],
                     None if q is None else q[at:at + m])
        acc.append(r[0])
        path += r[1]
        token.append(r[2])
        at += m
    return acc, path, token


def make(rows, V, seed, q=False, ld=None, spread=2.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    total = sum(rows)
    wide = torch.randn((total, ld or V), generator=gen, device="cuda") * spread
    logits = wide[:, :V]
    k = min(V, 4)
    tokens = logits.topk(k, -1).indices.gather(1, torch.randint(0, k, (total, 1), generator=gen, device="cuda"))
    tokens = tokens.roll(1, 0)[:, 0].int().contiguous()
    d = dict(logits=logits, tokens=tokens, T=torch.rand(len(rows), generator=gen, device="cuda") + 0.3,
             ua=torch.rand(total, generator=gen, device="cuda"), us=torch.rand(len(rows), generator=gen, device="cuda"))
    if q:
        y = torch.randn((total, (ld or V) + 3), generator=gen, device="cuda")[:, :V]
        d["q"] = torch.softmax(logits + 0.5 * y, -1)
        d["tokens"] = torch.multinomial(d["q"], 1, generator=gen).roll(1, 0)[:, 0].int().contiguous()
    return d


@pytest.mark.parametrize("V", [1, 2, 7, 63, 1000, 8191, 8192, 8193, 32001, 151936])
@pytest.mark.parametrize("q", [False, True])
@pytest.mark.parametrize("rows", [[1], [9], [3, 0, 1, 17, 8, 64]], ids=str)
def test_chains(ctx, V, q, rows):
    for seed in range(4):
        d = make(rows, V, seed, q)
        assert go(ctx, rows, **d) == want(rows, **d), seed


@pytest.mark.parametrize("V", [3, 500, 20000])
@pytest.mark.parametrize("seed", range(5))
def test_trees(ctx, V, seed):
    rng = np.random.default_rng(seed)
    rows = [17, 1, 30, 64, 0, 5]
    parents = [R.tree(m, rng) if m else [] for m in rows]
    d = make(rows, V, seed)
    # drafts that their parent's row finds probable, siblings often the same
    at = 0
    for m, par in zip(rows, parents):
        top = d["logits"][at:at + m].topk(min(3, V), -1).indices
        for r in range(1, m):
            d["tokens"][at + r] = top[par[r], int(rng.integers(0, min(3, V)))]
        at += m
    assert go(ctx, rows, parents=parents, pad=3, **{k: pad3(k, v) for k, v in d.items()}) == want(
        rows, parents=parents, **d)


def pad3(name, t):
    if name in ("T", "us"):
        return t
    return torch.cat([t, t[-1:].expand(3, *t.shape[1:])])


def test_wide_rows(ctx):
    """Rows that are slices of wider ones, off a 16-byte line."""
    rows = [5, 9]
    d = make(rows, 1001, 3, True, ld=1003)
    assert d["logits"].stride(0) == 1003
    assert go(ctx, rows, **d) == want(rows, **d)


@pytest.mark.parametrize("u", [0.0, 0.3, 0.7, 1.0 - 2.0 ** -24])
@pytest.mark.parametrize("refused", [1, 2, 3, 20, 63])
@pytest.mark.parametrize("near", [True, False])
def test_refusals_below_one_row(ctx, refused, near, u):
    """Drafts that were certain, all of one row and all refused, in the same chunk of ids or in many: the
    token is sampled from what they leave."""
    V, rows = 30011, [refused + 1]
    d = make(rows, V, refused)
    ids = torch.arange(refused) * (7 if near else V // refused - 1) + 4090
    d["tokens"][1:] = (ids % V).int().cuda()
    d["logits"] = d["logits"].clone()
    d["logits"][0, d["tokens"][1:].long()] += 3.0  # a good part of the row
    d["ua"].fill_(1.0)  # (u rest > e where the row has another id)
    d["us"].fill_(u)
    got = go(ctx, rows, parents=[[-1] + [0] * refused], **d)
    assert got == want(rows, parents=[[-1] + [0] * refused], **d)
    assert got[0] == [0] and got[2][0] not in d["tokens"][1:].tolist()


@pytest.mark.parametrize("rows,parents,q", [([3], None, False), ([3], None, True), ([6], [[-1, 0, 0, 0, 0, 1]], False)],
                         ids=["certain", "drawn", "tree"])
def test_the_largest_vocabulary(ctx, rows, parents, q):
    """2048 chunks of ids: several a thread of the block that samples."""
    V = 1 << 23
    for ua, us in ((1.0, 0.25), (0.0, 0.9999)):
        d = make(rows, V, 5, q, spread=6.0)
        d["ua"].fill_(ua)
        d["us"].fill_(us)
        assert go(ctx, rows, parents=parents, **d) == want(rows, parents=parents, **d), (ua, us)


@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0 ** -24])
@pytest.mark.parametrize("q", [False, True])
def test_ends_of_the_uniforms(ctx, u, q):
    rows = [6, 1, 9]
    d = make(rows, 700, 1, q)
    d["ua"].fill_(u)
    d["us"].fill_(u)
    d["logits"] = d["logits"].clone()
    d["logits"][:, :5] = -math.inf  # ids that u = 0 must not take
    d["logits"][:, -5:] = -math.inf  # nor u near 1
    if q:
        d["q"][:, :5] = 0.0
    got = go(ctx, rows, **d)
    assert got == want(rows, **d)
    assert all(5 <= t < 695 for t in got[2])


@pytest.mark.parametrize("T", [0.0, 1e-5, math.nan, -1.0])
@pytest.mark.parametrize("q", [False, True])
def test_greedy(ctx, T, q):
    """The lowest id of the greatest logit; drafts equal to it are kept."""
    rows = [9, 4]
    d = make(rows, 9000, 2, q)
    x = d["logits"] = d["logits"].clone()
    x[:, 8500], x[:, 17], x[:, 8191], x[:, 8192] = 50.0, 50.0, 50.0, 50.0  # ties over chunks
    d["tokens"].fill_(17)
    d["tokens"][5] = 8191
    d["T"].fill_(T)
    if q:
        d["q"][:, 17] = 0.3
    got = go(ctx, rows, **d)
    assert got == ([4, 3], [0, 1, 2, 3, 4, -1, -1, -1, -1, 0, 1, 2, 3], [17, 17])


def test_logits_that_are_no_numbers(ctx):
    """NaN and -inf have no probability, infinities share the row, a row without any gives -1."""
    V, rows = 9000, [1] * 6 + [3]
    d = make(rows, V, 5)
    x = d["logits"] = d["logits"].clone()
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 8300] = -5.0
    x[3, 100:8999] = math.nan
    x[4, [3, 8800]] = math.inf
    x[5] = math.inf
    x[6] = -math.inf  # a row of none whose draft has no probability either
    got = go(ctx, rows, **d)
    assert got == want(rows, **d)
    assert got[2][0] == got[2][1] == got[2][6] == -1 and got[2][2] == 8300 and got[2][4] in (3, 8800)


def test_drafts_that_are_no_ids(ctx):
    rows = [4, 4]
    d = make(rows, 500, 7)
    d["ua"].fill_(0.0)
    d["tokens"][1], d["tokens"][5] = -1, 500
    got = go(ctx, rows, **d)
    assert got == want(rows, **d) and got[0] == [0, 0]


@pytest.mark.parametrize("refused", [1, 2, 3])
@pytest.mark.parametrize("u", [0.0, 1e-9, 0.4, 0.99])
@pytest.mark.parametrize("others", [True, False])
def test_refused_drafts_that_were_almost_all(ctx, refused, u, others):
    """What is left of a chunk of ids, or of the row, is lost in the drafts' own weight."""
    V = 12301
    rows, parents = [refused + 1], [[-1] + [0] * refused]
    d = make(rows, V, refused)
    x = torch.randn(rows[0], V, generator=torch.Generator().manual_seed(refused)) - 27.0
    ids = [100 + 50 * i for i in range(refused)]
    x[0, ids] = 0.0
    if others:  # as much in another chunk
        x[0, 9000:9010] = 0.0
    d["logits"], d["T"] = x.cuda(), torch.ones(1, device="cuda")
    d["tokens"][1:] = cuda(ids)
    d["ua"].fill_(1.0)
    d["us"].fill_(u)
    if not others:
        d["ua"][refused] = 2.0  # (the last of them would be accepted for any u below 1)
    got = go(ctx, rows, parents=parents, **d)
    assert got == want(rows, parents=parents, **d)
    assert got[0] == [0] and got[2][0] not in ids


@pytest.mark.parametrize("V", [500, 20001])
@pytest.mark.parametrize("form", ["certain", "drawn", "tree"])
def test_drafts_far_from_any_id(ctx, V, form):
    """Below the first id and past the last by more than a chunk of ids, alone and beside drafts that are."""
    far = [-1, -4096, -4097, -5000, -2 ** 31, V, V + 4096, V + 100000, 2 ** 31 - 1, 2 ** 31 - 4096]
    for i, bad in enumerate(far):
        parents = [[-1, 0, 0, 0, 2]] if form == "tree" else None
        rows = [5] if parents else [2, 3]
        d = make(rows, V, i, form == "drawn")
        d["ua"].fill_(0.999)
        d["tokens"][1] = bad
        d["tokens"][4] = bad
        assert go(ctx, rows, parents=parents, **d) == want(rows, parents=parents, **d), bad


def test_draft_distributions_at_their_ends(ctx):
    """q of 0, below 0 and NaN at the draft: never accepted; q that covers p: the row's own probabilities
    stand in where nothing is left; q of 1 at the draft: what is left is p without it."""
    V, rows = 300, [2] * 6
    d = make(rows, V, 9, True)
    d["ua"].fill_(0.999)
    p = torch.softmax(d["logits"].double() / d["T"].double().repeat_interleave(2)[:, None], -1)
    for s, y in enumerate((0.0, -1.0, math.nan)):
        d["q"][2 * s, d["tokens"][2 * s + 1].long()] = y
    d["q"][6] = (p[6] * 1.01).float()
    d["q"][8] = 0.0
    d["q"][8, d["tokens"][9].long()] = 1.0
    d["q"][10] = math.nan
    got = go(ctx, rows, **d)
    assert got == want(rows, **d)
    assert got[0][:3] == [0, 0, 0] and got[0][5] == 0


def test_second_of_equal_siblings(ctx):
    """A refused token has nothing left: its twin is refused whatever its number."""
    V, rows = 50, [4]
    d = make(rows, V, 1)
    d["T"].fill_(1.0)
    d["logits"] = torch.zeros_like(d["logits"])
    d["tokens"].copy_(cuda([0, 7, 7, 8]))
    d["ua"].copy_(torch.tensor([0.0, 0.9, 0.0, 0.0]))
    got = go(ctx, rows, parents=[[-1, 0, 0, 0]], **d)
    assert got == ([1], [0, 3, -1, -1], got[2])
    assert got == want(rows, parents=[[-1, 0, 0, 0]], **d)


def test_rows_past_max_rows(ctx):
    rows = [9, 2]
    d = make(rows, 100, 1)
    d["ua"].fill_(0.0)
    b = RowBatch(cuda([0, 9, 11]), 11, 4)
    accepted, token, path = cuda([55] * 2), cuda([55] * 2), cuda([55] * 11)
    ctx.accept_rows(b, d["logits"], d["tokens"], d["T"], d["ua"], d["us"], accepted, path, token)
    ctx.sync()
    assert accepted.tolist() == [3, 1] and path.tolist() == [0, 1, 2, 3] + [55] * 5 + [0, 1]


def test_no_rows_at_all(ctx):
    b = RowBatch(cuda([0, 0, 0]), 0, 1)
    e = torch.zeros((0, 100), device="cuda")
    i, f = cuda([]), torch.zeros(0, device="cuda")
    accepted, token = cuda([5, 5]), cuda([5, 5])
    ctx.accept_rows(b, e, i, torch.ones(2, device="cuda"), f, torch.zeros(2, device="cuda"), accepted, i, token)
    ctx.sync()
    assert accepted.tolist() == [0, 0] and token.tolist() == [-1, -1]


def test_1024_sequences_and_repeats(ctx):
    rows = [1 + i % 3 for i in range(1024)]
    d = make(rows, 2000, 4, True)
    got = go(ctx, rows, **d)
    assert got == want(rows, **d)
    assert got == go(ctx, rows, **d)


@pytest.mark.parametrize("q", [False, True])
def test_the_first_token_is_the_targets(ctx, q):
    """Whatever the draft, the first token emitted has the target's probability: over 16384 sequences of the same
    row, counts within five standard deviations of it."""
    V, n = 6, 1024
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    x = torch.tensor([1.0, 0.3, -0.5, 2.0, 0.0, -2.0], device="cuda")
    y = torch.tensor([0.0, 0.8, 0.5, 1.0, -9.0, 0.4], device="cuda")
    p, dq = torch.softmax(x.double(), -1), torch.softmax(y, -1)
    count = torch.zeros(V, device="cuda")
    for _ in range(16):
        drawn = torch.multinomial(dq, n, replacement=True, generator=gen).int()
        tokens = torch.stack([torch.zeros_like(drawn), drawn], 1).reshape(-1).contiguous()
        acc, path, token = go(ctx, [2] * n, x.expand(2 * n, V).contiguous(), tokens, torch.ones(n, device="cuda"),
                              torch.rand(2 * n, generator=gen, device="cuda"),
                              torch.rand(n, generator=gen, device="cuda"),
                              q=dq.expand(2 * n, V).contiguous() if q else None)
        first = torch.where(cuda(acc) > 0, drawn, cuda(token))
        count += torch.bincount(first.long(), minlength=V)
    dev = (p * (1 - p) * 16 * n).sqrt()
    assert bool(((count.double() - p * 16 * n).abs() <= 5 * dev).all())
