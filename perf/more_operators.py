"""Timed calls of a verify step of many requests: their pages, the attention over them, their drafts.

A server keeps the keys and values of its requests in fp16 pages of one pool (every layer's page p at
the same index), a table row and a length for each.  A step makes room for a batch of rows (`reserve`;
shared pages are copied before they are written), appends their keys and values (normed and rotated),
attends over the pages, checks the drafts against the target's probabilities from given random numbers
(`accept`), and moves the rows of the accepted paths together (`commit`).  `fork` lets requests share
a prompt's pages, `truncate` frees them.

Heads of 128; the head counts are those of the benchmark model and of the tests, the rows a sequence
those of a pass: one (decode), 9 (a K = 8 chain), 17 (a 16-node tree), 64 (a prefill chunk).  Sizes of a
batch go by the case alone (lengths spread evenly over their logarithm, row counts over 1 .. M);
which sequence has which goes by the seed.

Pages hold 32, 64, 128 or 256 tokens of a layer, by KV head in units of 32 tokens by 128 dims, 8 KB of K
and of V each, in the order of the matrix operands.  Of token t (of the unit) and dim d, K is at
[t / 4 % 2][d / 32][d / 8 % 4][t / 8][t % 4][d % 8] and V at [d / 16][t / 8][d % 16][t % 8].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 128
EPS, ROPE_BASE = 1e-6, 1e6
GREEDY = 1e-5  # temperatures up to this one take the most probable token
VOCAB = 151936

_context = None


def context():
    """One context per program; the program's own torch work runs on the context's stream, so
    inputs and outputs need no events."""
    global _context
    if _context is None:
        from momij_amd.ops import Context

        _context = Context(0)
        torch.cuda.set_stream(_context.stream)
    return _context


# ------------------------------------------------------------------------------------ cases
def listed():
    heads = dict(nq=16, nkv=4)
    return [
        # a decode step of 64 requests of 200 to 8000 tokens; of one request far into a context
        dict(name="attn_decode_batch", kind="attn", **heads, n=64, M=1, ragged=False, tree=False,
             lo=200, hi=8000, page=64, window=0),
        dict(name="attn_decode_long", kind="attn", **heads, n=1, M=1, ragged=False, tree=False,
             lo=131000, hi=131000, page=64, window=0),
        # draft trees of up to 16 nodes of 16 requests
        dict(name="attn_verify_trees", kind="attn", **heads, n=16, M=17, ragged=True, tree=True,
             lo=500, hi=8000, page=32, window=0),
        # a prefill chunk of each of four requests
        dict(name="attn_prefill", kind="attn", **heads, n=4, M=64, ragged=False, tree=False, lo=4000,
             hi=16000, page=128, window=0),
        # queries and keys of one request's decode step; of the K = 8 chains of 64 requests
        dict(name="append_decode", kind="append", **heads, n=1, M=1, ragged=False, tree=False, lo=5000,
             hi=5000, page=64, rope=64),
        dict(name="append_chains", kind="append", **heads, n=64, M=9, ragged=True, tree=False, lo=100,
             hi=4000, page=64, rope=64),
        # three samples of one prompt; seven more of each of eight prompts, which go on themselves
        dict(name="branch_one", kind="branch", nkv=4, n=4, parents=1, M=1, lo=700, hi=700, page=64,
             layers=24, go_on=False),
        dict(name="branch_many", kind="branch", nkv=4, n=64, parents=8, M=9, lo=200, hi=3000, page=64,
             layers=24, go_on=True),
        # the accepted path of one request's draft tree; of 64 requests'
        dict(name="commit_one", kind="commit", nkv=4, n=1, M=17, ragged=False, tree=True, lo=90, hi=90,
             page=64, layers=24),
        dict(name="commit_batch", kind="commit", nkv=4, n=64, M=17, ragged=True, tree=True, lo=30,
             hi=120, page=64, layers=24),
        # one request's K = 8 chain, its drafts certain (a suffix index's); the chains that a draft
        # model proposed for 64 requests, with its distributions, a quarter of the requests greedy
        dict(name="accept_one", kind="accept", n=1, M=9, ragged=False, tree=False, V=VOCAB, q=False,
             greedy=0),
        dict(name="accept_batch", kind="accept", n=64, M=9, ragged=True, tree=False, V=VOCAB, q=True,
             greedy=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn"] * 5 + ["append", "branch", "commit", "accept", "accept"])
    nq, nkv = rng.choice([(16, 4), (16, 4), (16, 4), (8, 8), (16, 2), (32, 4), (12, 4), (16, 1)])
    page = rng.choice([32, 64, 64, 128, 256])
    if kind == "attn":
        n, M = _log(rng, 1, 64), _log(rng, 1, 64)
        most = min(131000, 130000 * 4 // (n * max(nkv, 4)), 16 * 64 * 36000 // (n * nq * M))
        hi = _log(rng, 64, max(most, 65))
        return dict(kind=kind, nq=nq, nkv=nkv, n=n, M=M, ragged=rng.random() < 0.5,
                    tree=rng.random() < 0.4, lo=rng.randint(0, hi), hi=hi, page=page,
                    window=rng.choice([0, 0, 0, 512, 1024]))
    if kind == "append":
        return dict(kind=kind, nq=nq, nkv=nkv, n=_log(rng, 1, 64), M=_log(rng, 1, 9),
                    ragged=rng.random() < 0.5, tree=rng.random() < 0.4, lo=rng.randint(0, 100),
                    hi=_log(rng, 101, 4000), page=page, rope=rng.choice([0, 32, 64, 64, 128]))
    if kind == "branch":
        n = _log(rng, 2, 64)
        return dict(kind=kind, nkv=nkv if nkv <= 4 else 4, n=n, parents=rng.randint(1, min(8, n - 1)),
                    M=_log(rng, 1, 9), lo=rng.randint(1, 200), hi=_log(rng, 201, 2000),
                    page=rng.choice([32, 64]), layers=rng.randint(1, 24), go_on=rng.random() < 0.5)
    if kind == "commit":
        return dict(kind=kind, nkv=nkv if nkv <= 4 else 4, n=_log(rng, 1, 64), M=_log(rng, 2, 17),
                    ragged=rng.random() < 0.5, tree=rng.random() < 0.8, lo=rng.randint(0, 30),
                    hi=_log(rng, 31, 120), page=rng.choice([32, 64]), layers=rng.randint(1, 24))
    n, tree = _log(rng, 1, 64), rng.random() < 0.3
    return dict(kind=kind, n=n, M=rng.randint(1, min(17, 300 // n)), ragged=rng.random() < 0.5,
                tree=tree, V=rng.choice([_log(rng, 500, 40000), _log(rng, 40000, VOCAB), VOCAB]),
                q=not tree and rng.random() < 0.6, greedy=rng.randint(0, n // 2))


def _sizes(case):
    """Committed lengths and row counts of the batch, before the seed deals them out."""
    n = case["n"]
    lo, hi = max(case.get("lo", 1), 1), max(case.get("hi", 1), 1)
    lens = [round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * (i / (n - 1) if n > 1 else 1)))
            for i in range(n)]
    if case.get("lo") == 0:
        lens[0] = 0
    rows = [case["M"] - (5 * i) % case["M"] if case.get("ragged") else case["M"] for i in range(n)]
    if case["kind"] == "branch":  # prompts first, then their branches
        p = case["parents"]
        lens = [lens[i * (n - 1) // max(p - 1, 1)] for i in range(p)]
        rows = [case["M"] if i >= p or case["go_on"] else 0 for i in range(n)]
    return lens, rows


# ----------------------------------------------------------------------------------- inputs
def _masks(rng, rows, tree):
    """Of each row, the rows of its sequence that it sees (its ancestors and itself) as bits, and the
    parents; in a tree every node hangs off one of the six rows before it."""
    anc, parents = [], []
    for m in rows:
        par = [-1] + [int(rng.integers(max(0, i - 6), i)) if tree else i - 1 for i in range(1, m)]
        bits = []
        for r in range(m):
            bits.append((bits[par[r]] if r else 0) | 1 << r)
        anc += bits
        parents.append(par[:m])
    return anc, parents


def _inputs(case, seed):
    """Everything the call reads, from the seed alone (also what exact() starts from)."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, n = case["kind"], case["n"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    def ints(x, dtype=torch.int32):
        return torch.from_numpy(np.asarray(x, np.int64)).to(dtype).cuda()

    lens, rows = _sizes(case)
    if kind != "branch":
        order = rng.permutation(n)
        lens, rows = [lens[i] for i in order], [rows[i] for i in order]
    start = np.concatenate([[0], np.cumsum(rows)])
    R = int(start[-1])
    tree = bool(case.get("tree"))
    anc, parents = _masks(rng, rows, tree)
    d = dict(row_start=ints(start), rows=R, parents=parents,
             anc=ints(np.array(anc, np.uint64).astype(np.int64), torch.int64) if tree else None)
    if kind == "accept":
        V = case["V"]
        # a few tokens of each row stand out, as after most texts
        logits = randn(R, V) * 2.0
        few = torch.linspace(2.0, 0.25, 8, device="cuda").expand(R, 8)
        logits.scatter_add_(1, logits.topk(8, dim=-1).indices, few)
        first = ints(start[np.repeat(np.arange(n), rows)], torch.int64)
        par = first + ints([max(p, 0) for ps in parents for p in ps], torch.int64)
        if case["q"]:
            # a draft model near the target, and the tokens drawn from it
            q = torch.softmax((logits + randn(R, V)) * 1.25, -1)
            g = torch.empty(R, V, device="cuda").exponential_(generator=gen)
            token = (q / g).argmax(-1)[par]
            d["q"] = q
        else:
            # what the target itself finds probable, another one for each sibling
            top = (logits + 0.3 * randn(R, V)).topk(8, dim=-1).indices
            at = [sum(p == ps[j] for j in range(i)) for ps in parents for i, p in enumerate(ps)]
            token = top[par, ints(at, torch.int64).clamp_max(7)]
        temp = np.where(np.arange(n) < case["greedy"], 0.0, rng.uniform(0.6, 1.1, n))
        d.update(logits=logits * 2.0, token=token.to(torch.int32),
                 temperature=torch.from_numpy(rng.permutation(temp).astype(np.float32)).cuda(),
                 u_accept=torch.rand(R, generator=gen, device="cuda"),
                 u_sample=torch.rand(n, generator=gen, device="cuda"))
        return d
    nkv, page, layers = case["nkv"], case["page"], case.get("layers", 1)
    if kind == "branch":
        # prompts, and old branches of a few tokens that the new ones take the place of
        lens += [int(x) for x in rng.integers(1, 2 * page, n - len(lens))]
    room = [x + (0 if kind == "branch" else m) for x, m in zip(lens, rows)]
    blocks = [-(-x // page) for x in room]
    if kind == "branch":  # (sizes that do not go by the seed)
        p = case["parents"]
        width = max(blocks[:p] + [2]) + 2
        pages = sum(blocks[:p]) + 2 * (n - p) + n * (2 + case["M"] // page)
    else:
        width, pages = max(blocks) + 2, sum(blocks) + sum(blocks) // 10 + 1
    perm = rng.permutation(pages)  # where the pages lie in the pool: anywhere, as after a while
    table = np.full((n, width), -1, np.int64)
    for i, b in enumerate(blocks):
        at = sum(blocks[:i])
        table[i, :b] = perm[at:at + b]
    refs = np.zeros(pages, np.int64)
    refs[table[table >= 0]] = 1
    d.update(lens=ints(lens), table=ints(table), refs=ints(refs),
             k=randn(layers, pages, nkv, page // 32, 2, 4, 4, 4, 4, 8, dtype=torch.float16),
             v=randn(layers, pages, nkv, page // 32, 8, 4, 16, 8, dtype=torch.float16))
    if kind == "attn":
        d["q"] = (randn(R, case["nq"] * D) * 2.0).half()
    elif kind == "append":
        d.update(qkv=(randn(R, (case["nq"] + 2 * nkv) * D) * 1.5).half(),
                 qw=(1.0 + 0.1 * randn(D)).half(), kw=(1.0 + 0.1 * randn(D)).half())
    elif kind == "branch":
        d["keep"] = ints([-1] * p + [0] * (n - p))
        d["source"] = ints([-1] * p + [i % p for i in range(n - p)])
    elif kind == "commit":
        accepted, path = [], []
        for ps in parents:  # the way to a row far down, as far as it was accepted
            r, way = int(rng.integers(len(ps) // 2, len(ps))), []
            while r >= 0:
                way.insert(0, r)
                r = ps[r]
            way = way[:int(rng.integers(1, len(way) + 1))]
            accepted.append(len(way) - 1)
            path += way + [-1] * (len(ps) - len(way))
        d.update(accepted=ints(accepted), path=ints(path))
    return d


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    kind, n, R = case["kind"], case["n"], st["rows"]

    def out(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    if kind in ("attn", "append"):
        st["out"] = out(R, case["nq"] * D, dtype=torch.float16)
    elif kind == "branch":
        st["reserved"] = out(n, 4)
    elif kind == "commit":
        st["new_lens"] = out(n)
    else:
        st.update(new_accepted=out(n), new_path=out(R), new_token=out(n))
    if own:
        from momij_amd.paged import PagedCache, RowBatch

        st["ctx"] = ctx = context()
        st["batch"] = RowBatch(st["row_start"], R, case["M"], st["anc"])
        if kind != "accept":
            st["cache"] = PagedCache.over(ctx, *(st[x] for x in ("k", "v", "table", "lens", "refs")))
        if kind == "append":
            st["cfg"] = dict(H=2048, nQ=case["nq"], nKV=case["nkv"], D=D, rope_dim=case["rope"],
                             rope_base=ROPE_BASE, eps=EPS, window=0, C=0, gs=64)
    return st


# -------------------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if "ctx" in st else _run_plain(st)


def _run_own(st):
    case, ctx, batch = st["case"], st["ctx"], st["batch"]
    kind, cache = case["kind"], st.get("cache")
    if kind == "attn":
        ctx.paged_attn(cache, 0, batch, st["q"], case["nq"], st["out"], window=case["window"])
        return dict(out=st["out"])
    if kind == "append":
        ctx.paged_append(st["cfg"], cache, 0, batch, st["qkv"], st["qw"], st["kw"], st["out"])
        return dict(q=st["out"], k=st["k"], v=st["v"])
    if kind == "branch":
        ctx.pages_truncate(cache, st["keep"])
        ctx.pages_fork(cache, st["source"])
        ctx.pages_reserve(cache, batch, st["reserved"])
        return {x: st[x] for x in ("table", "lens", "refs", "reserved", "k", "v")}
    if kind == "commit":
        ctx.pages_commit(cache, batch, st["accepted"], st["path"], st["new_lens"])
        return dict(k=st["k"], v=st["v"], lens=st["new_lens"])
    ctx.accept_rows(batch, st["logits"], st["token"], st["temperature"], st["u_accept"],
                    st["u_sample"], st["new_accepted"], st["new_path"], st["new_token"], q=st.get("q"))
    return dict(accepted=st["new_accepted"], path=st["new_path"], token=st["new_token"])


class _Rows:
    """The batch's rows, and the same by sequence, [n, M] with a mask of those that there are."""

    def __init__(self, st):
        case, start = st["case"], st["row_start"].long()
        M, R, dev = case["M"], st["rows"], start.device
        self.count = start[1:] - start[:-1]
        self.local = torch.arange(M, device=dev)
        self.there = self.local < self.count[:, None]
        self.row = (start[:-1, None] + self.local).clamp_max(max(R - 1, 0))
        self.seq = torch.searchsorted(start[1:], torch.arange(R, device=dev), right=True)
        self.at = torch.arange(R, device=dev) - start[self.seq]
        below = torch.ones((M, M), dtype=torch.bool, device=dev).tril()
        if st["anc"] is None:
            self.sees = below[self.at]
        else:
            self.sees = (st["anc"][:, None] >> self.local & 1).bool()
        self.depth = (self.sees & below[self.at]).sum(-1) - 1


def _run_plain(st):
    return globals()["_plain_" + st["case"]["kind"]](st)


def _rows_of_pages(st, pages):
    """K and V rows of pages [...] in 32 bits, [..., nkv, page, 128], of layer 0."""
    k, v = st["k"][0][pages], st["v"][0][pages]
    k = k.movedim((-3, -6, -2), (-6, -5, -4)).float()
    v = v.movedim((-3, -1), (-4, -3)).float()
    shape = pages.shape + (st["case"]["nkv"], st["case"]["page"], D)
    return k.reshape(shape), v.reshape(shape)


def _read(st, pages, t):
    """K and V of tokens t of pages, in all layers, as the pools' rows of them lie."""
    u, t = t // 32, t % 32
    return (st["k"][:, pages, :, u, t // 4 % 2, :, :, t // 8, t % 4],
            st["v"][:, pages, :, u, :, t // 8, :, t % 8])


def _write(st, pages, t, k, v):
    """The same the other way, [rows, nkv, 128] or as they were read."""
    head = (pages.shape[0], st["k"].shape[0], st["k"].shape[2])
    u, t = t // 32, t % 32
    st["k"][:, pages, :, u, t // 4 % 2, :, :, t // 8, t % 4] = k.reshape(head + (4, 4, 8))
    st["v"][:, pages, :, u, :, t // 8, :, t % 8] = v.reshape(head + (8, 16))


def _plain_attn(st):
    case, b = st["case"], _Rows(st)
    n, M, nq, nkv, page = (case[x] for x in ("n", "M", "nq", "nkv", "page"))
    G, blocks = nq // nkv, st["table"].shape[1] - 2  # (two spare entries)
    T = blocks * page
    k, v = _rows_of_pages(st, st["table"][:, :blocks].long().clamp_min(0))
    k, v = (x.transpose(1, 2).reshape(n * nkv, T, D) for x in (k, v))
    q = st["q"][b.row].float().reshape(n, M, nkv, G, D).transpose(1, 2).reshape(n * nkv, M * G, D)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * D ** -0.5
    pos, L = torch.arange(T, device=q.device), st["lens"].long()[:, None, None]
    first = (L + b.depth[b.row][..., None] - case["window"] + 1 if case["window"] else torch.zeros_like(L))
    new = (pos - L).clamp(0, M - 1).expand(n, M, T)
    ok = (pos < L) & (pos >= first) | (pos >= L) & (pos < L + M) & b.sees[b.row].gather(2, new)
    ok = ok[:, None, :, None].expand(n, nkv, M, G, T).reshape(n * nkv, M * G, T)
    s = s.masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p, v).reshape(n, nkv, M, G, D).transpose(1, 2).reshape(n, M, nq * D).half()
    return dict(out=o[b.seq, b.at])


def _slots(st, seq, pos):
    """Page and token in it of positions of sequences."""
    page = st["case"]["page"]
    return st["table"].long()[seq, pos // page], pos % page


def _plain_append(st):
    case, b = st["case"], _Rows(st)
    nq, nkv, rope = case["nq"], case["nkv"], case["rope"]
    x = st["qkv"].float().reshape(-1, nq + 2 * nkv, D)
    L = st["lens"].long()[b.seq]
    qk = x[:, :nq + nkv]
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    qk = qk * torch.cat([st["qw"].float().expand(nq, D), st["kw"].float().expand(nkv, D)])
    if rope:
        half = rope // 2
        f = ROPE_BASE ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
        th = (L + b.depth).double()[:, None, None] * f
        c, s = th.cos().float(), th.sin().float()
        y, z = qk[..., :half], qk[..., half:rope]
        qk = torch.cat([y * c - z * s, z * c + y * s, qk[..., rope:]], -1)
    pg, t = _slots(st, b.seq, L + b.at)
    _write(st, pg, t, qk[:, nq:].half(), x[:, nq + nkv:].half())
    return dict(q=qk[:, :nq].half().reshape(-1, nq * D), k=st["k"], v=st["v"])


def _drop(st, seqs, first):
    """Of sequences that `seqs` marks, the table's entries from `first` on given back."""
    at = torch.arange(st["table"].shape[1], device=first.device)
    gone = seqs[:, None] & (at >= first[:, None]) & (st["table"] >= 0)
    _refer(st, st["table"].long(), gone, -1)
    st["table"].masked_fill_(gone, -1)


def _refer(st, pages, which, step):
    st["refs"].scatter_add_(0, pages.clamp_min(0).reshape(-1), (which.int() * step).reshape(-1))


def _plain_branch(st):
    case, b = st["case"], _Rows(st)
    n, page = case["n"], case["page"]
    keep, src = st["keep"].long(), st["source"].long()
    # truncate: tokens past the length given, and the pages behind them, are given back
    lens = torch.where(keep >= 0, torch.minimum(keep, st["lens"].long()), st["lens"].long())
    _drop(st, keep >= 0, -(-lens // page))
    # fork: a branch gives back what it had, and shares its source's committed pages
    to = src >= 0
    _drop(st, to, torch.zeros_like(src))
    lens = torch.where(to, lens[src.clamp_min(0)], lens)
    at = torch.arange(st["table"].shape[1], device=src.device)
    shared = st["table"][src.clamp_min(0)].masked_fill(at >= -(-lens // page)[:, None], -1)
    st["table"].copy_(torch.where(to[:, None], shared, st["table"]))
    _refer(st, st["table"].long(), to[:, None] & (st["table"] >= 0), 1)
    st["lens"].copy_(lens)
    # reserve: blocks that rows go to and that have no page of their own take the lowest free ones, in
    # order; a sequence is served if its row has the entries and all before it and itself find room
    rows, old = b.count, st["table"].long()
    first, last = lens // page, (lens + rows - 1) // page
    fits = (rows > 0) & (last < at.numel())
    touched = fits[:, None] & (at >= first[:, None]) & (at <= last[:, None])
    refs = torch.where(old >= 0, st["refs"].long()[old.clamp_min(0)], torch.zeros_like(old))
    need = touched & (refs != 1)
    count = need.sum(1)
    free = st["refs"] == 0
    served = fits & ((count.cumsum(0) <= free.sum()) | (count == 0))
    need &= served[:, None]
    ids = torch.full((free.numel() + 1,), -1, dtype=torch.long, device=old.device)
    ids[torch.where(free, free.cumsum(0) - 1, free.numel())] = torch.arange(free.numel(), device=old.device)
    rank = (need.reshape(-1).cumsum(0) - 1).reshape(need.shape).clamp(0, free.numel())
    new = torch.where(need, ids[rank], old)
    held = need & (refs > 1)
    _refer(st, old, held, -1)
    _refer(st, new, need, 1)
    st["table"].copy_(new)
    # the block that rows and committed tokens share
    f = first.clamp_max(at.numel() - 1)[:, None]
    part = held.gather(1, f)[:, 0] & (lens % page > 0)
    here, there = old.gather(1, f)[:, 0], new.gather(1, f)[:, 0]
    res = torch.stack([served.long(), need.sum(1), torch.where(part, here, -1), torch.where(part, there, -1)], 1)
    st["reserved"].copy_(res)
    # tokens of the block that are committed, in whole groups of eight; the others hold nothing yet
    there, here = torch.where(part, there, 0), torch.where(part, here, 0)
    fill = (part[:, None] & (torch.arange(page, device=src.device) // 8 * 8 < (lens % page)[:, None]))
    i, t = torch.nonzero(fill, as_tuple=True)
    _write(st, there[i], t, *_read(st, here[i], t))
    return {x: st[x] for x in ("table", "lens", "refs", "reserved", "k", "v")}


def _plain_commit(st):
    b = _Rows(st)
    L, path = st["lens"].long()[b.seq], st["path"].long()
    kept = b.at <= st["accepted"].long()[b.seq]
    # rows that are not kept stay where they are
    pg, t = _slots(st, b.seq, L + torch.where(kept, path, b.at))
    pg2, t2 = _slots(st, b.seq, L + b.at)
    _write(st, pg2, t2, *_read(st, pg, t))
    new = st["lens"] + torch.where(b.count > 0, st["accepted"] + 1, 0).int()
    return dict(k=st["k"], v=st["v"], lens=new)


def _plain_accept(st):
    """In 64 bits throughout: a sampled token changes with the last bits of 150000 partial sums."""
    case, b = st["case"], _Rows(st)
    n, M, V = case["n"], case["M"], case["V"]
    x, tok, ids = st["logits"].double(), st["token"].long(), torch.arange(V, device="cuda")
    T = st["temperature"].double()[b.seq][:, None]
    m = x.amax(-1, keepdim=True)
    best = torch.where(x == m, ids, V).amin(-1, keepdim=True)
    e = torch.where(T > GREEDY, torch.exp((x - m) / T.clamp_min(GREEDY)), (ids == best).double())
    Z = e.sum(-1)
    # each row against its parent: the greatest row that it sees, below itself
    par = torch.where(b.sees & (b.local < b.at[:, None]), b.local, -1).amax(-1)
    above = b.row[b.seq, par.clamp_min(0)]
    ex = e[above, tok]
    # siblings, in order: by sequence, [n, M (row), M (a row before it)]
    par_n, tok_n = (torch.where(b.there, y[b.row], -1) for y in (par, tok))
    sib = (par_n[:, :, None] == par_n[:, None]) & (b.local[None, :] < b.local[:, None]) & (par_n[:, None] >= 0)
    again = (sib & (tok_n[:, :, None] == tok_n[:, None])).any(-1)[b.seq, b.at]
    ex = torch.where(again, torch.zeros_like(ex), ex)
    gone = torch.where(sib, ex[b.row][:, None], 0.0).sum(-1)[b.seq, b.at]
    q = st["q"].double()[above, tok] if case["q"] else torch.ones_like(ex)
    ok = (par >= 0) & (ex > 0) & (q > 0) & (st["u_accept"].double() * q * (Z[above] - gone) <= ex)
    ok_n = torch.where(b.there, ok[b.row], False)
    ok &= ~(sib & ok_n[:, None]).any(-1)[b.seq, b.at]
    # kept: rows whose whole way from row 0 passed
    ok_n = (torch.where(b.there, ok[b.row], False) | (b.local == 0))[b.seq]
    below = b.sees & (b.local <= b.at[:, None])
    kept = (~below | ok_n).all(-1)
    kept_n = torch.where(b.there, kept[b.row], False)
    accepted = kept_n.sum(-1) - 1
    path = torch.where(kept_n, b.local, M).sort(-1).values
    path = torch.where(path < M, path, -1)
    # the last kept row's own token: what its probabilities leave without the refused drafts
    end = torch.where(kept_n, b.local, 0).amax(-1)
    f = b.row[torch.arange(n, device="cuda"), end]
    child = (par_n == end[:, None]) & (par_n >= 0)
    r = e[f]
    if case["q"]:
        left = (r / Z[f][:, None] - st["q"].double()[f]).clamp_min(0)
        left = torch.where(child.any(-1)[:, None], left, r)
    else:
        left = r.clone()
        i, j = torch.nonzero(child, as_tuple=True)
        left[i, tok_n[i, j]] = 0.0
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, r)
    cum = left.cumsum(-1)
    over = cum > st["u_sample"].double()[:, None] * cum[:, -1:]
    last = torch.where(left > 0, ids, -1).amax(-1)
    token = torch.where(over.any(-1), torch.where(over, ids, V).amin(-1), last)
    return dict(accepted=accepted.int(), path=path[b.seq, b.at].int(), token=token.int())


# ------------------------------------------------------------------------------------- work
def work(case):
    kind, n = case["kind"], case["n"]
    lens, rows = _sizes(case)
    R, G = sum(rows), case.get("nq", 0) // case.get("nkv", 1)
    if kind == "accept":
        # every row's logits; of one row a sequence the draft model's distribution too
        return {"bytes": 4.0 * case["V"] * (R + (n if case["q"] else 0)), "flops": 8.0 * case["V"] * (R + n)}
    nkv, page = case["nkv"], case["page"]
    if kind == "append":
        return {"bytes": 4.0 * R * (case["nq"] + 2 * nkv) * D + 4 * D,
                "flops": 10.0 * R * (case["nq"] + nkv) * D}
    if kind == "attn":
        W = case["window"] or 1 << 40
        keys = sum(min(x, W - 1 + m - 1) + m for x, m in zip(lens, rows))
        pairs = sum(m * (min(x, W - 1) + (m + 1) // 2) for x, m in zip(lens, rows))
        return {"bytes": 4.0 * nkv * D * keys + 4.0 * R * case["nq"] * D, "flops": 4.0 * pairs * case["nq"] * D}
    token = 4.0 * nkv * D * case["layers"]  # bytes of a token's keys and values in all layers
    if kind == "commit":  # about half of the kept rows move
        return {"bytes": token * R / 4 + 8 * n, "flops": 1.0 * R}
    p = case["parents"]
    part = sum(-(-(lens[i] % page) // 8) * 8 * (-(-(n - p - i) // p) + case["go_on"]) for i in range(p))
    blocks = sum(-(-x // page) for x in lens)
    return {"bytes": 2 * token * part + 8.0 * blocks * n / p + 4.0 * blocks, "flops": 1.0 * n}


# -------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    d = _inputs(case, seed)
    return globals()["_exact_" + case["kind"]](case, d)


def _at(tokens):
    """Where a head's K and V of tokens [T] lie in a page, each [T, 128]."""
    u, t = tokens[:, None] // 32 * 4096, tokens[:, None] % 32
    i = torch.arange(D, device=tokens.device)
    return (u + 2048 * (t // 4 % 2) + 512 * (i // 32) + 128 * (i // 8 % 4) + 32 * (t // 8) + 8 * (t % 4) + i % 8,
            u + 512 * (i // 16) + 128 * (t // 8) + 8 * (i % 16) + t % 8)


def _flat(d):
    return (d[x].reshape(d[x].shape[:3] + (-1,)) for x in "kv")


def _move(src, dst, p, t, p2, t2):
    """K and V of tokens t of page p of flat pools to tokens t2 of page p2."""
    for a, b, i, j in zip(src, dst, _at(t), _at(t2)):
        b[:, p2, :, j] = a[:, p, :, i]


def _host(d, *names):
    return [d[x].cpu().tolist() for x in names]


def _exact_attn(case, d):
    nq, nkv, page, W = case["nq"], case["nkv"], case["page"], case["window"]
    G = nq // nkv
    start, lens, table = _host(d, "row_start", "lens", "table")
    K, V = _flat(d)
    out = torch.zeros((d["rows"], nq, D), dtype=torch.float64, device="cuda")
    q = d["q"].double().reshape(-1, nq, D)
    for s, L in enumerate(lens):
        m, par = start[s + 1] - start[s], d["parents"][s]
        pos = torch.arange(L + m, device="cuda")
        pg = torch.tensor(table[s], device="cuda")[pos // page]
        ik, iv = _at(pos % page)
        k, v = (x[0][pg[:, None], :, i].double().transpose(1, 2) for x, i in ((K, ik), (V, iv)))  # [T, nkv, D]
        for r in range(m):
            way, a = [], r
            while a >= 0:
                way.append(L + a)
                a = par[a]
            first = max(0, L + len(way) - W) if W else 0
            at = torch.tensor(sorted(way), device="cuda")
            keys, vals = (torch.cat([x[first:L], x[at]]) for x in (k, v))
            for g in range(nkv):
                sc = keys[:, g] @ q[start[s] + r, g * G:(g + 1) * G].T / math.sqrt(D)
                out[start[s] + r, g * G:(g + 1) * G] = torch.softmax(sc, 0).T @ vals[:, g]
    return dict(out=out.reshape(-1, nq * D))


def _exact_append(case, d):
    nq, nkv, rope, page = case["nq"], case["nkv"], case["rope"], case["page"]
    start, lens, table = _host(d, "row_start", "lens", "table")
    x = d["qkv"].double().reshape(-1, nq + 2 * nkv, D)
    pos, where = [], []
    for s, L in enumerate(lens):
        for r in range(start[s + 1] - start[s]):
            up, a = 0, d["parents"][s][r]
            while a >= 0:
                up, a = up + 1, d["parents"][s][a]
            pos.append(L + up)
            where.append((table[s][(L + r) // page], (L + r) % page))
    P = torch.tensor(pos, dtype=torch.float64, device="cuda")
    y = x.clone()
    for h in range(nq + nkv):
        z = x[:, h] / ((x[:, h] ** 2).sum(1, keepdim=True) / D + EPS).sqrt()
        z = z * d["qw" if h < nq else "kw"].double()
        y[:, h] = z
        for i in range(rope // 2):
            th = P * ROPE_BASE ** (-2.0 * i / rope)
            a, b = z[:, i], z[:, i + rope // 2]
            y[:, h, i] = a * th.cos() - b * th.sin()
            y[:, h, i + rope // 2] = a * th.sin() + b * th.cos()
    k, v = d["k"].double(), d["v"].double()
    K, V = _flat(dict(k=k, v=v))
    ik, iv = _at(torch.tensor([t for _, t in where], device="cuda"))
    for r, (pg, _) in enumerate(where):
        K[0, pg, :, ik[r]] = y[r, nq:nq + nkv]
        V[0, pg, :, iv[r]] = y[r, nq + nkv:]
    return dict(q=y[:, :nq].reshape(-1, nq * D), k=k, v=v)


def _exact_branch(case, d):
    page = case["page"]
    start, lens, table, refs, keep, src = _host(d, "row_start", "lens", "table", "refs", "keep", "source")
    n, width = len(lens), len(table[0])

    def drop(s, first):
        for j in range(first, width):
            if table[s][j] >= 0:
                refs[table[s][j]] -= 1
                table[s][j] = -1

    for s in range(n):
        if keep[s] >= 0:
            lens[s] = min(lens[s], keep[s])
            drop(s, -(-lens[s] // page))
    for s in range(n):
        if src[s] >= 0:
            drop(s, 0)
            lens[s] = lens[src[s]]
            for j in range(-(-lens[s] // page)):
                table[s][j] = table[src[s]][j]
                refs[table[s][j]] += 1
    before, free = list(refs), [p for p, c in enumerate(refs) if c == 0]
    total, out, k, v = 0, [], d["k"].clone(), d["v"].clone()
    pools, copies = list(_flat(d)), list(_flat(dict(k=k, v=v)))
    for s in range(n):
        m, L = start[s + 1] - start[s], lens[s]
        row = [0, 0, -1, -1]
        if m > 0 and (L + m - 1) // page < width:
            js = range(L // page, (L + m - 1) // page + 1)
            need = [j for j in js if table[s][j] < 0 or before[table[s][j]] != 1]
            total += len(need)
            if total <= len(free) or not need:
                row[:2] = 1, len(need)
                for i, j in enumerate(need):
                    p, o = free[total - len(need) + i], table[s][j]
                    table[s][j] = p
                    refs[p] += 1
                    if o >= 0 and before[o] > 1:
                        refs[o] -= 1
                        if j == L // page and L % page:
                            row[2:] = o, p
                            t = torch.arange(-(-(L % page) // 8) * 8, device="cuda")
                            _move(pools, copies, o, t, p, t)
        out.append(row)
    res = [torch.tensor(x) for x in (table, lens, refs, out)]
    return dict(zip(("table", "lens", "refs", "reserved"), res), k=k.double(), v=v.double())


def _exact_commit(case, d):
    page = case["page"]
    start, lens, table, accepted, path = _host(d, "row_start", "lens", "table", "accepted", "path")
    k, v, new = d["k"].clone(), d["v"].clone(), []
    pools = list(_flat(dict(k=k, v=v)))
    for s, L in enumerate(lens):
        for i in range(accepted[s] + 1):  # (a path goes upwards: nothing is read after it was written)
            a, b = L + path[start[s] + i], L + i
            pa, pb = table[s][a // page], table[s][b // page]
            a, b = (torch.tensor([x % page], device="cuda") for x in (a, b))
            _move(pools, pools, pa, a, pb, b)
        new.append(L + accepted[s] + 1)
    return dict(k=k.double(), v=v.double(), lens=torch.tensor(new))


def _exact_accept(case, d):
    start, tok, temp, ua, us = _host(d, "row_start", "token", "temperature", "u_accept", "u_sample")
    accepted, path, token = [], [], []
    for s, t in enumerate(temp):
        at, m, par = start[s], start[s + 1] - start[s], d["parents"][s]
        way = [0]
        while True:
            x = d["logits"][at + way[-1]].double()
            if t <= GREEDY:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
            else:
                p = torch.softmax(x / t, 0)
            r, mass, refused, go = p.clone(), 1.0, 0, None
            for c in range(way[-1] + 1, m):
                if par[c] != way[-1]:
                    continue
                y = tok[at + c]
                q = float(d["q"][at + way[-1], y]) if case["q"] else 1.0
                if float(r[y]) > 0 and q > 0 and ua[at + c] * q * mass <= float(r[y]):
                    go = c
                    break
                refused += 1
                if not case["q"]:
                    mass -= float(r[y])
                    r[y] = 0.0
            if go is None:
                break
            way.append(go)
        if case["q"] and refused:
            r = (p - d["q"][at + way[-1]].double()).clamp_min(0)
        if float(r.sum()) <= 0:
            r = p
        cum = torch.cumsum(r, 0)
        over = (cum > us[s] * cum[-1]).nonzero()
        token.append(int(over[0]) if len(over) else int((r > 0).nonzero()[-1]))
        accepted.append(len(way) - 1)
        path += way + [-1] * (m - len(way))
    return dict(accepted=torch.tensor(accepted), path=torch.tensor(path), token=torch.tensor(token))
