"""Timed calls of the key-value cache held in 8 bits: what fills it, reads it and thins it.

The context of a long prompt, two tiers: an fp16 ring takes the newest rows of K and V as a pass
appends them (queries and keys normed and rotated), and blocks of 64 tokens are sealed from it
into pages of 8-bit codes with one scale for each block and head.  Attention reads both, over all
sealed blocks or over those a cheap score selects for each row, and may add up the attention
weight that each block got, by which blocks are evicted.  Heads of 128; the head counts are those
of the benchmark model and of the tests (one to sixteen query heads a KV head), the rows those a
pass has: one (decode), 9 (a K = 8 chain), 17 (a 16-node tree), 64 (a prefill chunk).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

NQ, NKV, D, B = 16, 4, 128, 64
EPS, ROPE_BASE = 1e-6, 1e6

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
    heads = dict(nq=NQ, nkv=NKV)
    return [
        # queries and keys of one decode step far into a context; of a 64-row draft tree
        dict(name="append_decode", kind="append", **heads, M=1, L=131071, C=128, rope=64,
             tree=False),
        dict(name="append_tree", kind="append", **heads, M=64, L=60000, C=192, rope=128, tree=True),
        # the block that 64 decoded tokens filled; a whole prompt of 131072 tokens
        dict(name="seal_block", kind="seal", **heads, n=1, pos=5000, C=192),
        dict(name="seal_prompt", kind="seal", **heads, n=2048, pos=0, C=131072),
        # one decode step after 2000 tokens, and after 131000
        dict(name="attn_decode_short", kind="attn", **heads, M=1, n=30, open=80, tree=False,
             mass=False),
        dict(name="attn_decode_long", kind="attn", **heads, M=1, n=2047, open=63, tree=False,
             mass=False),
        # a 16-node draft tree at 32000 tokens, the blocks' weights added up
        dict(name="attn_tree_mass", kind="attn", **heads, M=17, n=500, open=17, tree=True,
             mass=True),
        # a prefill chunk at 65000 tokens
        dict(name="attn_prefill", kind="attn", **heads, M=64, n=1023, open=1, tree=False,
             mass=False),
        # one decode step reading 64 of 2047 blocks; a K = 8 chain reading 32 of 500
        dict(name="sparse_decode", kind="sparse", **heads, M=1, n=2047, n_sel=64, first=1, last=2,
             open=30, tree=False),
        dict(name="sparse_chain", kind="sparse", **heads, M=9, n=500, n_sel=32, first=1, last=2,
             open=50, tree=False),
        # the budget of a short context by one block; half of a long context's blocks
        dict(name="evict_one", kind="evict", **heads, n=65, keep=64, first=1, last=4),
        dict(name="evict_half", kind="evict", **heads, n=2047, keep=1024, first=1, last=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "seal", "seal", "attn", "attn", "attn", "sparse",
                       "sparse", "sparse", "evict", "evict"])
    nq, nkv = rng.choice([(16, 4), (16, 4), (16, 4), (8, 8), (16, 2), (32, 4), (12, 4), (16, 1)])
    heads = dict(nq=nq, nkv=nkv)
    if kind == "append":
        M = _log(rng, 1, 64)
        return dict(kind=kind, **heads, M=M, L=_log(rng, 1, 131072), C=M + rng.randint(0, 200),
                    rope=rng.choice([0, 32, 64, 64, 128]), tree=rng.random() < 0.4)
    if kind == "seal":
        n = _log(rng, 1, 2048 * NKV // max(nkv, NKV))
        return dict(kind=kind, **heads, n=n, pos=_log(rng, 1, 100000),
                    C=n * B + rng.randint(0, 200))
    if kind == "evict":
        n = _log(rng, 8, 4096)
        first, last = rng.randint(0, 2), rng.randint(0, 4)
        return dict(kind=kind, **heads, n=n, keep=rng.randint(first + last, n), first=first,
                    last=last)
    if kind == "attn":
        M = _log(rng, 1, 64)
        n = _log(rng, 1, min(2047, 1023 * 64 * NQ // (M * nq), 2047 * NKV // nkv))
        return dict(kind=kind, **heads, M=M, n=n, open=rng.randint(0, 150),
                    tree=rng.random() < 0.4, mass=rng.random() < 0.4)
    M = _log(rng, 1, 17)
    n = _log(rng, 8, 2047 * NKV // max(nkv, NKV))
    first, last = rng.randint(0, 2), rng.randint(0, 3)
    return dict(kind=kind, **heads, M=M, n=n, n_sel=_log(rng, first + last + 1, min(n, 64)),
                first=first, last=last, open=rng.randint(0, 150), tree=rng.random() < 0.4)


# ----------------------------------------------------------------------------------- inputs
def _tree(rng, M, tree):
    """A chain, or a tree of which every node hangs off one of the six rows before it."""
    if not tree:
        return None
    return [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, M)]


def _rows(parents, M):
    """Depth of each row, and which of the pass's rows it attends: its ancestors and itself."""
    depth, sees = [0] * M, np.eye(M, dtype=bool)
    for r in range(1, M):
        p = r - 1 if parents is None else parents[r]
        depth[r] = depth[p] + 1
        sees[r] |= sees[p]
    return depth, sees


def _inputs(case, seed):
    """Everything the call reads, from the seed alone (also what exact() starts from).

    Keys have a component that drifts from one stretch of 192 tokens to the next and channels of
    their own size, as the keys of a text have; the queries of a pass resemble each other and lean
    to a few of those stretches."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, nq, nkv = case["kind"], case["nq"], case["nkv"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if kind == "evict":
        n = case["n"]
        mass = torch.rand((nkv, n), generator=gen, device="cuda").pow(6) * 20.0
        mass[:, :: 7] = 0.0  # blocks that no row has looked at: ties
        table = torch.stack([torch.randperm(n, generator=gen, device="cuda") + g * n
                             for g in range(nkv)]).to(torch.int32)
        return dict(mass=mass, table=table)
    if kind == "append":
        M, C = case["M"], case["C"]
        return dict(qkv=(randn(M, (nq + 2 * nkv) * D) * 1.5).half(),
                    qw=(1.0 + 0.1 * randn(D)).half(), kw=(1.0 + 0.1 * randn(D)).half(),
                    ring=[randn(nkv, C, D).half() for _ in range(2)],
                    parents=_tree(rng, M, case["tree"]))
    n = case["n"]
    if kind == "seal":
        T, C = n * B, case["C"]
    else:
        T, C = n * B, case["open"] + case["M"]
    size = torch.exp(0.4 * randn(nkv, 1, D))
    topics = randn(nkv, (T + C) // 192 + 1, D)

    def keys(t0, count):
        at = torch.arange(t0, t0 + count, device="cuda") // 192
        return ((0.6 * topics[:, at] + 0.8 * randn(nkv, count, D)) * size).half()

    d = {}
    if kind == "seal":
        d["ring"] = [keys(0, C), randn(nkv, C, D).half()]
        return d
    M = case["M"]
    d["k"], d["v"] = keys(0, T), (randn(nkv, T, D) * torch.exp(0.3 * randn(nkv, 1, D))).half()
    d["ring"] = [keys(T, C), randn(nkv, C, D).half()]
    G = nq // nkv
    near = topics[:, torch.randint(0, topics.shape[1], (3,), generator=gen, device="cuda")].sum(1)
    q = (0.7 * near[None, :, None] + randn(1, nkv, G, D) + 0.5 * randn(M, nkv, G, D)) / size[None]
    d["q"] = q.reshape(M, nq * D).half()
    d["parents"] = _tree(rng, M, case["tree"])
    # where the pages lie in the pool: anywhere, as after some evictions
    d["table"] = torch.stack([torch.randperm(n, generator=gen, device="cuda") + g * n
                              for g in range(nkv)]).to(torch.int32)
    if kind == "attn" and case["mass"]:
        d["mass"] = torch.rand((nkv, n), generator=gen, device="cuda")
    return d


def _ratio(a, b):
    """a / b in the inputs' own precision (a quotient by a plain number may become a product)."""
    return a / torch.full_like(a, b)


def _quantise(x):
    """Codes (whole numbers) and scales of blocks [..., 64, 128]: the scale is the block's greatest
    magnitude over 127, a code the nearest whole number to x (127 / greatest)."""
    a = x.float().abs().amax((-2, -1))
    s = _ratio(a, 127.0)
    r = torch.where(a > 0, torch.full_like(a, 127.0) / a, torch.zeros_like(a))
    return (x.float() * r[..., None, None]).round().clamp(-127, 127), s


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    kind, nq, nkv = case["kind"], case["nq"], case["nkv"]
    if own:
        from momij_amd.kv8 import Kv8Cache, KvRing

        st["ctx"] = ctx = context()

    def out(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    if kind == "append":
        if own:
            st["kvring"] = KvRing(*st["ring"])
            st["cfg"] = dict(H=2048, nQ=nq, nKV=nkv, D=D, rope_dim=case["rope"],
                             rope_base=ROPE_BASE, eps=EPS, window=0, C=case["C"], gs=64)
            st["q"] = out(case["M"], nq * D)
        return st
    n = case["n"]
    if kind == "seal":
        if own:
            st["cache"] = Kv8Cache(ctx, nkv, n)
            st["kvring"] = KvRing(*st["ring"])
            st["back"] = KvRing(out(nkv, n * B, D), out(nkv, n * B, D))
        return st
    if kind == "evict":
        if own:
            st["cache"] = Kv8Cache(ctx, nkv, n)
            st["cache"].table.copy_(st["table"])
            st["new_table"], st["new_mass"] = torch.empty_like(st["table"]), torch.empty_like(st["mass"])
        return st
    M = case["M"]
    if own:
        st["cache"] = cache = Kv8Cache(ctx, nkv, n)
        cache.table.copy_(st["table"])
        ctx.kv8_seal(cache, KvRing(st.pop("k"), st.pop("v")), 0, n, 0)
        st["kvring"] = KvRing(*st["ring"])
        st["out"] = out(M, nq * D)
        if kind == "sparse":
            st["sel"] = out(M, nkv, case["n_sel"], dtype=torch.int32)
        elif case["mass"]:
            st["new_mass"] = torch.empty_like(st["mass"])
        ctx.sync()
        return st
    for x in "kv":
        st[x + "c"], st[x + "s"] = _quantise(st.pop(x).reshape(nkv, n, B, D))
        st[x + "c"] = st[x + "c"].to(torch.int8)
    # the greatest and the least code of each dim in each block
    st["hi"], st["lo"] = st["kc"].amax(2), st["kc"].amin(2)
    st["sees"] = torch.from_numpy(_rows(st["parents"], M)[1]).cuda()
    return st


# -------------------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if "ctx" in st else _run_plain(st)


def _run_own(st):
    case, ctx = st["case"], st["ctx"]
    kind = case["kind"]
    if kind == "append":
        ctx.qkv_append(st["cfg"], st["qkv"], st["qw"], st["kw"], st["kvring"], case["L"],
                       st["parents"], case["M"], st["q"])
        return dict(q=st["q"], k=st["ring"][0], v=st["ring"][1])
    n, cache = case["n"], st["cache"]
    if kind == "seal":
        # the values come back the way they do for a rewind into sealed blocks
        ctx.kv8_seal(cache, st["kvring"], case["pos"], n, 0)
        ctx.kv8_unseal(cache, 0, n, st["back"], 0)
        return dict(k=st["back"].k, v=st["back"].v, ks=cache.k_scale, vs=cache.v_scale,
                    bounds=cache.k_bounds)
    if kind == "evict":
        ctx.kv8_evict(cache, n, case["keep"], case["first"], case["last"], st["mass"],
                      st["new_table"], st["new_mass"])
        return dict(table=st["new_table"], mass=st["new_mass"])
    start = n * B
    L = start + case["open"]
    if kind == "sparse":
        ctx.kv8_select(cache, st["q"], case["M"], case["nq"], n, case["n_sel"], case["first"],
                       case["last"], st["sel"])
        ctx.kv8_attn(cache, st["kvring"], st["q"], case["M"], case["nq"], n, start, L,
                     st["parents"], st["out"], sel=st["sel"])
        return dict(out=st["out"], sel=st["sel"])
    ctx.kv8_attn(cache, st["kvring"], st["q"], case["M"], case["nq"], n, start, L, st["parents"],
                 st["out"], mass_in=st.get("mass"), mass_out=st.get("new_mass"))
    return dict(out=st["out"], mass=st["new_mass"]) if case["mass"] else dict(out=st["out"])


def _norm_rope(x, w, pos, rope):
    """Per-head RMS norm, then the rotation of dims (i, i + rope / 2) at the rows' positions; the
    angles in 64 bits."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    if rope == 0:
        return x
    half = rope // 2
    f = ROPE_BASE ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    th = pos.double()[:, None, None] * f
    c, s = th.cos().float(), th.sin().float()
    a, b = x[..., :half], x[..., half:rope]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rope:]], -1)


def _ring_slots(C, n_rows, first):
    return (first + torch.arange(n_rows, device="cuda")) % C


def _softmax_av(q, k, v, ok):
    """softmax(q k^T / sqrt(128)) v over the keys that ok allows; rows without any give zeros.
    q [.., R, D], k, v [.., T, D], ok broadcast to [.., R, T]; also the weights."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * D ** -0.5
    s = s.masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return torch.matmul(p, v), p


def _run_plain(st):
    case = st["case"]
    kind, nq, nkv = case["kind"], case["nq"], case["nkv"]
    G = nq // nkv
    if kind == "append":
        M, L = case["M"], case["L"]
        x = st["qkv"].float().reshape(M, nq + 2 * nkv, D)
        pos = L + torch.tensor(_rows(st["parents"], M)[0], device="cuda")
        q = _norm_rope(x[:, :nq], st["qw"], pos, case["rope"]).half().reshape(M, nq * D)
        k = _norm_rope(x[:, nq:nq + nkv], st["kw"], pos, case["rope"]).half()
        K, V = (t.clone() for t in st["ring"])
        slots = _ring_slots(case["C"], M, L)
        K[:, slots] = k.transpose(0, 1)
        V[:, slots] = x[:, nq + nkv:].half().transpose(0, 1)
        return dict(q=q, k=K, v=V)
    n = case["n"]
    if kind == "seal":
        slots = _ring_slots(case["C"], n * B, case["pos"])
        res = {}
        for x, ring in zip("kv", st["ring"]):
            c, s = _quantise(ring[:, slots].reshape(nkv, n, B, D))
            res[x] = (c * s[..., None, None]).half().reshape(nkv, n * B, D)
            res[x + "s"] = s.reshape(-1)
            if x == "k":
                res["bounds"] = torch.stack([c.amax(2), c.amin(2)], 2).to(torch.int8)
        res["bounds"] = res["bounds"].reshape(nkv * n, 2, D)
        return res
    if kind == "evict":
        keep, first, last = case["keep"], case["first"], case["last"]
        rank = st["mass"].clone()
        rank[:, :first] = math.inf
        rank[:, n - last:] = math.inf
        order = rank.sort(dim=1, descending=True, stable=True).indices  # ties: the lowest index
        order = torch.cat([order[:, :keep].sort(1).values, order[:, keep:].sort(1).values], 1)
        mass = st["mass"].gather(1, order)
        mass[:, keep:] = 0.0
        return dict(table=st["table"].gather(1, order), mass=mass)
    M, op = case["M"], case["open"]
    q = st["q"].float().reshape(M, nkv, G, D)
    slots = _ring_slots(op + M, op + M, n * B)
    rk, rv = (t[:, slots].float() for t in st["ring"])
    sees = torch.cat([torch.ones((M, op), dtype=torch.bool, device="cuda"), st["sees"]], 1)
    if kind == "sparse":
        sel = _select(case, q, st["hi"].float(), st["lo"].float(), st["ks"])
        at = sel.transpose(0, 1).long()  # [nkv, M, n_sel]
        g = torch.arange(nkv, device="cuda")[:, None, None]
        k, v = ((st[x + "c"][g, at].float() * st[x + "s"][g, at][..., None, None])
                .reshape(nkv, M, -1, D) for x in "kv")
        k = torch.cat([k, rk[:, None].expand(-1, M, -1, -1)], 2)
        v = torch.cat([v, rv[:, None].expand(-1, M, -1, -1)], 2)
        ok = torch.cat([torch.ones((M, at.shape[2] * B), dtype=torch.bool, device="cuda"), sees], 1)
        o, _ = _softmax_av(q.transpose(0, 1).contiguous(), k, v, ok[None, :, None])
        return dict(out=o.transpose(0, 1).reshape(M, nq * D).half(), sel=sel)
    k, v = ((st[x + "c"].float() * st[x + "s"][..., None, None]).reshape(nkv, n * B, D)
            for x in "kv")
    k, v = torch.cat([k, rk], 1), torch.cat([v, rv], 1)
    ok = torch.cat([torch.ones((M, n * B), dtype=torch.bool, device="cuda"), sees], 1)
    qg = q.transpose(0, 1).reshape(nkv, M * G, D)
    o, p = _softmax_av(qg, k, v, ok.repeat_interleave(G, 0)[None])
    res = dict(out=o.reshape(nkv, M, G, D).transpose(0, 1).reshape(M, nq * D).half())
    if case["mass"]:
        res["mass"] = st["mass"] + p[:, :, :n * B].sum(1).reshape(nkv, n, B).sum(-1)
    return res


def _select(case, q, hi, lo, ks):
    """Blocks each row reads, [M, nkv, n_sel] ascending: the first and last ones, and those of the
    greatest score among the others.  The score bounds q k over a block from the greatest and the
    least code of each dim: the query's own 8-bit codes against whichever is the larger product
    (whole numbers), times the block's scale and then the query's; the largest over the heads of
    the group."""
    n, first, last, n_sel = case["n"], case["first"], case["last"], case["n_sel"]
    a = q.abs().amax(-1, keepdim=True)
    r = torch.where(a > 0, torch.full_like(a, 127.0) / a, torch.zeros_like(a))
    c = (q * r).round().clamp(-127, 127)  # [M, nkv, G, D]
    c = c.permute(1, 0, 2, 3)
    M, G = q.shape[0], q.shape[2]
    up, dn = (t.reshape(t.shape[0], M * G, D) for t in (c.clamp_min(0), c.clamp_max(0)))
    u = (torch.matmul(up, hi.transpose(1, 2).contiguous()) +
         torch.matmul(dn, lo.transpose(1, 2).contiguous()))
    sq = _ratio(a, 127.0).permute(1, 0, 2, 3).reshape(-1, M * G, 1)
    score = (u * ks[:, None] * sq).reshape(-1, M, G, n).amax(2).transpose(0, 1)
    score = score.clone()
    score[..., :first] = math.inf
    score[..., n - last:] = math.inf
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :n_sel]
    return order.sort(-1).values.to(torch.int32)


# ------------------------------------------------------------------------------------- work
def work(case):
    kind, nq, nkv = case["kind"], case["nq"], case["nkv"]
    G = nq // nkv
    if kind == "append":
        M = case["M"]
        return {"bytes": 4.0 * M * (nq + 2 * nkv) * D + 4 * D, "flops": 10.0 * M * (nq + nkv) * D}
    n = case["n"]
    if kind == "seal":
        e = 2.0 * nkv * n * B * D  # elements of K and V
        return {"bytes": 2 * e + e + nkv * n * (2 * D + 8) + 2 * e, "flops": 5.0 * e}
    if kind == "evict":
        return {"bytes": 16.0 * nkv * n, "flops": 4.0 * nkv * n}
    M, op = case["M"], case["open"]
    page = 2.0 * B * D + 8
    b = 4.0 * M * nq * D + 4.0 * nkv * (op + M) * D  # queries, outputs, ring rows
    if kind == "sparse":
        # every block's bounds; at the least the blocks of one row, where all rows choose the same
        return {"bytes": b + nkv * n * (2 * D + 4) + nkv * case["n_sel"] * page +
                4.0 * M * nkv * case["n_sel"],
                "flops": 4.0 * M * nq * D * (n + case["n_sel"] * B + op + M)}
    if case["mass"]:
        b += 8.0 * nkv * n
    return {"bytes": b + nkv * n * page, "flops": 4.0 * M * nq * D * (n * B + op + M)}


# -------------------------------------------------------------------- the same in 64 bits
def _codes64(x, dims):
    """8-bit codes and scale over `dims`: scale = greatest / 127 and code = x (127 / greatest), each
    formed in 64 bits and held in 32, the code then rounded to the nearest whole number."""
    x = x.double()
    top = x.abs().amax(dims, keepdim=True)
    scale = (top / torch.full_like(top, 127.0)).float()
    back = torch.where(top > 0, 127.0 / top, torch.zeros_like(top)).float()
    return (x * back.double()).float().round().clamp(-127, 127).double(), scale


def exact(case, seed):
    d = _inputs(case, seed)
    kind, nq, nkv = case["kind"], case["nq"], case["nkv"]
    G = nq // nkv
    if kind == "append":
        M, L, rope, C = case["M"], case["L"], case["rope"], case["C"]
        depth, par = [0] * M, d["parents"]
        for r in range(1, M):
            depth[r] = depth[par[r] if par else r - 1] + 1
        rows = d["qkv"].double().reshape(M, -1, D)
        res = dict(k=d["ring"][0].double(), v=d["ring"][1].double())
        outs = []
        for h in range(nq + nkv):
            w = d["qw" if h < nq else "kw"].double()
            x = rows[:, h]
            x = x / ((x ** 2).sum(1, keepdim=True) / D + EPS).sqrt() * w
            y = x.clone()
            for i in range(rope // 2):
                th = torch.tensor([(L + t) * ROPE_BASE ** (-2.0 * i / rope) for t in depth],
                                  dtype=torch.float64, device="cuda")
                a, b = x[:, i], x[:, i + rope // 2]
                y[:, i] = a * th.cos() - b * th.sin()
                y[:, i + rope // 2] = a * th.sin() + b * th.cos()
            outs.append(y)
        for r in range(M):
            for g in range(nkv):
                res["k"][g, (L + r) % C] = outs[nq + g][r]
                res["v"][g, (L + r) % C] = rows[r, nq + nkv + g]
        return dict(q=torch.stack(outs[:nq], 1).reshape(M, nq * D), **res)
    n = case["n"]
    if kind == "seal":
        at = (case["pos"] + torch.arange(n * B, device="cuda")).remainder(case["C"])
        res = {}
        for x, ring in zip("kv", d["ring"]):
            c, s = _codes64(ring[:, at].reshape(nkv * n, B, D), (1, 2))
            res[x] = (c * s.double()).reshape(nkv, n * B, D)
            res[x + "s"] = s.double().reshape(-1)
            if x == "k":
                res["bounds"] = torch.stack([c.max(1).values, c.min(1).values], 1).to(torch.int8)
        return res
    if kind == "evict":
        mass, table = d["mass"].cpu().numpy(), d["table"].cpu().numpy()
        new_t, new_m = np.empty_like(table), np.zeros(mass.shape)
        for g in range(nkv):
            held = set(range(case["first"])) | set(range(n - case["last"], n))
            for i in sorted(range(n), key=lambda i: (-float(mass[g, i]), i)):
                if len(held) < case["keep"]:
                    held.add(i)
            kept = sorted(held)
            gone = [i for i in range(n) if i not in held]
            new_t[g] = table[g, kept + gone]
            new_m[g, :len(kept)] = mass[g, kept]
        return dict(table=torch.from_numpy(new_t), mass=torch.from_numpy(new_m))
    M, op = case["M"], case["open"]
    C = op + M
    q = d["q"].double().reshape(M, nkv, G, D)
    par = d["parents"]
    anc = [[0]]
    for r in range(1, M):
        anc.append(anc[par[r] if par else r - 1] + [r])
    at = (n * B + torch.arange(C, device="cuda")).remainder(C)
    out = torch.empty((M, nkv, G, D), dtype=torch.float64, device="cuda")
    sel = torch.empty((M, nkv, case.get("n_sel", 0)), dtype=torch.int32)
    mass = d["mass"].double() if case.get("mass") else None
    for g in range(nkv):
        codes, ks = _codes64(d["k"][g].reshape(n, B, D), (1, 2))
        vcodes, vs = _codes64(d["v"][g].reshape(n, B, D), (1, 2))
        K, V = codes * ks.double(), vcodes * vs.double()
        rk, rv = d["ring"][0][g, at].double(), d["ring"][1][g, at].double()
        if kind == "sparse":
            qc, sq = _codes64(q[:, g], (2,))  # [M, G, D], [M, G, 1]
            hi, lo = codes.max(1).values, codes.min(1).values
            for r in range(M):
                u = torch.maximum(qc[r][:, None] * hi, qc[r][:, None] * lo).sum(-1)  # [G, n]
                sc = (u * ks.double().reshape(1, n)).float()  # the score is held in 32 bits
                sc = (sc.double() * sq[r].double()).float().max(0).values.cpu().tolist()
                held = set(range(case["first"])) | set(range(n - case["last"], n))
                for i in sorted(range(n), key=lambda i: (-sc[i], i)):
                    if len(held) < case["n_sel"]:
                        held.add(i)
                held = sorted(held)
                sel[r, g] = torch.tensor(held)
                own_rows = torch.tensor(list(range(op)) + [op + a for a in anc[r]], device="cuda")
                keys = torch.cat([K[held].reshape(-1, D), rk[own_rows]])
                vals = torch.cat([V[held].reshape(-1, D), rv[own_rows]])
                out[r, g] = torch.softmax(q[r, g] @ keys.T / math.sqrt(D), -1) @ vals
            continue
        K, V = K.reshape(-1, D), V.reshape(-1, D)
        for r in range(M):
            own_rows = torch.tensor(list(range(op)) + [op + a for a in anc[r]], device="cuda")
            s = torch.cat([q[r, g] @ K.T, q[r, g] @ rk[own_rows].T], 1) / math.sqrt(D)
            p = torch.softmax(s, -1)
            out[r, g] = p[:, :n * B] @ V + p[:, n * B:] @ rv[own_rows]
            if mass is not None:
                mass[g] += p[:, :n * B].sum(0).reshape(n, B).sum(1)
    res = dict(out=out.reshape(M, nq * D))
    if kind == "sparse":
        res["sel"] = sel
    elif mass is not None:
        res["mass"] = mass
    return res
