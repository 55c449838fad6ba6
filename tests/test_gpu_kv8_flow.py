"""GPU: the 8-bit KV cache in use: the attention block over it, a generation that appends, attends,
commits, seals, chooses, evicts and rewinds, captured calls, refusals while capturing, the abort
word, two contexts at once, a model's own caches, and pools past 4 GiB."""
import math

import numpy as np
import pytest

from momij_amd import synth
from tests import kv8_ref as ref
from tests import restate64 as r64
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu
D, B = 128, 64


@pytest.fixture(scope="module")
def ctx():
    from momij_amd.ops import Context

    c = Context(0)
    yield c
    c.close()


def cfg_of(nQ=16, nKV=4, H=2048, rope=64, gs=64):
    return dict(H=H, nQ=nQ, nKV=nKV, D=D, rope_dim=rope, rope_base=1e6, eps=1e-6, window=0, C=0, gs=gs)


def attend(q, k, v, ok, G):
    """kv8_ref.attention of rows q [M, G * 128] of one head's group."""
    M = q.shape[0]
    return ref.attention(q.double().reshape(M * G, D), k, v, ok.repeat_interleave(G, 0))


# -------------------------------------------------------------------------------- the block
def block64(cfg, aw, h, ks, vs, kr, vr, L, parents, pick):
    """The block at 64 bits, fp16 where it stores fp16: sealed keys ks, vs [nKV][n * 64][128], open ring
    rows kr, vr [nKV][R][128]; pick(q [M][nQ][128]) -> [nKV][M][n] the blocks each row reads.  Also
    the rows' weights a block [nKV][M][G][n], and a bound of a weight's relative error when every
    stored query and key value is a step off."""
    nQ, nKV = cfg["nQ"], cfg["nKV"]
    M, G, n = h.shape[0], nQ // nKV, ks.shape[1] // B
    h = np.asarray(h, np.float64)
    par, depth, anc = r64.tree_of(parents if parents is not None else list(range(-1, M - 1)), M)
    x = r64.rms(h, aw["norm_w"], cfg["eps"])
    qkv = r64.f16(x @ synth.dequant(aw["qkv_w"], aw["qkv_s"], aw["qkv_b"], cfg["gs"]).T)
    heads = qkv.reshape(M, nQ + 2 * nKV, D)

    def turn(lo, hi, w):
        return np.stack([r64.rope_heads(heads[r, lo:hi], aw[w], L + depth[r], cfg["rope_dim"],
                                        cfg["rope_base"], cfg["eps"]) for r in range(M)])

    q, kn, vn = turn(0, nQ, "q_norm_w"), turn(nQ, nQ + nKV, "k_norm_w"), heads[:, nQ + nKV:]
    seen = pick(q)
    o, w, es = np.zeros((M, nQ, D)), np.zeros((nKV, M, G, n)), 0.0
    for g in range(nKV):
        k = np.concatenate([ks[g], kr[g], kn[:, g]])
        v = np.concatenate([vs[g], vr[g], vn[:, g]])
        for r in range(M):
            ok = np.concatenate([np.repeat(seen[g, r], B), np.ones(kr.shape[1], bool), anc[r].astype(bool)])
            s = q[r, g * G:(g + 1) * G] @ k.T / math.sqrt(D)
            es = max(es, float((np.abs(q[r, g * G:(g + 1) * G]) @ np.abs(k[ok]).T).max() / math.sqrt(D)))
            s[:, ~ok] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            o[r, g * G:(g + 1) * G] = p @ v
            w[g, r] = p[:, :n * B].reshape(G, n, B).sum(2)
    proj = r64.f16(r64.f16(o.reshape(M, -1)) @ synth.dequant(aw["o_w"], aw["o_s"], aw["o_b"], cfg["gs"]).T)
    return r64.f16(h + proj), proj, kn, vn, w, 4 * es * 2.0 ** -10


@pytest.mark.parametrize("M,nQ,nKV,n,open_,n_sel,tree,mass,H,gs", [
    (1, 16, 4, 20, 30, 0, False, False, 2048, 64), (9, 16, 4, 20, 65, 0, False, True, 2048, 64),
    (17, 32, 4, 5, 3, 0, True, True, 4096, 128), (64, 16, 2, 12, 130, 0, True, False, 2048, 64),
    (1, 16, 4, 20, 30, 6, False, False, 2048, 128), (9, 16, 4, 20, 0, 7, True, False, 2048, 64),
    (5, 16, 4, 6, 9, 6, True, False, 2048, 64), (3, 8, 4, 0, 0, 4, False, False, 2048, 64),
    (2, 4, 1, 0, 70, 0, False, True, 2048, 64)])
def test_block(ctx, M, nQ, nKV, n, open_, n_sel, tree, mass, H, gs):
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    rng = np.random.default_rng(1000 * M + n + n_sel)
    cfg = cfg_of(nQ, nKV, H, gs=gs)
    aw = synth.attn_weights(rng, H, nQ, nKV, D, gs)
    h = synth.normal_f16(rng, (M, H))
    start, cap = n * B, open_ + M + 2
    L = start + open_
    parents = ref.tree(M, rng) if tree else None
    # blocks of different sizes: which ones a row takes is not a matter of roundings
    size = 0.02 * 1.25 ** np.stack([rng.permutation(max(n, 1)) for _ in range(nKV)])
    kk = (rng.standard_normal((nKV, max(n, 1), B, D)) * size[..., None, None]).astype(np.float16)
    vv = rng.standard_normal((nKV, max(n, 1), B, D)).astype(np.float16)
    rk, rv = (synth.normal_f16(rng, (nKV, cap, D)) for _ in range(2))
    cache = Kv8Cache(ctx, nKV, n + 1)
    cache.table.copy_(torch.from_numpy(rng.permutation(nKV * (n + 1)).astype(np.int32)).reshape(nKV, -1))
    flat = [dev(t.reshape(nKV, -1, D)) for t in (kk, vv)]
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(*flat), 0, n, 0)
    kc, ksc = ref.seal(torch.from_numpy(kk[:, :n]))
    vc, vsc = ref.seal(torch.from_numpy(vv[:, :n]))
    ks, vs = ((c * s.double()[..., None, None]).reshape(nKV, n * B, D).numpy()
              for c, s in ((kc, ksc), (vc, vsc)))
    slots = [(start + i) % cap for i in range(open_ + M)]
    G, first, last = nQ // nKV, min(1, n_sel), min(2, max(n_sel - 1, 0))

    def pick(q):
        seen = np.ones((nKV, M, n), bool)
        if n_sel == 0 or n_sel >= n:
            return seen
        sc = ref.scores(torch.from_numpy(q).half().reshape(M, nKV, G, D), kc.amax(2), kc.amin(2), ksc)
        for g in range(nKV):
            for r in range(M):
                at = ref.choose(sc[r, g].tolist(), first, last, n_sel)
                seen[g, r] = False
                seen[g, r, at] = True
                # a query value one step off moves a score by far less than 1%
                free = range(first, n - last)
                low = min(float(sc[r, g, i]) for i in free if i in at)
                high = max(float(sc[r, g, i]) for i in free if i not in at)
                assert low > high + 0.01 * abs(high), "the test's own blocks are too close"
        return seen

    want, proj, kn, vn, w, rel = block64(cfg, aw, h, ks, vs, rk[:, slots[:open_]].astype(np.float64),
                                         rv[:, slots[:open_]].astype(np.float64), L, parents, pick)
    daw = {k: dev(v) for k, v in aw.items()}
    m0 = torch.rand((nKV, n + 1), device="cuda") if mass else None
    bits = []
    for _ in range(2):  # a call repeats bit for bit
        dk, dv, dh = dev(rk), dev(rv), dev(h)
        m1 = torch.full_like(m0, -2.0) if mass else None
        torch.cuda.synchronize()
        ctx.attn_block_kv8(cfg, daw, cache, KvRing(dk, dv), dh, n, start, L, parents, M, n_sel, first, last,
                           m0, m1)
        ctx.sync()
        bits.append([host(t).tobytes() for t in (dh, dk, dv) + ((m1,) if mass else ())])
    assert bits[0] == bits[1]
    # six stored fp16 stages, each at most a step from its 64-bit statement's; the sum's own step
    got = host(dh).astype(np.float64)
    err = np.linalg.norm(got - want, axis=1)
    tol = 6 * 2.0 ** -10 * np.linalg.norm(proj, axis=1) + 2.0 ** -10 * np.linalg.norm(want, axis=1)
    assert (err <= tol).all(), (err / tol).max()
    for t, new, old in ((dk, kn, rk), (dv, vn, rv)):
        x = host(t).astype(np.float64)
        e = np.linalg.norm(x[:, slots[open_:]] - new.transpose(1, 0, 2), axis=2)
        assert (e <= 3 * 2.0 ** -10 * np.linalg.norm(new.transpose(1, 0, 2), axis=2)).all()
        rest = [s for s in range(cap) if s not in slots[open_:]]
        assert (host(t)[:, rest].view(np.uint16) == old[:, rest].view(np.uint16)).all()
    if mass:
        add = w.sum((1, 2))
        m = host(m1)
        tol = add * (rel + 2.0 ** -10) + (host(m0)[:, :n] + add) * (M * G + 4) * 2.0 ** -24
        assert (np.abs(m[:, :n] - host(m0)[:, :n] - add) <= tol).all()
        assert (m[:, n:] == -2.0).all()


def test_block_without_pages_is_the_fp16_block(ctx):
    """Everything still in the ring: the block over the fp16 cache computes the same."""
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    rng = np.random.default_rng(77)
    cfg = dict(cfg_of(), C=320)
    aw = {k: dev(v) for k, v in synth.attn_weights(rng, 2048, 16, 4, D, 64).items()}
    parents = ref.tree(9, rng)
    h = synth.normal_f16(rng, (9, 2048))
    kc, vc = (synth.normal_f16(rng, (4, 320, D)) for _ in range(2))
    outs = []
    for eight in (False, True):
        dh, dk, dv = dev(h), dev(kc), dev(vc)
        torch.cuda.synchronize()
        if eight:
            ctx.attn_block_kv8(cfg, aw, Kv8Cache(ctx, 4, 1), KvRing(dk, dv), dh, 0, 0, 300, parents, 9)
        else:
            ctx.attn_block(cfg, aw, dh, dk, dv, 300, parents, 9)
        ctx.sync()
        outs.append([host(t).astype(np.float64) for t in (dh, dk, dv)])
    assert (outs[0][2] == outs[1][2]).all()
    for a, b in zip(*outs):  # the angles are formed at 32 and at 64 bits: a step here and there
        assert np.linalg.norm(a - b) <= 4 * 2.0 ** -10 * np.linalg.norm(b)


# ---------------------------------------------------------------------------- a generation
class Shadow:
    """What the cache should hold, at 64 bits: each head's blocks and the pages they lie in."""

    def __init__(self, cache):
        self.pages = cache.table.tolist()
        self.blocks = [[] for _ in range(cache.n_kv_heads)]  # (K [64, 128], V)

    def keys(self, g, ring, slots, at=None):
        import torch

        bl = self.blocks[g] if at is None else [self.blocks[g][i] for i in at]
        return [torch.cat([b[x] for b in bl] + [t[g, slots].double()]) for x, t in enumerate(ring)]


def test_generation(ctx):
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    nQ, nKV, cap, blocks = 16, 4, 64 + 48 + 64, 14
    G, cfg, rng = nQ // nKV, cfg_of(), np.random.default_rng(2)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda")

    with torch.cuda.stream(ctx.stream):
        cache = Kv8Cache(ctx, nKV, blocks)
        kv = [torch.full((nKV, cap, D), math.nan, device="cuda").half() for _ in range(2)]
        ring, sh = KvRing(*kv), Shadow(cache)
        qw, kw = ((1 + 0.1 * rnd(D)).half() for _ in range(2))
        mass = torch.zeros((nKV, blocks), dtype=torch.float64, device="cuda")
        n = start = L = 0
        evicted, worst = 0, [0.0] * nKV
        for step in range(34):
            M = 64 if step % 2 == 0 else int(rng.integers(1, 17))
            parents = None if M == 64 or step % 4 == 1 else ref.tree(M, rng)
            qkv = (rnd(M, (nQ + 2 * nKV) * D) * torch.exp(0.3 * rnd(1, (nQ + 2 * nKV) * D))).half()
            q = torch.empty((M, nQ * D), device="cuda").half()
            out = torch.empty_like(q)
            ctx.qkv_append(cfg, qkv, qw, kw, ring, L, parents, M, q)
            slots = [(start + i) % cap for i in range(L - start + M)]
            own = ref.sees(parents, M)[0].cuda()
            sparse = n > 6 and step % 3 == 2
            sel = None
            if sparse:
                sel = torch.empty((M, nKV, 5), dtype=torch.int32, device="cuda")
                ctx.kv8_select(cache, q, M, nQ, n, 5, 1, 2, sel)
                ctx.kv8_attn(cache, ring, q, M, nQ, n, start, L, parents, out, sel=sel)
            else:
                ctx.kv8_attn(cache, ring, q, M, nQ, n, start, L, parents, out, mass_in=cache.mass,
                             mass_out=cache.mass)
            for g in range(nKV):
                k, v = sh.keys(g, kv, slots)
                ok = torch.cat([torch.ones((M, k.shape[0] - M), dtype=torch.bool, device="cuda"), own], 1)
                if sparse:
                    at = sel[:, g].long()
                    assert (at[:, 1:] > at[:, :-1]).all() and (at[:, 0] == 0).all()
                    assert (at[:, -2:] == torch.tensor([n - 2, n - 1], device="cuda")).all()
                    seen = torch.zeros((M, n), dtype=torch.bool, device="cuda").scatter_(1, at, True)
                    ok[:, :n * B] = seen.repeat_interleave(B, 1)
                qg = q.reshape(M, nKV, G, D)[:, g]
                want, p, tol, rel = attend(qg, k, v, ok, G)
                err = (out.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D) - want).abs()
                assert (err <= tol).all(), (step, g, float((err / tol).max()))
                if not sparse and n:
                    add = p[:, :n * B].reshape(M * G, n, B).sum(2).sum(0)
                    mass[g, :n] += add
                    # one call's bound, of the greatest relative error so far and a pass's most rows
                    worst[g] = max(worst[g], float(rel.max()) + 2.0 ** -20)
                    tol = mass[g, :n] * (worst[g] + (step + 1) * (64 * G + 4) * ref.E32)
                    assert ((cache.mass[g, :n].double() - mass[g, :n]).abs() <= tol + 1e-30).all()
            # commit: a path from the root
            path = list(range(M)) if M == 64 else [0]
            while M != 64:
                nxt = [r for r in range(1, M) if (r - 1 if parents is None else parents[r]) == path[-1]]
                if not nxt or len(path) > 6:
                    break
                path.append(nxt[0])
            for t in kv:
                t[:, [(L + i) % cap for i in range(len(path))]] = t[:, [(L + r) % cap for r in path]].clone()
            L += len(path)
            while L - start >= 64 + 32 or (L - start >= 64 and step == 33):
                pos = [(start + i) % cap for i in range(64)]
                for g in range(nKV):
                    two = [ref.seal(t[g, pos]) for t in kv]
                    sh.blocks[g].append([c * s.double() for c, s in two])
                ctx.kv8_seal(cache, ring, start, 1, n)
                n, start = n + 1, start + 64
            if n >= 12:
                old, before = cache.mass.clone(), [list(p) for p in sh.pages]
                cache.evict(n, 8, n_first=1, n_last=4)
                for g in range(nKV):
                    keep = ref.choose(old[g, :n].tolist(), 1, 4, 8)
                    gone = [i for i in range(n) if i not in keep]
                    sh.pages[g] = [before[g][i] for i in keep + gone] + before[g][n:]
                    sh.blocks[g] = [sh.blocks[g][i] for i in keep]
                    assert cache.table[g].tolist() == sh.pages[g]
                    assert torch.equal(cache.mass[g, :8], old[g, keep]) and (cache.mass[g, 8:] == 0).all()
                    mass[g, :8], mass[g, 8:] = mass[g, keep].clone(), 0.0
                n, evicted = 8, evicted + 1
        assert evicted >= 2 and n >= 8 and L > 1000  # (the run came where it should)
        # a rewind into the last sealed block
        n, start = n - 1, start - 64
        ctx.kv8_unseal(cache, n, 1, ring, start)
        L = start + 21
        for g in range(nKV):
            for x, t in enumerate(kv):
                assert torch.equal(t[g, [(start + i) % cap for i in range(64)]],
                                   sh.blocks[g][n][x].float().half())
            sh.blocks[g].pop()
        q, out = rnd(1, nQ * D).half(), torch.empty((1, nQ * D), device="cuda").half()
        ctx.kv8_attn(cache, ring, q, 1, nQ, n, start, L, None, out)
        slots = [(start + i) % cap for i in range(22)]
        for g in range(nKV):
            k, v = sh.keys(g, kv, slots)
            want, _, tol, _ = attend(q.reshape(nKV, G * D)[g:g + 1], k, v,
                                     torch.ones((1, k.shape[0]), dtype=torch.bool, device="cuda"), G)
            assert ((out.double().reshape(nKV, G, D)[g] - want).abs() <= tol).all()
    ctx.sync()


# --------------------------------------------------------------------------------- capture
def filled(ctx, nKV, n, cap, seed, spare=2):
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda")

    cache = Kv8Cache(ctx, nKV, n + spare)
    src = [rnd(nKV, n * B, D).half() for _ in range(2)]
    kv = [rnd(nKV, cap, D).half() for _ in range(2)]
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(*src), 0, n, 0)
    ctx.sync()
    return cache, kv, KvRing(*kv), rnd


@pytest.mark.parametrize("M,n", [(1, 40), (9, 700), (64, 30)])
def test_captured(ctx, M, n):
    """All calls of a pass in one graph, replayed on new inputs between eager work: the eager calls'
    bits each time."""
    import torch

    nQ, nKV, open_, n_sel = 16, 4, 70, 12
    cfg, start = cfg_of(), n * B
    L, cap = start + open_, open_ + M + 64
    cache, kv, ring, rnd = filled(ctx, nKV, n, cap, M)
    qkv = rnd(M, (nQ + 2 * nKV) * D).half()
    w = [(1 + 0.1 * rnd(D)).half() for _ in range(2)]
    q, o1, o2 = (torch.zeros((M, nQ * D), device="cuda").half() for _ in range(3))
    sel = torch.zeros((M, nKV, n_sel), dtype=torch.int32, device="cuda")
    mass = torch.zeros_like(cache.mass)
    table, mass2 = torch.zeros_like(cache.table), torch.zeros_like(mass)
    back = [torch.zeros((nKV, 64, D), device="cuda").half() for _ in range(2)]
    from momij_amd.kv8 import KvRing

    bring = KvRing(*back)
    ws = torch.empty(max(ctx.kv8_workspace(nQ, nKV, M, n, s, open_ + M, m)
                         for s, m in ((0, True), (n_sel, False))), dtype=torch.uint8, device="cuda")
    results = [q, sel, o1, o2, mass, cache.k_codes, cache.v_scale, cache.k_bounds, table, mass2, *kv, *back]

    def calls(ws):
        ctx.qkv_append(cfg, qkv, *w, ring, L, None, M, q)
        ctx.kv8_select(cache, q, M, nQ, n, n_sel, 1, 2, sel, ws=ws)
        ctx.kv8_attn(cache, ring, q, M, nQ, n, start, L, None, o1, sel=sel, ws=ws)
        ctx.kv8_attn(cache, ring, q, M, nQ, n, start, L, None, o2, mass_in=mass, mass_out=mass, ws=ws)
        ctx.kv8_seal(cache, ring, start, 1, n)
        ctx.kv8_unseal(cache, n, 1, bring, 0)
        ctx.kv8_evict(cache, n, n // 2, 1, 2, mass, table, mass2)

    torch.cuda.synchronize()
    calls(None)
    ctx.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(ctx.stream):
        g.capture_begin(capture_error_mode="thread_local")
        calls(ws)
        g.capture_end()
    for i in range(4):
        qkv.copy_(rnd(*qkv.shape).half())
        mass.copy_(torch.rand_like(mass))
        m0 = mass.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(ctx.stream):
            g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        mass.copy_(m0)
        for t in (q, o1, o2, table, mass2, *back):
            t.zero_()
        sel.fill_(-7)
        (rnd(500, 500) @ rnd(500, 500)).sum().item()
        torch.cuda.synchronize()
        calls(None if i % 2 else ws)
        ctx.sync()
        for a, b in zip(got, results):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_refused_while_capturing(ctx):
    """Scratch of the context and host trees are refused while the stream is captured; the capture goes
    on."""
    import torch

    from momij_amd._lib import MomijError

    nQ, nKV, n, M = 16, 4, 6, 3
    cache, kv, ring, rnd = filled(ctx, nKV, n, 80, 5)
    q, out = rnd(M, nQ * D).half(), torch.zeros((M, nQ * D), device="cuda").half()
    qkv, w = rnd(M, 24 * D).half(), rnd(D).half()
    sel = torch.zeros((M, nKV, 2), dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(3)
    aw = {k: dev(v) for k, v in synth.attn_weights(rng, 2048, nQ, nKV, D, 64).items()}
    h = dev(synth.normal_f16(rng, (M, 2048)))
    tree = [-1, 0, 0]
    refused = [lambda: ctx.kv8_select(cache, q, M, nQ, n, 2, 0, 0, sel),
               lambda: ctx.kv8_attn(cache, ring, q, M, nQ, n, n * B, n * B, None, out),
               lambda: ctx.kv8_attn(cache, ring, q, M, nQ, n, n * B, n * B, tree, out, ws=ws),
               lambda: ctx.qkv_append(cfg_of(), qkv, w, w, ring, 0, tree, M, q),
               lambda: ctx.attn_block_kv8(cfg_of(), aw, cache, ring, h, n, n * B, n * B, None, M)]
    torch.cuda.synchronize()
    before = [t.clone() for t in (q, sel, h, *kv)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(ctx.stream):
        g.capture_begin(capture_error_mode="thread_local")
        try:
            for f in refused:
                with pytest.raises(MomijError) as e:
                    f()
                assert e.value.status == 6
        finally:
            ctx.kv8_attn(cache, ring, q, M, nQ, n, n * B, n * B, None, out, ws=ws)
            g.capture_end()
        assert (out == 0).all()
        g.replay()
    torch.cuda.synchronize()
    got = out.clone()
    assert all(torch.equal(a, b) for a, b in zip(before, (q, sel, h, *kv)))
    ctx.kv8_attn(cache, ring, q, M, nQ, n, n * B, n * B, None, out)
    ctx.sync()
    assert torch.equal(got, out)
    for f in refused:  # and each is taken outside of a capture
        f()
    ctx.sync()


# ------------------------------------------------------------------------- abort, contexts
def test_abort_leaves_everything(ctx):
    import torch

    from momij_amd._lib import MomijError

    nQ, nKV, n, M = 16, 4, 600, 3
    cache, kv, ring, rnd = filled(ctx, nKV, n, 160, 6)
    q, out = rnd(M, nQ * D).half(), rnd(M, nQ * D).half()
    qkv, w = rnd(M, 24 * D).half(), rnd(D).half()
    sel = torch.full((M, nKV, 2), 5, dtype=torch.int32, device="cuda")
    mass, table = torch.rand_like(cache.mass), torch.full_like(cache.table, 3)
    mass2 = torch.rand_like(mass)
    rng = np.random.default_rng(3)
    aw = {k: dev(v) for k, v in synth.attn_weights(rng, 2048, nQ, nKV, D, 64).items()}
    h = dev(synth.normal_f16(rng, (M, 2048)))
    held = [q, out, sel, mass, table, mass2, h, cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale,
            cache.k_bounds, *kv]

    def calls():
        for m in (n, 40):  # both ways of choosing, both of evicting
            ctx.kv8_select(cache, q, M, nQ, m, 2, 0, 0, sel)
            ctx.kv8_attn(cache, ring, q, M, nQ, m, n * B, n * B + 64, None, out, mass_in=mass, mass_out=mass)
            ctx.kv8_evict(cache, m, m // 2, 0, 0, mass, table, mass2)
        ctx.kv8_seal(cache, ring, n * B, 1, 3)
        ctx.kv8_unseal(cache, 5, 1, ring, n * B)
        ctx.attn_block_kv8(cfg_of(), aw, cache, ring, h, n, n * B, n * B + 64, None, M)
        ctx.qkv_append(cfg_of(), qkv, w, w, ring, n * B + 64, None, M, q)

    before = [t.clone() for t in held]
    torch.cuda.synchronize()
    ctx.set_abort(True)
    try:
        calls()
        torch.cuda.synchronize()
        for a, b in zip(before, held):
            assert torch.equal(a, b)
    finally:
        ctx.set_abort(False)
    with pytest.raises(MomijError):  # the waiting call after an abort reports it
        ctx.sync()
    calls()
    ctx.sync()
    changed = [not torch.equal(a, b) for a, b in zip(before, held)]
    assert all(changed), changed


def test_two_contexts(ctx):
    """Calls of two contexts on their own streams, queued together over one pool: each has the result
    that it has alone."""
    import torch

    from momij_amd.ops import Context

    other = Context(0)
    nQ, nKV, n = 16, 4, 200
    cache, kv, ring, rnd = filled(ctx, nKV, n, 200, 8)
    jobs = []
    for i in range(12):
        M = [1, 9, 33][i % 3]
        q = rnd(M, nQ * D).half()
        jobs.append((M, q, torch.empty_like(q), torch.empty((M, nKV, 9), dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()

    def go(c, job):
        M, q, out, sel = job
        c.kv8_select(cache, q, M, nQ, n, 9, 1, 1, sel)
        c.kv8_attn(cache, ring, q, M, nQ, n, n * B, n * B + 80, None, out, sel=sel if M == 9 else None)

    alone = []
    for job in jobs:
        go(ctx, job)
        ctx.sync()
        alone.append((job[2].clone(), job[3].clone()))
        job[2].zero_(), job[3].zero_()
    torch.cuda.synchronize()
    for i, job in enumerate(jobs):
        go((ctx, other)[i % 2], job)
    ctx.sync()
    other.sync()
    for (o, s), job in zip(alone, jobs):
        assert torch.equal(o, job[2]) and torch.equal(s, job[3])
    other.close()


# ------------------------------------------------------------------- a model's caches, far memory
def test_model_caches_as_rings(ctx):
    """A resident model's fp16 caches sealed and read where they are."""
    import ctypes as C

    import torch

    from momij_amd.engine import MapleLikeConfig, VerifyEngine, random_model
    from momij_amd.kv8 import Kv8Cache, KvRing

    cfg = MapleLikeConfig(n_layers=2, window=0, kv_capacity=400, E=16, top_k=4, vocab=2048)
    layers, embed, fnorm, head = random_model(cfg, seed=3)
    torch.cuda.synchronize()
    eng = VerifyEngine(ctx, cfg, layers, embed, fnorm, head)
    eng.prefill(np.random.default_rng(1).integers(0, 2048, 230).astype(np.int32))
    nKV, nQ, cap = 4, 16, 400
    addr = eng.kv(1)
    kv = []
    for a in addr:
        t = np.empty((nKV, cap, D), np.float16)
        ctx.check(ctx.lib.mj_d2h(ctx.h, t.ctypes.data_as(C.c_void_p), a, t.nbytes))
        kv.append(dev(t))
    cache, ring = Kv8Cache(ctx, nKV, 3), KvRing(*addr, capacity=cap)
    q = torch.randn((1, nQ * D), device="cuda").half()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, ring, 0, 3, 0)
    ctx.kv8_attn(cache, ring, q, 1, nQ, 3, 192, 229, None, out)
    ctx.sync()
    for g in range(nKV):
        k, v = (torch.cat([(c * s.double()[:, None, None]).reshape(-1, D), t[g, 192:230].double()])
                for t in kv for c, s in [ref.seal(t[g, :192].reshape(3, B, D))])
        want, _, tol, _ = attend(q.reshape(nKV, -1)[g:g + 1], k, v,
                                 torch.ones((1, 230), dtype=torch.bool, device="cuda"), nQ // nKV)
        assert ((out.double().reshape(nKV, -1, D)[g] - want).abs() <= tol).all()


def test_past_32_bits(ctx):
    """Pages past 4 GiB of codes and ring rows past 2 GiB."""
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    blocks, cap, n, M, nQ = 600000, 9000000, 5, 2, 4
    cache = Kv8Cache(ctx, 1, blocks)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    kv = [torch.zeros((1, cap, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    start = 3 * cap + 8900000
    for t in kv:
        t[:, 8900000:8900700] = torch.randn((1, 700, D), generator=gen, device="cuda").half()
    ring = KvRing(*kv)
    at = blocks - n
    cache.mass[0, :n] = torch.tensor([1.0, 3.0, 2.0, 5.0, 4.0], device="cuda")
    q = torch.randn((M, nQ * D), generator=gen, device="cuda").half()
    out, sel = torch.empty_like(q), torch.empty((M, 1, 2), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, ring, start, n, at)
    cache.table[0, :n] = torch.arange(at, blocks, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_attn(cache, ring, q, M, nQ, n, start + n * B, start + n * B + 100, None, out)
    ctx.kv8_select(cache, q, M, nQ, n, 2, 0, 0, sel)
    cache.evict(n, 2, 0, 0)
    ctx.kv8_unseal(cache, 0, 1, ring, start + 600)
    ctx.sync()
    s0 = 8900000
    two = [ref.seal(t[0, s0:s0 + n * B].reshape(n, B, D)) for t in kv]
    k, v = (torch.cat([(c * s.double()[:, None, None]).reshape(-1, D), t[0, s0 + n * B:s0 + n * B + 102].double()])
            for t, (c, s) in zip(kv, two))
    ok = torch.ones((M, k.shape[0]), dtype=torch.bool, device="cuda")
    ok[0, -1] = False
    want, _, tol, _ = attend(q, k, v, ok, nQ)
    assert ((out.double().reshape(M * nQ, D) - want).abs() <= tol).all()
    sc = ref.scores(q.reshape(M, 1, nQ, D), two[0][0].amax(1)[None], two[0][0].amin(1)[None], two[0][1][None])
    assert sel[:, 0].tolist() == [ref.choose(sc[r, 0].tolist(), 0, 0, 2) for r in range(M)]
    assert cache.table[0, :n].tolist() == [at + i for i in (3, 4, 0, 1, 2)]
    c, s = two[0]
    assert torch.equal(kv[0][0, s0 + 600:s0 + 664], (c[3] * s[3].double()).float().half())


# ----------------------------------------------------------------------- where the rules turn
@pytest.mark.parametrize("M,nQ,nKV,n,open_", [(1, 16, 4, 40, 5000), (9, 16, 4, 300, 4200), (3, 64, 64, 9, 700),
                                              (64, 16, 4, 2, 2100), (2, 8, 1, 0, 20000)])
def test_long_rings(ctx, M, nQ, nKV, n, open_):
    """More ring units than a head's share of the chip: they and the pages are all read."""
    import torch

    from tests.test_gpu_kv8 import Ctx8, check_rows, gen, run_attn

    rnd = gen(open_)
    c = Ctx8(ctx, rnd, nKV, n, open_, M)
    q = rnd(M, nQ * D).half()
    mass = torch.zeros((nKV, n + 2), device="cuda")
    out, _ = run_attn(ctx, c, q, nQ, nKV, None, mass=mass)
    check_rows(c, q, out, nQ, nKV, c.mask(None))


@pytest.mark.parametrize("n", [511, 512, 513, 640])
@pytest.mark.parametrize("M", [1, 7])
def test_select_either_way(ctx, M, n):
    """Lists around the length from which choosing takes two launches, equal scores among them."""
    import torch

    from momij_amd.kv8 import Kv8Cache

    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    nQ, nKV, n_sel, pages = 12, 4, 70, 100  # pages listed several times: ties
    cache = Kv8Cache(ctx, nKV, n)
    cache.k_bounds.copy_(torch.randint(-127, 128, cache.k_bounds.shape, generator=gen, device="cuda"))
    cache.k_bounds.copy_(torch.stack([cache.k_bounds.amax(1), cache.k_bounds.amin(1)], 1))
    cache.k_scale.copy_(torch.rand(cache.k_scale.shape, generator=gen, device="cuda") + 0.5)
    cache.table.copy_(torch.randint(0, pages, cache.table.shape, generator=gen, device="cuda"))
    q = torch.randn((M, nQ * D), generator=gen, device="cuda").half()
    sel = torch.empty((M, nKV, n_sel), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kv8_select(cache, q, M, nQ, n, n_sel, 3, 5, sel)
    ctx.sync()
    at = cache.table.long()
    sc = ref.scores(q.reshape(M, nKV, nQ // nKV, D), cache.k_bounds[at, 0].double(),
                    cache.k_bounds[at, 1].double(), cache.k_scale[at]).cpu()
    for r in range(M):
        for g in range(nKV):
            assert sel[r, g].tolist() == ref.choose(sc[r, g].tolist(), 3, 5, n_sel), (r, g)


LONG = [
    # M, nQ, nKV, blocks, open rows, tree: sizes on the far side of each rule
    (1, 16, 4, 100, 5, False), (3, 16, 4, 321, 0, True),             # a tile, pages of each wave's own
    (5, 128, 32, 81, 3, True), (8, 64, 16, 161, 64, False),          # two tiles
    (9, 128, 32, 115, 50, False), (13, 128, 32, 111, 1, True),       # three, four: pages of two waves
    (12, 16, 4, 900, 17, True), (16, 16, 4, 877, 9, False),
    (64, 16, 4, 360, 10, True), (33, 64, 16, 91, 0, False),          # two tiles a wave, pages shared
    (2, 16, 1, 300, 66, False)]                                      # parts past one round of the join


@pytest.mark.parametrize("M,nQ,nKV,n,open_,tree", LONG)
@pytest.mark.parametrize("mass", [False, True])
def test_long_contexts(ctx, M, nQ, nKV, n, open_, tree, mass):
    import torch

    from tests.test_gpu_kv8 import Ctx8, gen, run_attn

    rnd = gen(M + n)
    c = Ctx8(ctx, rnd, nKV, n, open_, M)
    parents = ref.tree(M, np.random.default_rng(n)) if tree else None
    c.cache.table[nKV - 1, n // 2] = -1  # one head lacks a block
    q = rnd(M, nQ * D).half()
    m0 = torch.rand((nKV, n + 2), device="cuda") if mass else None
    out, m1 = run_attn(ctx, c, q, nQ, nKV, parents, mass=m0)
    again, m2 = run_attn(ctx, c, q, nQ, nKV, parents, mass=m0)
    assert torch.equal(out, again) and (not mass or torch.equal(m1, m2))
    G, seen = nQ // nKV, c.mask(parents)
    for g in range(nKV):
        ok = seen.clone()
        if g == nKV - 1:
            ok[:, n // 2 * B:(n // 2 + 1) * B] = False
        want, p, tol, rel = attend(q.reshape(M, nKV, G, D)[:, g], *c.keys(g), ok, G)
        err = (out.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D) - want).abs()
        assert (err <= tol).all(), (g, float((err / tol).max()))
        if mass:
            add = p[:, :n * B].reshape(M * G, n, B).sum(2)
            want = m0[g, :n].double() + add.sum(0)
            tol = (add * (rel + 2.0 ** -20)).sum(0) + want * (M * G + 4) * ref.E32 + 1e-30
            assert ((m1[g, :n].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("M,nQ,nKV,n,n_sel", [(8, 384, 8, 90, 64), (40, 80, 4, 30, 20), (5, 64, 1, 700, 9)])
def test_long_lists_of_rows(ctx, M, nQ, nKV, n, n_sel):
    """Rows with lists of their own and more than a tile of heads."""
    import torch

    from tests.test_gpu_kv8 import Ctx8, check_rows, gen, run_attn

    rnd = gen(nQ)
    c = Ctx8(ctx, rnd, nKV, n, 20, M)
    rng = np.random.default_rng(n)
    sel = np.stack([[np.sort(rng.permutation(n)[:n_sel]) for _ in range(nKV)] for _ in range(M)])
    blocks = torch.zeros((M, nKV, n), dtype=torch.bool).scatter_(2, torch.from_numpy(sel), True)
    q = rnd(M, nQ * D).half()
    out, _ = run_attn(ctx, c, q, nQ, nKV, None, sel=torch.from_numpy(sel.astype(np.int32)).cuda())
    check_rows(c, q, out, nQ, nKV, torch.stack([c.mask(None, blocks[:, g]) for g in range(nKV)]))


@pytest.mark.parametrize("M,nQ,nKV,n,open_,tree", [(1, 16, 4, 30, 8192, False), (9, 8, 2, 3, 20001, True),
                                                   (64, 16, 2, 0, 9000, True), (3, 64, 16, 1, 16500, False)])
def test_rings_of_several_units_a_part(ctx, M, nQ, nKV, n, open_, tree):
    """Open rows past 8192, an infinity and a NaN among the values in different units."""
    import torch

    from tests.test_gpu_kv8 import Ctx8, gen, run_attn

    rnd = gen(open_ + 1)
    c = Ctx8(ctx, rnd, nKV, n, open_, M, spread=0.5)
    parents = ref.tree(M, np.random.default_rng(M)) if tree else None
    q = rnd(M, nQ * D).half()
    out, _ = run_attn(ctx, c, q, nQ, nKV, parents)
    G, ok = nQ // nKV, c.mask(parents)

    def check(skip=()):
        for g in range(nKV):
            want, _, tol, _ = attend(q.reshape(M, nKV, G, D)[:, g], *c.keys(g), ok, G)
            err = (out.double().reshape(M, nKV, G, D)[:, g].reshape(M * G, D) - want).abs()
            keep = [d for d in range(D) if (g, d) not in skip]
            assert (err <= tol)[:, keep].all(), g

    check()
    c.rv[0, c.slots[5], 3], c.rv[nKV - 1, c.slots[open_ - 70], 77] = math.inf, math.nan
    out, _ = run_attn(ctx, c, q, nQ, nKV, parents)
    o = out.reshape(M, nKV, G, D)
    assert (o[:, 0, :, 3] == math.inf).all() and o[:, nKV - 1, :, 77].isnan().all()
    c.rv[0, c.slots[5], 3], c.rv[nKV - 1, c.slots[open_ - 70], 77] = 0.0, 0.0
    check(skip={(0, 3), (nKV - 1, 77)})


# -------------------------------------------------------------------------- scales far apart
@pytest.mark.parametrize("nQ,lead", [(4, 0.6), (4, 0.2), (32, 0.6), (64, 1.2)])
def test_v_scales_far_apart(ctx, nQ, lead):
    """Blocks of V from the least fp16 number to the greatest, one of zeros; each row attends to one block
    above all.  The weights carry the V scale into fp16, so a block's bound counts the steps of weights
    below fp16's normal range: 2^-25 of a code, in units of at most the greatest weight times scale."""
    import torch

    from momij_amd.kv8 import Kv8Cache, KvRing

    gen = torch.Generator(device="cuda")
    gen.manual_seed(nQ)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda")

    n = M = 21
    way = rnd(n, 1, D)
    kk = (0.3 * rnd(n, B, D) + 3 * way).half()
    amp = 2.0 ** torch.linspace(-24, 13, n, device="cuda")[torch.randperm(n, generator=gen, device="cuda")]
    vv = (rnd(n, B, D) * amp[:, None, None]).clamp(-65504, 65504).half()
    vv[4] = 0.0
    vv[9] = 0.0
    vv[9, 3, 7] = 2.0 ** -24
    rk, rv = rnd(1, M + 40, D).half(), rnd(1, M + 40, D).half()
    q = (0.5 * rnd(M, nQ, D) + lead * way).half().reshape(M, nQ * D)
    cache, out = Kv8Cache(ctx, 1, n), torch.empty_like(q)
    torch.cuda.synchronize()
    ctx.kv8_seal(cache, KvRing(kk.reshape(1, -1, D), vv.reshape(1, -1, D)), 0, n, 0)
    ctx.kv8_attn(cache, KvRing(rk, rv), q, M, nQ, n, n * B, n * B + 40, None, out, mass_out=cache.mass)
    ctx.sync()
    (kc, ks), (vc, vs) = ref.seal(kk), ref.seal(vv)
    at = [(n * B + i) % (M + 40) for i in range(M + 40)]
    k = torch.cat([(kc * ks.double()[:, None, None]).reshape(-1, D), rk[0, at].double()])
    scale = torch.cat([vs.double().repeat_interleave(B), torch.ones(M + 40, device="cuda").double()])
    code = torch.cat([vc.reshape(-1, D), rv[0, at].double()])
    ok = torch.cat([torch.ones((M, n * B + 40), dtype=torch.bool), ref.sees(None, M)[0]], 1).cuda()
    want, p, _, rel = attend(q, k, code * scale[:, None], ok, nQ)
    unit = (p * scale).amax(1, keepdim=True)
    tol = (p @ (code * scale[:, None]).abs()) * (ref.E16 + rel + 2.0 ** -20) + want.abs() * ref.E16
    tol += 2.0 ** -25 * (1 + unit * code.abs().sum(0))
    err = (out.double().reshape(M * nQ, D) - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    add = p[:, :n * B].reshape(M * nQ, n, B).sum(2)
    tol = (add * (rel + 2.0 ** -20)).sum(0) + add.sum(0) * (M * nQ + 4) * ref.E32 + 1e-30
    assert ((cache.mass[0].double() - add.sum(0)).abs() <= tol).all()
