"""CPU: what the calls of the 8-bit KV cache refuse, each before anything is launched, and the
workspace sizes.  The context is the library's own struct without a device (a shim built here), so
every refusal comes from the argument checks; no call with valid arguments is made."""
import ctypes as C
import itertools
import os
import shutil
import subprocess

import pytest

from momij_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, SHAPE, ROOM = 4, 3, 7  # MJ_INVALID_ARG, MJ_UNSUPPORTED_SHAPE, MJ_CAPACITY
P = 1 << 20  # an aligned address nobody reads


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    import torch

    if torch.cuda.is_available():
        pytest.skip("arguments here are addresses that no device may see")
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not installed")
    d = tmp_path_factory.mktemp("kv8")
    src, so = str(d / "ctx.cpp"), str(d / "ctx.so")
    with open(src, "w") as f:
        f.write('#include "mj_abi_internal.h"\nextern "C" mj_ctx* fake_ctx() { return new mj_ctx; }\n')
    subprocess.run([hipcc, "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "momij_amd", "csrc"),
                    src, "-o", so], check=True)
    shim = C.CDLL(so)
    shim.fake_ctx.restype = C.c_void_p
    lib, ctx = _lib.load(), shim.fake_ctx()

    def go(name, *args):
        st = getattr(lib, name)(ctx, *[C.byref(a) if isinstance(a, C.Structure) else a for a in args])
        return st, lib.mj_last_error(ctx).decode()

    return go


def kv8(**kw):
    f = dict(n_kv=4, n_pages=64, kc=P, vc=P, ks=P, vs=P, kb=P, table=P, stride=16)
    f.update(kw)
    return _lib.Kv8(*f.values())


def ring(k=P, v=P, cap=256):
    return _lib.KvRingStruct(k, v, cap)


def cfg(**kw):
    f = dict(H=2048, nQ=16, nKV=4, D=128, rope=64, base=1e6, eps=1e-6, window=0, C=0, gs=64)
    f.update(kw)
    return _lib.AttnConfig(*f.values())


def parents(*p):
    return (C.c_int32 * len(p))(*p)


POOLS = [dict(kc=None), dict(vc=None), dict(ks=None), dict(vs=None), dict(kb=None), dict(table=None),
         dict(n_kv=0), dict(n_kv=1025), dict(n_pages=0), dict(stride=0), dict(stride=(1 << 20) + 1),
         dict(kc=P + 8), dict(vc=P + 1), dict(ks=P + 4), dict(kb=P + 8), dict(table=P + 4)]
RINGS = [dict(k=None), dict(v=None), dict(cap=0), dict(cap=-5), dict(cap=1 << 30), dict(k=P + 2),
         dict(v=P + 8)]


def refused(call, status, name, *args):
    st, msg = call(name, *args)
    assert st == status, (name, st, msg)
    assert msg.startswith((name[3:], "bad tree")), msg  # (the tree check is every call's)


def attn(call, status, cache=None, rg=None, nq=16, q=P, ldq=0, M=2, n=8, sel=None, n_sel=0, start=512,
         L=520, par=None, out=P, ldo=0, mi=None, mo=None, ws=P, ws_bytes=1 << 40):
    refused(call, status, "mj_kv8_attn", cache or kv8(), rg or ring(), nq, q, ldq, M, n, sel, n_sel,
            start, L, par, out, ldo, mi, mo, ws, ws_bytes)


def select(call, status, cache=None, nq=16, q=P, ldq=0, M=2, n=8, n_sel=4, first=1, last=1, sel=P, ws=P,
           ws_bytes=1 << 40):
    refused(call, status, "mj_kv8_select", cache or kv8(), nq, q, ldq, M, n, n_sel, first, last, sel, ws,
            ws_bytes)


def evict(call, status, cache=None, n=8, keep=4, first=1, last=1, mi=P, to=3 * P, mo=4 * P):
    refused(call, status, "mj_kv8_evict", cache or kv8(), n, keep, first, last, mi, to, mo)


def span(call, status, cache=None, rg=None, pos=0, count=2, at=0):
    c, r = cache or kv8(), rg or ring()
    refused(call, status, "mj_kv8_seal", c, r, pos, count, at)
    refused(call, status, "mj_kv8_unseal", c, at, count, r, pos)


def append(call, status, c=None, qkv=P, ld=0, qw=P, kw=P, rg=None, L=0, par=None, M=2, q=P):
    refused(call, status, "mj_qkv_append", c or cfg(), qkv, ld, qw, kw, rg or ring(), L, par, M, q)


def block(call, status, c=None, w=None, cache=None, rg=None, h=P, n=8, n_sel=0, first=0, last=0,
          start=512, L=520, par=None, M=2, mi=None, mo=None):
    refused(call, status, "mj_attn_block_kv8", c or cfg(), w or _lib.AttnWeights(*[P] * 9),
            cache or kv8(), rg or ring(), h, n, n_sel, first, last, start, L, par, M, mi, mo)


@pytest.mark.parametrize("bad", POOLS, ids=str)
def test_caches(call, bad):
    c = kv8(**bad)
    attn(call, BAD, cache=c)
    select(call, BAD, cache=c)
    evict(call, BAD, cache=c)
    span(call, BAD, cache=c)
    block(call, BAD, cache=c)


@pytest.mark.parametrize("bad", RINGS, ids=str)
def test_rings(call, bad):
    r = ring(**bad)
    attn(call, BAD, rg=r)
    span(call, BAD, rg=r)
    append(call, BAD, rg=r)
    block(call, BAD, rg=r)


def test_spans(call):
    for kw in (dict(pos=-1), dict(pos=(1 << 52) + 1), dict(count=-1), dict(at=-1), dict(at=15),
               dict(at=2 ** 31 - 1), dict(count=2 ** 31 - 1)):
        span(call, BAD, **kw)
    span(call, ROOM, count=5)
    span(call, ROOM, rg=ring(cap=127))


def test_rows(call):
    for f in (attn, select):
        for kw in (dict(q=None), dict(M=0), dict(M=65), dict(ldq=2047), dict(ldq=2052), dict(ldq=-8),
                   dict(ldq=1 << 32), dict(q=P + 8)):
            f(call, BAD, **kw)
        for kw in (dict(nq=0), dict(nq=18), dict(nq=4 * 65), dict(nq=-4)):
            f(call, SHAPE, **kw)
    for kw in (dict(out=None), dict(ldo=2040), dict(ldo=2052), dict(out=P + 4)):
        attn(call, BAD, **kw)


def test_attention(call):
    for kw in (dict(n=-1), dict(n=17), dict(start=-1), dict(start=521), dict(L=(1 << 52) + 1),
               dict(sel=P, n_sel=0), dict(sel=P, n_sel=-1), dict(sel=P, n_sel=(1 << 20) + 1),
               dict(n_sel=3), dict(mi=P), dict(sel=P, n_sel=3, mo=P), dict(ws=P + 8), dict(ws_bytes=16),
               dict(par=parents(0, 0)), dict(par=parents(-1, 1)), dict(par=parents(-1, -2))):
        attn(call, BAD, **kw)
    attn(call, ROOM, L=512 + 255)
    attn(call, ROOM, start=0, L=1 << 40)


def test_selection_and_eviction(call):
    for kw in (dict(n=-1), dict(n=17), dict(n_sel=0), dict(n_sel=-1), dict(n_sel=(1 << 20) + 1),
               dict(first=-1), dict(last=-1), dict(first=3, last=2), dict(first=2 ** 31 - 1),
               dict(sel=None), dict(ws=P + 4), dict(ws_bytes=0)):
        select(call, BAD, **kw)
    for kw in (dict(n=-1), dict(n=17), dict(keep=-1), dict(keep=9), dict(first=-1), dict(last=-1),
               dict(first=3, last=2), dict(keep=1), dict(mi=None), dict(to=None), dict(mo=None),
               dict(to=P), dict(mo=P), dict(to=P + 252), dict(mo=P - 252)):
        evict(call, BAD, **kw)


def test_append(call):
    for kw in (dict(qkv=None), dict(qw=None), dict(kw=None), dict(q=None), dict(q=P + 8), dict(kw=P + 2),
               dict(ld=24 * 128 - 8), dict(ld=24 * 128 + 4), dict(M=0), dict(M=65), dict(L=-1),
               dict(L=(1 << 52) + 1), dict(c=cfg(eps=-1.0)), dict(c=cfg(eps=float("nan"))),
               dict(c=cfg(base=0.0)), dict(c=cfg(base=float("nan"))), dict(par=parents(-1, 1)),
               dict(c=cfg(eps=float("inf")))):
        append(call, BAD, **kw)
    for c in (cfg(D=64), cfg(nQ=18), cfg(nKV=0), cfg(nQ=0), cfg(rope=48), cfg(rope=256), cfg(rope=-2),
              cfg(nQ=260)):
        append(call, SHAPE, c=c)
    append(call, ROOM, rg=ring(cap=1))


def test_block(call):
    for i in range(9):
        block(call, BAD, w=_lib.AttnWeights(*[None if j == i else P for j in range(9)]))
    for kw in (dict(h=None), dict(h=P + 8), dict(M=0), dict(M=65), dict(n=17), dict(n=-1), dict(n_sel=-1),
               dict(n_sel=2, first=2, last=1), dict(n_sel=4, mo=P), dict(n_sel=9, mo=P), dict(mi=P),
               dict(start=521), dict(par=parents(-1, 1)), dict(c=cfg(eps=-1.0))):
        block(call, BAD, **kw)
    for c in (cfg(H=1024), cfg(H=8192), cfg(H=2560), cfg(gs=32), cfg(window=512), cfg(nQ=8, nKV=8),
              cfg(nQ=6, nKV=2), cfg(D=256)):
        block(call, SHAPE, c=c)
    block(call, ROOM, L=512 + 255)


def test_no_context():
    lib = _lib.load()
    c, r = kv8(), ring()
    b = C.byref
    assert lib.mj_kv8_seal(None, b(c), b(r), 0, 1, 0) == BAD
    assert lib.mj_kv8_unseal(None, b(c), 0, 1, b(r), 0) == BAD
    assert lib.mj_kv8_select(None, b(c), 16, P, 0, 1, 8, 4, 1, 1, P, None, 0) == BAD
    assert lib.mj_kv8_attn(None, b(c), b(r), 16, P, 0, 1, 8, None, 0, 0, 0, None, P, 0, None, None, None,
                           0) == BAD
    assert lib.mj_kv8_evict(None, b(c), 8, 4, 1, 1, P, P, P) == BAD
    assert lib.mj_qkv_append(None, b(cfg()), P, 0, P, P, b(r), 0, None, 1, P) == BAD
    assert lib.mj_attn_block_kv8(None, b(cfg()), b(_lib.AttnWeights(*[P] * 9)), b(c), b(r), P, 0, 0, 0, 0,
                                 0, 0, None, 1, None, None) == BAD


def test_workspace():
    """Enough for the outputs of every part, and 0 for sizes that no call takes."""
    ws = _lib.load().mj_kv8_workspace
    for nq, nkv, M, n, n_sel, rows, mass in itertools.product(
            (4, 16, 64), (1, 4), (1, 9, 64), (0, 1, 300, 1 << 20), (0, 64), (0, 100, 5000), (0, 1)):
        got = ws(nq, nkv, M, n, n_sel, M + rows, mass)
        units = (rows + M + 63) // 64  # a part of its own each, beside the pages'
        need = M * nq * (units + (n > 0)) * (128 * 4 + 8)
        need += M * nq * n * 8 if mass and not n_sel else 0
        assert got >= max(need, M * nkv * n * 4 if n_sel else 0), (nq, nkv, M, n, n_sel, rows, mass)
        assert got >= ws(nq, nkv, M, n, n_sel, M + rows, 0)
    for args in ((16, 0, 1, 8, 0, 1, 0), (16, 3, 1, 8, 0, 1, 0), (0, 4, 1, 8, 0, 1, 0),
                 (260, 4, 1, 8, 0, 1, 0), (16, 4, 0, 8, 0, 1, 0), (16, 4, 65, 8, 0, 65, 0),
                 (16, 4, 2, -1, 0, 2, 0), (16, 4, 2, (1 << 20) + 1, 0, 2, 0), (16, 4, 2, 8, -1, 2, 0),
                 (16, 4, 2, 8, (1 << 20) + 1, 2, 0), (16, 4, 2, 8, 0, 1, 0), (16, 4, 2, 8, 0, 1 << 30, 0)):
        assert ws(*args) == 0, args


def test_workspace_serves_smaller_calls(call):
    """What a call asks for (it is refused without) is within the workspace of its sizes and of any
    greater ones."""
    import random
    import re

    ws, rng = _lib.load().mj_kv8_workspace, random.Random(4)
    big = kv8(stride=1 << 20, n_pages=1 << 30)

    def need(nkv, nq, M, n, n_sel, rows, mass):
        big.n_kv_heads = nkv
        st, msg = call("mj_kv8_attn", big, ring(cap=1 << 29), nq, P, 0, M, n, P if n_sel else None, n_sel,
                       0, rows - M, None, P, 0, None, P if mass else None, P, 0)
        assert st == BAD, msg
        return int(re.search(r"needs (\d+)", msg).group(1))

    for nkv, g in ((4, 4), (1, 8), (1, 64), (8, 8), (32, 1), (64, 1), (1024, 1), (2, 64), (300, 3)):
        for _ in range(40):
            M, n, rows = rng.choice([1, 2, 9, 17, 33, 64]), rng.choice([0, 1, 75, 76, 2047, 99999]), \
                rng.choice([0, 1, 80, 8000, 8300, 131000, 2 ** 28])
            n_sel, mass = rng.choice([0, 0, 5, 64, 3000]), rng.choice([0, 1])
            mass = 0 if n_sel else mass
            bound = ws(nkv * g, nkv, M, n, n_sel, rows + M, mass)
            for k in range(12):
                m = M if k % 3 == 0 else rng.randint(1, M)
                s = n_sel and rng.randint(1, n_sel)
                size = (m, n if k % 2 else rng.randint(0, n), s, m + (rows if k % 4 else rng.randint(0, rows)))
                assert need(nkv, nkv * g, *size, mass) <= bound, (nkv, g, M, n, n_sel, rows, mass, size)
                assert ws(nkv * g, nkv, *size, mass) <= bound


def test_ring_addresses_need_a_capacity():
    from momij_amd.kv8 import KvRing

    with pytest.raises(ValueError):
        KvRing(P, P)
    assert KvRing(P, P, capacity=7).struct.capacity == 7


def test_outputs_over_inputs(call):
    """Arrays that a call would overwrite before it has read them, in whole or in part: refused."""
    row = 24 * 128 * 2  # bytes of a row of qkv; q_out's rows are packed
    for q in (2 * P, 2 * P + row - 16, 2 * P + 9 * row + 16 * 256 - 16, 2 * P - 3 * 16 * 256 + 16):
        append(call, BAD, qkv=2 * P, q=q, ld=9 * 24 * 128, M=2 if q > 2 * P else 3, rg=ring(64 * P, 80 * P))
    # evict: 4 rows of 16 entries
    for kw in (dict(to=9 * P, mi=9 * P), dict(to=9 * P + 240, mi=9 * P), dict(to=9 * P, mi=9 * P + 240),
               dict(mo=P), dict(mo=P + 240), dict(mo=P - 240), dict(to=9 * P, mo=9 * P),
               dict(to=9 * P, mo=9 * P - 240)):
        evict(call, BAD, **dict(dict(mi=6 * P), **kw))
    # attention: masses added in place, or apart
    for mi in (9 * P + 16, 9 * P - 240):
        attn(call, BAD, mi=mi, mo=9 * P)
        block(call, BAD, mi=mi, mo=9 * P)


def test_plan_restated(call):
    """The split that the GPU tests name their sizes by gives the workspaces that the calls ask for."""
    import random
    import re

    from tests.kv8_plan import plan

    rng, big, seen = random.Random(7), kv8(stride=1 << 20, n_pages=1 << 30), set()
    for _ in range(3000):
        nkv, g = rng.choice([(4, 4), (1, 16), (1, 64), (8, 4), (32, 4), (64, 4), (128, 1), (2, 7)])
        M, n = rng.choice([1, 2, 5, 9, 17, 20, 40, 64]), rng.choice([1, 9, 75, 76, 200, 520, 2047, 20000])
        n_sel, mass = rng.choice([0, 0, 5, 64, 600]), rng.choice([0, 1])
        mass = 0 if n_sel else mass
        rows = M + rng.choice([0, 1, 80, 8000, 16300, 131000])
        big.n_kv_heads = nkv
        st, msg = call("mj_kv8_attn", big, ring(cap=1 << 29), nkv * g, P, 0, M, n, P if n_sel else None, n_sel,
                       0, rows - M, None, P, 0, None, P if mass else None, P, 0)
        assert st == BAD, msg
        p = plan(nkv * g, nkv, M, n, n_sel, rows, mass)
        assert int(re.search(r"needs (\d+)", msg).group(1)) == p["bytes"], (nkv, g, M, n, n_sel, rows, mass, p)
        seen.add((p["shared"], p["pair"], p["tiles"], p["upp"] > p["batch"], p["parts"] > 256))
    assert {s[:3] for s in seen} == {(True, 1, 1), (True, 1, 2), (False, 1, 1), (False, 1, 2), (False, 2, 2)}
