"""CPU: what the calls of the verify step of many requests refuse, each before anything is launched, and
their workspace sizes.  The context is the library's own struct without a device (a shim built here), so
every refusal comes from the argument checks; no call with valid arguments is made."""
import ctypes as C
import itertools
import os
import random
import re
import shutil
import subprocess

import pytest

from momij_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, SHAPE = 4, 3  # MJ_INVALID_ARG, MJ_UNSUPPORTED_SHAPE
P = 1 << 24  # an aligned address nobody reads; every array of the calls here is below 1 << 24 bytes


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    import torch

    if torch.cuda.is_available():
        pytest.skip("arguments here are addresses that no device may see")
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not installed")
    d = tmp_path_factory.mktemp("paged")
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


def pages(**kw):
    f = dict(n_layers=4, n_kv=4, n_pages=64, page=64, k=20 * P, v=30 * P, table=P, n_seqs=3, stride=16,
             lens=2 * P, refs=3 * P)
    f.update(kw)
    return _lib.Pages(*f.values())


def batch(**kw):
    f = dict(start=4 * P, anc=5 * P, n_seqs=3, rows=9, max_rows=5)
    f.update(kw)
    return _lib.Batch(*f.values())


def cfg(**kw):
    f = dict(H=2048, nQ=16, nKV=4, D=128, rope=64, base=1e6, eps=1e-6, window=0, C=0, gs=64)
    f.update(kw)
    return _lib.AttnConfig(*f.values())


def refused(call, status, name, *args):
    st, msg = call(name, *args)
    assert st == status, (name, st, msg)
    assert msg.startswith(name[3:]), msg


def append(call, status, c=None, p=None, layer=0, b=None, qkv=10 * P, ld=0, qw=6 * P, kw=7 * P, q=11 * P):
    refused(call, status, "mj_paged_append", c or cfg(), p or pages(), layer, b or batch(), qkv, ld, qw, kw, q)


def attn(call, status, p=None, layer=0, b=None, nq=16, window=0, q=10 * P, ldq=0, out=11 * P, ldo=0, ws=12 * P,
         ws_bytes=1 << 40):
    refused(call, status, "mj_paged_attn", p or pages(), layer, b or batch(), nq, window, q, ldq, out, ldo, ws,
            ws_bytes)


def reserve(call, status, p=None, b=None, out=10 * P):
    refused(call, status, "mj_pages_reserve", p or pages(), b or batch(), out)


def fork(call, status, p=None, src=10 * P):
    refused(call, status, "mj_pages_fork", p or pages(), src)


def truncate(call, status, p=None, lens=10 * P):
    refused(call, status, "mj_pages_truncate", p or pages(), lens)


def commit(call, status, p=None, b=None, accepted=10 * P, path=11 * P, lens=12 * P):
    refused(call, status, "mj_pages_commit", p or pages(), b or batch(), accepted, path, lens)


def accept(call, status, b=None, logits=40 * P, ld=0, V=1000, tokens=6 * P, q=None, ldq=0, temp=7 * P, ua=8 * P,
           us=9 * P, accepted=10 * P, path=11 * P, token=12 * P, ws=13 * P, ws_bytes=1 << 40):
    refused(call, status, "mj_accept_rows", b or batch(), logits, ld, V, tokens, q, ldq, temp, ua, us, accepted,
            path, token, ws, ws_bytes)


ON_PAGES = [append, attn, reserve, fork, truncate, commit]
ON_BATCHES = [append, attn, reserve, commit, accept]


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(refs=None), dict(n_kv=0),
    dict(n_kv=1025), dict(n_pages=0), dict(n_pages=(1 << 28) + 1), dict(n_layers=0), dict(n_layers=4097), dict(n_seqs=0), dict(n_seqs=1025),
    dict(n_seqs=-1), dict(stride=0), dict(stride=(1 << 24) + 1), dict(page=256, stride=(1 << 22) + 1),
    dict(k=20 * P + 8), dict(v=30 * P + 2), dict(table=P + 4), dict(lens=2 * P + 4), dict(refs=3 * P + 8)],
    ids=str)
@pytest.mark.parametrize("f", ON_PAGES)
def test_pages(call, f, bad):
    f(call, BAD, p=pages(**bad))


@pytest.mark.parametrize("f", ON_PAGES)
def test_page_sizes(call, f):
    for n in (0, -64, 1, 16, 31, 33, 48, 96, 512, 1 << 30):
        f(call, SHAPE, p=pages(page=n))


@pytest.mark.parametrize("f", ON_BATCHES)
def test_batches(call, f):
    for kw in (dict(start=None), dict(n_seqs=0), dict(n_seqs=1025), dict(rows=-1), dict(rows=65536),
               dict(max_rows=0), dict(max_rows=65), dict(max_rows=-1), dict(start=4 * P + 2),
               dict(anc=5 * P + 4)):
        f(call, BAD, b=batch(**kw))
    if f is not accept:  # as many sequences as the pages
        f(call, BAD, b=batch(n_seqs=4))
        f(call, BAD, b=batch(n_seqs=2))


def test_append(call):
    for kw in (dict(qkv=None), dict(q=None), dict(qkv=10 * P + 8), dict(q=11 * P + 8), dict(qw=6 * P + 2),
               dict(kw=7 * P + 8), dict(ld=24 * 128 - 8), dict(ld=24 * 128 + 4), dict(ld=-8),
               dict(ld=1 << 32), dict(layer=-1), dict(layer=4), dict(c=cfg(eps=-1.0)),
               dict(c=cfg(eps=float("nan"))), dict(c=cfg(eps=float("inf"))), dict(c=cfg(base=0.0)),
               dict(c=cfg(base=float("nan")))):
        append(call, BAD, **kw)
    for c in (cfg(D=64), cfg(nQ=18), cfg(nKV=0), cfg(nQ=0), cfg(rope=48), cfg(rope=256), cfg(rope=-2),
              cfg(rope=16), cfg(nQ=260), cfg(nQ=16, nKV=8), cfg(nKV=2)):
        append(call, SHAPE, c=c)
    # q_out over rows of qkv that are read after it is written
    row = 24 * 256
    for q in (10 * P, 10 * P + row - 16, 10 * P + 8 * row, 10 * P - 16 * 256 + 16):
        append(call, BAD, q=q)


def test_attention(call):
    for kw in (dict(q=None), dict(out=None), dict(q=10 * P + 8), dict(out=11 * P + 2), dict(ldq=2040),
               dict(ldo=2052), dict(ldq=-8), dict(ldo=1 << 32), dict(layer=-1), dict(layer=4),
               dict(window=-1), dict(ws=12 * P + 8), dict(ws_bytes=16), dict(ws_bytes=0),
               dict(out=10 * P), dict(out=10 * P + 4096 * 9 - 16), dict(q=11 * P + 16),
               # columns of a common buffer that meet
               dict(ldq=6144, ldo=6144, out=10 * P + 4080)):
        attn(call, BAD, **kw)
    for nq in (0, -4, 18, 4 * 65):
        attn(call, SHAPE, nq=nq)


def test_bookkeeping(call):
    for kw in (dict(out=None), dict(out=10 * P + 4), dict(out=P), dict(out=P + 4 * 48 - 16), dict(out=2 * P),
               dict(out=3 * P), dict(out=4 * P)):
        reserve(call, BAD, **kw)
    for kw in (dict(src=None), dict(src=10 * P + 2), dict(src=P + 4), dict(src=2 * P), dict(src=3 * P + 8)):
        fork(call, BAD, **kw)
    for kw in (dict(lens=None), dict(lens=10 * P + 1), dict(lens=P), dict(lens=3 * P), dict(lens=2 * P + 4)):
        truncate(call, BAD, **kw)
    for kw in (dict(accepted=None), dict(lens=None), dict(accepted=10 * P + 2), dict(path=11 * P + 2),
               dict(lens=12 * P + 1), dict(lens=P), dict(lens=2 * P + 4), dict(lens=3 * P), dict(lens=4 * P),
               dict(lens=10 * P), dict(lens=10 * P + 8), dict(lens=11 * P + 32)):
        commit(call, BAD, **kw)


def test_acceptance(call):
    for kw in (dict(V=0), dict(V=-1), dict(V=(1 << 23) + 1), dict(ld=999), dict(ld=1 << 32), dict(ld=-1000),
               dict(b=batch(anc=None), q=50 * P, ldq=999), dict(logits=None), dict(tokens=None),
               dict(temp=None), dict(ua=None), dict(us=None), dict(accepted=None), dict(path=None),
               dict(token=None), dict(logits=40 * P + 2), dict(tokens=6 * P + 1), dict(us=9 * P + 2),
               dict(token=12 * P + 3), dict(ws=13 * P + 8), dict(ws_bytes=64)):
        accept(call, BAD, **kw)
    accept(call, SHAPE, q=50 * P)  # (of a tree)
    inputs = dict(start=4 * P, anc=5 * P, tokens=6 * P, temp=7 * P, ua=8 * P, us=9 * P, logits=40 * P,
                  last=40 * P + 4 * 8999)
    for at in inputs.values():
        for o in ("accepted", "path", "token"):
            accept(call, BAD, **{o: at})
    for a, b in itertools.permutations(("accepted", "path", "token"), 2):
        at = dict(accepted=10 * P, path=11 * P, token=12 * P)
        accept(call, BAD, **{a: at[b] + 8})
    accept(call, BAD, b=batch(anc=None), q=50 * P, path=50 * P + 64)


def test_no_context():
    lib, b = _lib.load(), C.byref
    p, r = pages(), batch()
    assert lib.mj_paged_append(None, b(cfg()), b(p), 0, b(r), P, 0, P, P, P) == BAD
    assert lib.mj_paged_attn(None, b(p), 0, b(r), 16, 0, P, 0, P, 0, None, 0) == BAD
    assert lib.mj_pages_reserve(None, b(p), b(r), P) == BAD
    assert lib.mj_pages_fork(None, b(p), P) == BAD
    assert lib.mj_pages_truncate(None, b(p), P) == BAD
    assert lib.mj_pages_commit(None, b(p), b(r), P, P, P) == BAD
    assert lib.mj_accept_rows(None, b(r), P, 0, 10, P, None, 0, P, P, P, P, P, P, None, 0) == BAD


def test_attention_workspace(call):
    """Enough for two partial results a block, what the call asks for, and no less for a larger batch."""
    ws = _lib.load().mj_paged_workspace
    for nkv, g, M in itertools.product((1, 2, 4, 64), (1, 3, 4, 16, 64), (1, 4, 5, 16, 63, 64)):
        got = ws(nkv * g, nkv, M)
        assert got >= 512 * min(M * g, 256) * (128 * 4 + 8), (nkv, g, M)
        assert got >= ws(nkv * g, nkv, max(M // 2, 1)) and got >= ws(nkv * max(g // 2, 1), nkv, M)
        st, msg = call("mj_paged_attn", pages(n_kv=nkv), 0, batch(max_rows=M, rows=2), nkv * g, 0, 10 * P, 0,
                       11 * P, 0, 12 * P, 0)
        assert st == BAD and int(re.search(r"needs (\d+)", msg).group(1)) == got, (nkv, g, M, msg)
    for args in ((0, 4, 1), (16, 0, 1), (18, 4, 1), (4 * 65, 4, 1), (16, 4, 0), (16, 4, 65), (-4, 4, 1),
                 (2048, 1025, 1)):
        assert ws(*args) == 0, args


def test_acceptance_workspace(call):
    """What the call asks for, and enough for any smaller one."""
    ws, rng = _lib.load().mj_accept_workspace, random.Random(5)
    for _ in range(300):
        n, rows, V = rng.randint(1, 1024), rng.randint(0, 9000), rng.choice([1, 7, 4096, 4097, 151936, 1 << 23])
        got = ws(n, rows, V)
        assert got >= (rows + n) * ((V + 4095) // 4096) * 8
        assert got >= ws(rng.randint(1, n), rng.randint(0, rows), rng.randint(1, V))
        st, msg = call("mj_accept_rows", batch(n_seqs=n, rows=rows), 1 << 50, 0, V, 6 * P, None, 0, 7 * P, 8 * P,
                       9 * P, 10 * P, 11 * P, 12 * P, 13 * P, 0)
        assert st == BAD and int(re.search(r"needs (\d+)", msg).group(1)) == got, (n, rows, V, msg)
    for args in ((0, 1, 10), (1025, 1, 10), (1, -1, 10), (1, 65536, 10), (1, 1, 0), (1, 1, (1 << 23) + 1)):
        assert ws(*args) == 0, args
