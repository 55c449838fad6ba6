"""CPU: outputs and workspaces of the verify step of many requests that lie over what a call still reads or writes
are refused before anything is launched."""
import itertools

import pytest

from test_paged_refusals import BAD, P, accept, append, attn, batch, call, commit, pages, reserve  # noqa: F401

POOL = 4 * 64 * 4 * 64 * 256  # bytes of K, and of V, of pages()
SERVED = 14 * P
ON_PAGES = dict(k=(20 * P, POOL), v=(30 * P, POOL), table=(P, 3 * 16 * 4), lens=(2 * P, 12), refs=(3 * P, 256),
                served=(SERVED, 12), start=(4 * P, 16), anc=(5 * P, 72))


def known():
    p = pages()
    p.served = SERVED
    return p


def ends(at, size, own, step):
    """Addresses of an array of `own` bytes that just meets [at, at + size), in whole steps."""
    return at, at - (own - 1) // step * step, at + (size - 1) // step * step


@pytest.mark.parametrize("name", list(ON_PAGES) + ["qw", "kw"])
def test_append(call, name):  # noqa: F811
    at, size = dict(ON_PAGES, qw=(6 * P, 256), kw=(7 * P, 256))[name]
    for q in ends(at, size, 9 * 4096, 16):
        append(call, BAD, p=known(), q=q)


@pytest.mark.parametrize("name", list(ON_PAGES))
def test_attention_outputs(call, name):  # noqa: F811
    at, size = ON_PAGES[name]
    for out in ends(at, size, 9 * 4096, 16):
        attn(call, BAD, p=known(), out=out)
    # columns of a wide buffer: over some row's, not beside them
    for row, col in itertools.product((0, 4, 8), (0, 16, 4080)):
        attn(call, BAD, p=known(), out=at - row * 3 * 4096 - col, ldo=3 * 2048)


@pytest.mark.parametrize("name", list(ON_PAGES) + ["q", "out"])
def test_attention_workspace(call, name):  # noqa: F811
    from momij_amd import _lib

    need = _lib.load().mj_paged_workspace(16, 4, 5)
    at, size = dict(ON_PAGES, q=(50 * P, 9 * 4096), out=(51 * P, 9 * 4096))[name]
    for ws in ends(at, size, need, 16):
        attn(call, BAD, p=known(), q=50 * P, out=51 * P, ws=ws)


def test_bookkeeping(call):  # noqa: F811
    for at, size in (ON_PAGES["k"], ON_PAGES["v"]):
        for out in ends(at, size, 48, 16):
            reserve(call, BAD, p=known(), out=out)
        for lens in ends(at, size, 12, 4):
            commit(call, BAD, p=known(), lens=lens)


@pytest.mark.parametrize("name", ["start", "anc", "tokens", "temp", "ua", "us", "accepted", "path", "token", "logits", "q"])
def test_acceptance_workspace(call, name):  # noqa: F811
    from momij_amd import _lib

    need = _lib.load().mj_accept_workspace(3, 9, 1000)
    at, size = dict(start=(4 * P, 16), anc=(5 * P, 72), tokens=(6 * P, 36), temp=(7 * P, 12), ua=(8 * P, 36), us=(9 * P, 12),
                    accepted=(10 * P, 12), path=(11 * P, 36), token=(12 * P, 12), logits=(40 * P, 36000),
                    q=(50 * P, 36000))[name]
    for ws in ends(at, size, need, 16):
        accept(call, BAD, b=batch(anc=None) if name == "q" else None, q=50 * P if name == "q" else None, ws=ws)
