"""CPU: who has room in a step (`served` of the pages): the tensors that the Python side takes, and what the
calls refuse."""
import pytest
import torch

from momij_amd import _lib
from momij_amd.paged import PagedCache
from test_paged_arguments import F32, I32, I64, N, arrays, cache_of, ctx, ctx_on, z  # noqa: F401
from test_paged_refusals import BAD, ON_PAGES, P, call, commit, fork, pages, reserve, truncate  # noqa: F401

SERVED = 14 * P


def known(at=SERVED, **kw):
    p = pages(**kw)
    p.served = at
    return p


def test_not_known_to_begin_with(ctx):  # noqa: F811
    c = cache_of(ctx)
    assert c.served.dtype == I32 and c.served.tolist() == [-1] * N
    assert c._ref._obj.served == c.served.data_ptr()
    s = z(N, dtype=I32)
    c = PagedCache.over(ctx, **arrays(), served=s)
    assert c.served is s and c._ref._obj.served == s.data_ptr()
    assert _lib.Pages(1, 1, 1, 32, P, P, P, 1, 1, P, P).served is None


@pytest.mark.parametrize("bad", [z(N, dtype=I64), z(N, dtype=F32), z(N + 1, dtype=I32), z(N - 1, dtype=I32),
                                 z(N, 1, dtype=I32), z(2 * N, dtype=I32)[::2]],
                         ids=lambda t: f"{tuple(t.shape)}{str(t.dtype)[6:]}")
def test_tensors(ctx, bad):  # noqa: F811
    with pytest.raises(ValueError):
        PagedCache.over(ctx, **arrays(), served=bad)


@pytest.mark.parametrize("f", ON_PAGES)
def test_unaligned(call, f):  # noqa: F811
    for at in (SERVED + 1, SERVED + 4, SERVED + 8):
        f(call, BAD, p=known(at))


def test_outputs_over_it(call):  # noqa: F811
    for at in (SERVED, SERVED - 32):
        reserve(call, BAD, p=known(), out=at)
    for at in (SERVED, SERVED + 8, SERVED - 8):
        fork(call, BAD, p=known(), src=at)
        truncate(call, BAD, p=known(), lens=at)
        commit(call, BAD, p=known(), lens=at)


@pytest.mark.parametrize("shape", [(2, 4100), (1, 8200), (2, 4096 + 1), (8192 + 64,), (64, 130)])
def test_pages_of_no_whole_tokens(ctx, shape):  # noqa: F811
    """Halves of a head's page that are no multiple of a token's: the pages behind would be looked for elsewhere."""
    with pytest.raises(ValueError):
        cache_of(ctx, **{x: z(2, 8, 2, *shape) for x in "kv"})
