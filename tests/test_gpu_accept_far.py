"""GPU: the drafts of a batch checked where logits are finite and large (masks of the lowest float, peaks, rows
far from 0), against the rules in 64 bits (tests/paged_ref.py); whole numbers, compared exactly."""
import math

import numpy as np
import pytest
import torch

from test_gpu_accept_rows import cuda, ctx, go, want  # noqa: F401

pytestmark = pytest.mark.gpu
LOWEST = -3.4028234663852886e38
# three chunks of ids and a few; no multiple of a power of two, so no running sum meets a uniform's multiple of all
V, N = 12301, 48


def rows_and_drafts(form):
    """The rows of N sequences, and the parents where they are trees."""
    return [4] * N, ([[-1, 0, 0, 1]] * N if form == "tree" else None)


def case(form, seed, logits):
    """logits(gen): [4 N, V].  Drafts: of every second sequence what stands out in its parent's row, else any id;
    uniforms of which a third are small."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    total = 4 * N
    x = logits(gen, total)
    par = torch.arange(total, device="cuda").reshape(N, 4)[:, [0, 0, 0 if form == "tree" else 1, 1 if form == "tree" else 2]]
    some = torch.randint(0, V, (total,), generator=gen, device="cuda")
    best = x.argmax(-1)[par.reshape(-1)]
    tokens = torch.where(torch.arange(total, device="cuda") // 4 % 2 == 0, best, some).int()
    u = torch.rand(total, generator=gen, device="cuda")
    d = dict(logits=x, tokens=tokens.contiguous(), T=torch.linspace(0.3, 1.3, N, device="cuda"),
             ua=torch.where(torch.rand(total, generator=gen, device="cuda") < 0.33, u * 1e-5, u),
             us=torch.rand(N, generator=gen, device="cuda"))
    if form == "drawn":
        y = torch.randn((total, V), generator=gen, device="cuda")
        d["q"] = torch.softmax(y * 2.0, -1)
    return d


def same(ctx, form, d):  # noqa: F811
    rows, parents = rows_and_drafts(form)
    got = go(ctx, rows, parents=parents, **d)
    assert got == want(rows, parents=parents, **d)
    return got


FORMS = ["certain", "tree", "drawn"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("c", [LOWEST, -1e30, -1e25, -1e20, -1e9, 1e15, 1e17, 1e20, 1e30, -LOWEST])
def test_rows_of_one_number(ctx, form, c):  # noqa: F811
    """Every id as probable as any other, wherever the logits lie."""
    got = same(ctx, form, case(form, 1, lambda gen, n: torch.full((n, V), c, device="cuda")))
    assert all(0 <= t < V for t in got[2])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("c", [LOWEST, -1e30, -1e25, -1e20, -1e9, -1e6])
@pytest.mark.parametrize("part", ["chunk", "all but one chunk", "all but one id"])
def test_masked_by_a_finite_number(ctx, form, c, part):  # noqa: F811
    """Masked ids have no probability beside ordinary ones, also where they are a whole chunk of a row."""
    def logits(gen, n):
        x = torch.randn((n, V), generator=gen, device="cuda") * 3.0
        if part == "chunk":
            x[:, 4096:8192] = c
        elif part == "all but one chunk":
            x[:, :8192] = c
        else:
            x[:, :7000], x[:, 7001:] = c, c
        return x

    got = same(ctx, form, case(form, 2, logits))
    lo, hi = {"chunk": (0, V), "all but one chunk": (8192, V), "all but one id": (7000, 7001)}[part]
    free = [s for s in range(N) if form != "tree"]  # (a tree's refused ids may be all that is not masked)
    assert all(lo <= got[2][s] < hi and not (part == "chunk" and 4096 <= got[2][s] < 8192) for s in free)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("c", [1e9, 1e15, 1e17, 1e20, 1e30, -LOWEST])
def test_peaks(ctx, form, c):  # noqa: F811
    """One id far above the others has everything; two share it."""
    def logits(gen, n):
        x = torch.randn((n, V), generator=gen, device="cuda") * 3.0
        x[:, 5000] = c
        x[n // 2:, 9000] = c
        return x

    got = same(ctx, form, case(form, 3, logits))
    assert all(t == 5000 for t in got[2][:N // 2]) if form == "certain" else set(got[2]) <= set(range(V))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("c,size", [(1e5, 4.0), (-1e5, 4.0), (1e7, 4.0), (-1e7, 4.0), (3e8, 40.0), (-3e8, 40.0)])
def test_rows_far_from_0(ctx, form, c, size):  # noqa: F811
    """The same differences as near 0 (as fp32 holds them there) weigh the same."""
    same(ctx, form, case(form, 4, lambda gen, n: torch.randn((n, V), generator=gen, device="cuda") * size + c))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("T", [1.0001e-5, 1e-3, 1e6, 1e30, math.inf])
@pytest.mark.parametrize("c", [0.0, 1e4, LOWEST])
def test_cold_and_hot(ctx, form, T, c):  # noqa: F811
    """Temperatures down to where the greatest logit is taken, and up to those at which every finite logit weighs
    the same."""
    def logits(gen, n):
        x = torch.randn((n, V), generator=gen, device="cuda") * 3.0
        x[:, ::2] = c
        return x

    d = case(form, 5, logits)
    d["T"].fill_(T)
    same(ctx, form, d)


def test_infinities_have_nothing_at_any_temperature(ctx):  # noqa: F811
    """-inf and NaN, also at an infinite temperature."""
    x = torch.full((4 * N, V), -math.inf, device="cuda")
    x[:, 1::2] = math.nan
    x[:, 6000:6003] = torch.tensor([1.0, -1e30, 7.0], device="cuda")
    d = case("certain", 6, lambda gen, n: x.clone())
    d["T"].fill_(math.inf)
    d["tokens"].fill_(11)
    got = go(ctx, [4] * N, **d)
    assert got[0] == [0] * N and got[2] == [6000 + min(2, int(np.float32(u) * 3)) for u in d["us"].tolist()]
