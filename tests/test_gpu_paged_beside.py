"""GPU: arrays that lie beside the rows of an output, in the columns that the rows leave, are taken."""
import pytest
import torch

from momij_amd.paged import RowBatch
from test_gpu_paged_attn import D, chains, check, ctx, make  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 9, 40])
def test_starts_and_masks_in_the_columns_beside(ctx, M):  # noqa: F811
    nq, lens, rows = 16, [70, 200], [M, M]
    cache, gen, _ = make(ctx, lens, rows, 64, 4, seed=M)
    q = (torch.randn((2 * M, nq * D), generator=gen, device="cuda") * 2).half()
    wide = torch.full((2 * M, nq * D + 768), 7.0, dtype=torch.float16, device="cuda")
    out = wide[:, :nq * D]
    start = wide[0, nq * D:nq * D + 6].view(torch.int32)
    anc = wide[2 * M - 1, nq * D + 32:nq * D + 32 + 8 * M].view(torch.int64)
    start.copy_(torch.tensor([0, M, 2 * M], dtype=torch.int32))
    anc.copy_(torch.tensor([(2 << r) - 1 for _ in rows for r in range(M)], dtype=torch.int64))
    ctx.paged_attn(cache, 0, RowBatch(start, 2 * M, M, anc), q, nq, out)
    check(cache, rows, chains(rows), q, out, nq)
    assert start.tolist() == [0, M, 2 * M]
