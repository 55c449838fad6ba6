"""GPU: whatever the device arrays of a batch and of the pages hold, nothing around the arrays that a call may
write, and nothing of those that it only reads, is changed."""
import math

import pytest
import torch

from momij_amd.paged import PagedCache, RowBatch
from test_gpu_paged_attn import D, cfg, ctx, cuda  # noqa: F401

pytestmark = pytest.mark.gpu
MAX, LOW = 2 ** 31 - 1, -(2 ** 31)
N, ROWS, NQ, NKV, V, PAGES, BLOCKS, LAYERS, PAGE = 4, 6, 16, 4, 5000, 24, 6, 2, 32
GUARD = 4096  # bytes before and behind


class Guarded:
    """Tensors that lie within larger ones."""

    def __init__(self):
        self.around = []

    def __call__(self, *shape, dtype=torch.int32, fill=0):
        size = torch.empty((), dtype=dtype).element_size()
        n = math.prod(shape) * size
        pad = -n % 256
        whole = torch.full((2 * GUARD + n + pad,), 0xA5, dtype=torch.uint8, device="cuda")
        self.around.append((whole, GUARD + n))
        t = whole[GUARD:GUARD + n].view(dtype).view(shape)
        return t.copy_(fill) if torch.is_tensor(fill) else t.fill_(fill)

    def untouched(self):
        for i, (whole, end) in enumerate(self.around):
            assert bool((whole[:GUARD] == 0xA5).all()) and bool((whole[end:] == 0xA5).all()), i


STARTS = [[0, 100, -5, 3, 6], [5, 4, 3, 2, 1], [-9, -8, MAX, 7, 0], [MAX] * 5, [LOW] * 5, [0, 1, 3, 3, 6], [0, 0, 0, 0, 600],
          [6, 6, 6, 6, 6], [0, 6, 6, 6, 6], [0, 4, LOW, MAX, 6]]
TABLES = {"pages": list(range(PAGES)), "nonsense": [MAX, LOW, -1, PAGES, PAGES - 1, 0] * 4, "one page": [5] * PAGES}
LENS = {"50": [50] * N, "ends": [MAX, LOW, BLOCKS * PAGE, BLOCKS * PAGE - 1], "small": [0, 1, 31, 95]}


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("table", list(TABLES))
@pytest.mark.parametrize("max_rows", [3, 64])
def test_nothing_around_the_arrays_is_written(ctx, table, lens, max_rows):  # noqa: F811
    f16, f32, i64, u8 = (dict(dtype=x) for x in (torch.float16, torch.float32, torch.int64, torch.uint8))
    new, torn = Guarded(), []
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    refs = [max(0, TABLES[table].count(p)) for p in range(PAGES)]
    shape = (LAYERS, PAGES, NKV, PAGE // 32, 4096)
    for start in STARTS:
        c = dict(k=new(*shape, **f16), v=new(*shape, **f16), table=new(N, BLOCKS, fill=cuda(TABLES[table]).view(N, BLOCKS)),
                 lens=new(N, fill=cuda(LENS[lens])), refs=new(PAGES, fill=cuda(refs)))
        cache = PagedCache.over(ctx, *c.values())
        fixed = dict(start=new(N + 1, fill=cuda(start)), anc=new(ROWS, **i64, fill=-1),
                     qkv=new(ROWS, (NQ + 2 * NKV) * D, **f16, fill=1.0), w=new(D, **f16, fill=1.0),
                     logits=new(ROWS, V, **f32, fill=torch.randn((ROWS, V), generator=gen, device="cuda")),
                     dist=new(ROWS, V, **f32, fill=1.0 / V), tokens=new(ROWS, fill=cuda([1, -1, MAX, LOW, V, V - 1])),
                     T=new(N, **f32, fill=1.0), ua=new(ROWS, **f32, fill=0.5), us=new(N, **f32, fill=0.999),
                     accepted=new(N, fill=cuda([99, -99, 2, MAX])), path=new(ROWS, fill=cuda([0, 2, 1, -7, MAX, 5])),
                     source=new(N, fill=cuda([3, MAX, LOW, 3])), cut=new(N, fill=cuda([40, LOW, MAX, -1])))
        q, out, lens_out = new(ROWS, NQ * D, **f16), new(ROWS, NQ * D, **f16), new(N)
        reserved, acc, way, tok = new(N, 4), new(N), new(ROWS), new(N)
        ws = [new(ctx.paged_workspace(NQ, NKV, max_rows), **u8), new(ctx.accept_workspace(N, ROWS, V), **u8)]
        before = {k: t.clone() for k, t in fixed.items()}
        tree = RowBatch(fixed["start"], ROWS, max_rows, fixed["anc"])
        chain = RowBatch(fixed["start"], ROWS, max_rows)
        for b in (tree, chain):
            ctx.pages_reserve(cache, b, reserved)
            ctx.paged_append(cfg(NQ, NKV, 64), cache, 1, b, fixed["qkv"], fixed["w"], fixed["w"], q)
            ctx.paged_attn(cache, 1, b, q, NQ, out, ws=ws[0])
            ctx.paged_attn(cache, 1, b, q, NQ, out, window=40, ws=ws[0])
            for dist in (None, fixed["dist"]) if b is chain else (None,):
                ctx.accept_rows(b, fixed["logits"], fixed["tokens"], fixed["T"], fixed["ua"], fixed["us"], acc, way, tok,
                                q=dist, ws=ws[1])
            ctx.pages_commit(cache, b, fixed["accepted"], fixed["path"], lens_out)
            ctx.pages_commit(cache, b, fixed["accepted"], fixed["path"])
            ctx.pages_commit(cache, b, fixed["accepted"])
            ctx.pages_fork(cache, fixed["source"])
            ctx.pages_truncate(cache, fixed["cut"])
        ctx.sync()
        new.untouched()
        torn += [(start, k) for k, t in before.items() if not torch.equal(t, fixed[k])]
        assert not torn
        new.around.clear()
