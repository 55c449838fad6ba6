"""CPU: tensors that the Python calls of the verify step of many requests do not take.  A tensor of another
type, layout, size or device than the call reads would be read or written out of range, so each is a
ValueError before the library is reached.  The library is a recorder here and the device is torch's "none"
(-1), which the CPU tensors have."""
import pytest
import torch

from momij_amd.ops import Context
from momij_amd.paged import PagedCache, RowBatch, tree_masks

NQ, NKV, D, N, BLOCKS, PAGES, LAYERS, R, V = 10, 2, 128, 3, 5, 8, 2, 7, 50
F16, F32, I32, I64 = torch.float16, torch.float32, torch.int32, torch.int64


class Recorder:
    """Every entry succeeds; what was called with what."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


def ctx_on(device):
    c = object.__new__(Context)
    c.lib, c.h, c.device = Recorder(), None, device
    return c


@pytest.fixture
def ctx():
    return ctx_on(-1)


def arrays(**kw):
    f = dict(k=z(LAYERS, PAGES, NKV, 2, 4096), v=z(LAYERS, PAGES, NKV, 2, 4096), table=z(N, BLOCKS, dtype=I32),
             lens=z(N, dtype=I32), refs=z(PAGES, dtype=I32))
    f.update(kw)
    return f


def cache_of(ctx, **kw):
    return PagedCache.over(ctx, **arrays(**kw))


def batch_of(anc=True, rows=R):
    return RowBatch(z(N + 1, dtype=I32), rows, 4, z(rows, dtype=I64) if anc else None)


def cfg(**kw):
    return dict(dict(H=2048, nQ=NQ, nKV=NKV, D=D, rope_dim=64, rope_base=1e6, eps=1e-6, window=0, C=0,
                     gs=64), **kw)


def append(ctx, cache=None, batch=None, qkv=None, qw=None, kw=None, q=None, rows=R):
    ctx.paged_append(cfg(), cache or cache_of(ctx), 1, batch or batch_of(rows=rows),
                     z(rows, (NQ + 2 * NKV) * D) if qkv is None else qkv, qw, kw,
                     z(rows, NQ * D) if q is None else q)


def attn(ctx, cache=None, batch=None, q=None, out=None, ws=None, rows=R):
    ctx.paged_attn(cache or cache_of(ctx), 1, batch or batch_of(rows=rows), z(rows, NQ * D) if q is None else q,
                   NQ, z(rows, NQ * D) if out is None else out, 0, ws)


def reserve(ctx, cache=None, batch=None, out=None):
    ctx.pages_reserve(cache or cache_of(ctx), batch or batch_of(), z(N, 4, dtype=I32) if out is None else out)


def fork(ctx, cache=None, source=None):
    ctx.pages_fork(cache or cache_of(ctx), z(N, dtype=I32) if source is None else source)


def truncate(ctx, cache=None, lengths=None):
    ctx.pages_truncate(cache or cache_of(ctx), z(N, dtype=I32) if lengths is None else lengths)


def commit(ctx, cache=None, batch=None, accepted=None, path=None, lens_out=None):
    ctx.pages_commit(cache or cache_of(ctx), batch or batch_of(), z(N, dtype=I32) if accepted is None else accepted,
                     path, lens_out)


def accept(ctx, batch=None, ws=None, **kw):
    f = dict(logits=z(R, V, dtype=F32), tokens=z(R, dtype=I32), temperature=z(N, dtype=F32),
             u_accept=z(R, dtype=F32), u_sample=z(N, dtype=F32), accepted=z(N, dtype=I32), path=z(R, dtype=I32),
             token=z(N, dtype=I32), q=None)
    f.update(kw)
    ctx.accept_rows(batch or batch_of(anc=False), **f, ws=ws)


def refused(ctx, f, **kw):
    with pytest.raises(ValueError):
        f(ctx, **kw)
    assert ctx.lib.calls == []


def taken(ctx, f, **kw):
    f(ctx, **kw)
    (name, args), = ctx.lib.calls
    ctx.lib.calls.clear()
    return args


# ------------------------------------------------------------------------- pages and batches
@pytest.mark.parametrize("bad", [
    dict(k=z(LAYERS, PAGES, NKV, 2, 4096, dtype=F32)), dict(v=z(LAYERS, PAGES, NKV, 2, 4096).bfloat16()),
    dict(v=z(LAYERS, PAGES, NKV, 1, 4096)), dict(k=z(LAYERS, PAGES, 2 * NKV, 1, 4096)),
    dict(k=z(LAYERS, PAGES, 2 * NKV, 2, 4096)[:, :, ::2]), dict(k=z(PAGES, NKV, 8192)),
    dict(k=z(LAYERS, PAGES, NKV, 100, 64), v=z(LAYERS, PAGES, NKV, 100, 64)),
    dict(table=z(N, BLOCKS, dtype=I64)), dict(table=z(N * BLOCKS, dtype=I32)),
    dict(table=z(N, 2 * BLOCKS, dtype=I32)[:, ::2]), dict(table=z(BLOCKS, N, dtype=I32).T),
    dict(lens=z(N + 1, dtype=I32)), dict(lens=z(N - 1, dtype=I32)), dict(lens=z(N, dtype=I64)),
    dict(lens=z(2 * N, dtype=I32)[::2]), dict(refs=z(PAGES - 1, dtype=I32)), dict(refs=z(PAGES, dtype=F32)),
    dict(refs=z(2 * PAGES, dtype=I32)[::2])],
    ids=lambda b: " ".join(f"{k}{tuple(t.shape)}{str(t.dtype)[6:]}" for k, t in b.items()))
def test_page_tensors(ctx, bad):
    with pytest.raises(ValueError):
        cache_of(ctx, **bad)


def test_pages_taken(ctx):
    c = cache_of(ctx)
    assert (c.n_layers, c.n_pages, c.n_kv_heads, c.page_tokens, c.n_seqs, c.blocks) == (
        LAYERS, PAGES, NKV, 64, N, BLOCKS)
    f = c._ref._obj
    assert (f.k, f.v, f.table, f.lens, f.refs) == tuple(t.data_ptr() for t in (c.k, c.v, c.table, c.lens, c.refs))
    assert (f.n_layers, f.n_pages, f.n_kv_heads, f.page_tokens, f.n_seqs, f.table_stride) == (
        LAYERS, PAGES, NKV, 64, N, BLOCKS)
    with pytest.raises(ValueError):
        cache_of(ctx_on(0))  # tensors of another device


def test_batch_tensors():
    ok = z(N + 1, dtype=I32)
    for start, anc in ((z(N + 1, dtype=I64), None), (z(N + 1, 1, dtype=I32), None), (z(1, dtype=I32), None),
                       (z(2 * N, dtype=I32)[::2], None), (ok, z(R, dtype=I32)), (ok, z(R - 1, dtype=I64)),
                       (ok, z(2 * R, dtype=I64)[::2])):
        with pytest.raises(ValueError):
            RowBatch(start, R, 4, anc)
    b = RowBatch(ok, R, 4, z(R, dtype=I64))
    assert (b.n_seqs, b._ref._obj.rows, b._ref._obj.max_rows) == (N, R, 4)
    for f in (append, attn, reserve, commit, accept):
        refused(ctx_on(0), f, **(dict(batch=b) if f is accept else dict(batch=b, cache=cache_of(ctx_on(-1)))))


def test_tree_masks():
    assert tree_masks([-1]) == [1]
    assert tree_masks([-1, 0, 0, 1, 2]) == [1, 3, 5, 11, 21]
    chain = tree_masks([i - 1 for i in range(64)])
    assert chain == [(1 << (i + 1)) - 1 for i in range(63)] + [-1]
    assert torch.tensor(chain, dtype=I64)[63] == -1
    for bad in ([0], [-1, 1], [-1, -1], [-1, 2, 0], [i - 1 for i in range(65)]):
        with pytest.raises(ValueError):
            tree_masks(bad)


@pytest.mark.parametrize("f", [append, attn, reserve, fork, truncate, commit])
def test_pages_of_another_device(f):
    refused(ctx_on(0), f, cache=cache_of(ctx_on(-1)))


# -------------------------------------------------------------------------------------- rows
def bad_rows(width, m=R):
    """Tensors that do not hold m rows of `width` fp16 values side by side."""
    return [z(m, width, dtype=F32), z(m, width).bfloat16(), z(m - 1, width), z(m, width - 8),
            z(1, width).expand(m, width), z(width, m).T, z(m, 2 * width)[:, ::2],
            z(m * width).as_strided((m, width), (8, 1)), z(m, 2, width)[:, :, : width // 2]]


@pytest.mark.parametrize("f,name,width,at", [
    (append, "qkv", (NQ + 2 * NKV) * D, 5), (attn, "q", NQ * D, 6), (attn, "out", NQ * D, 8)])
def test_strided_rows(ctx, f, name, width, at):
    for t in bad_rows(width):
        refused(ctx, f, **{name: t})
    for t, stride in ((z(R, width), 0), (z(R + 2, width), width), (z(R, width + 64)[:, 8:8 + width], width + 64),
                      (z(R, width // D, D), 0), (z(R, 2, width)[:, 1], 2 * width)):
        args = taken(ctx, f, **{name: t})
        assert args[at] == t.data_ptr() and args[at + 1] == stride
    args = taken(ctx, f, **{name: z(3, width + 8)[:, :width], "rows": 1})
    assert args[at + 1] == 0


def test_packed_rows_and_norm_weights(ctx):
    for t in bad_rows(NQ * D) + [z(R, NQ * D + 64)[:, :NQ * D]]:
        refused(ctx, append, q=t)
    for w in (z(D, dtype=F32), z(D - 1), z(2 * D)[::2]):
        refused(ctx, append, qw=w)
        refused(ctx, append, kw=w)
    args = taken(ctx, append, qw=z(D))
    assert args[8] is None or not args[8]  # (keys are not normed)


def test_no_rows(ctx):
    """A batch without rows: nothing to append or to attend, whatever the tensors."""
    for f in (append, attn):
        f(ctx, rows=0)
        assert ctx.lib.calls == []


# --------------------------------------------------------------------------- numbers a sequence
def bad_ids(n, dtype=I32):
    other = F32 if dtype is I32 else F16
    return [z(n - 1, dtype=dtype), z(n, dtype=other), z(n, dtype=I64), z(2 * n, dtype=dtype)[::2],
            z(1, dtype=dtype).expand(n)]


@pytest.mark.parametrize("f,name,n", [(reserve, "out", 4 * N), (fork, "source", N), (truncate, "lengths", N),
                                      (commit, "accepted", N), (commit, "path", R), (commit, "lens_out", N)])
def test_bookkeeping(ctx, f, name, n):
    for t in bad_ids(n):
        refused(ctx, f, **{name: t})
    taken(ctx, f, **{name: z(n, dtype=I32)})
    taken(ctx, f, **{name: z(n + 3, dtype=I32)})


def test_commit_defaults(ctx):
    c = cache_of(ctx)
    args = taken(ctx, commit, cache=c)
    assert args[4] is None and args[5] == c.lens.data_ptr()


@pytest.mark.parametrize("name,n,dtype", [
    ("tokens", R, I32), ("temperature", N, F32), ("u_accept", R, F32), ("u_sample", N, F32), ("accepted", N, I32),
    ("path", R, I32), ("token", N, I32)])
def test_acceptance_numbers(ctx, name, n, dtype):
    for t in bad_ids(n, dtype):
        refused(ctx, accept, **{name: t})
    taken(ctx, accept, **{name: z(n + 1, dtype=dtype)})


@pytest.mark.parametrize("name,at", [("logits", 2), ("q", 6)])
def test_acceptance_rows(ctx, name, at):
    for t in (z(R, V), z(R - 1, V, dtype=F32), z(V, R, dtype=F32).T, z(R, 2 * V, dtype=F32)[:, ::2],
              z(1, V, dtype=F32).expand(R, V), z(R * V, dtype=F32), z(R, 1, V, dtype=F32),
              z(R * V, dtype=F32).as_strided((R, V), (8, 1)), z(R, V, dtype=torch.float64)):
        refused(ctx, accept, **{name: t})
    for t, ld in ((z(R, V, dtype=F32), V), (z(R + 3, V, dtype=F32), V), (z(R, V + 6, dtype=F32)[:, 3:3 + V], V + 6)):
        args = taken(ctx, accept, **{name: t})
        assert args[at] == t.data_ptr() and args[at + 1] == ld
    for cols in (V - 1, V + 1):  # as many ids in both
        refused(ctx, accept, q=z(R, cols, dtype=F32))


def test_workspaces(ctx):
    for f in (attn, accept):
        refused(ctx, f, ws=z(8192, dtype=torch.uint8)[::2])
        ws = z(4096, dtype=torch.uint8)
        assert taken(ctx, f, ws=ws)[-2:] == (ws.data_ptr(), 4096)
        assert taken(ctx, f)[-2:] == (None, 0)
