"""CPU: tensors that the Python calls of the 8-bit KV cache do not take.  A tensor of another type,
layout, size or device than the call reads would be read or written out of range, so each is a
ValueError before the library is reached.  The library is a recorder here and the device is torch's
"none" (-1), which the CPU tensors have."""
import pytest
import torch

from momij_amd.kv8 import Kv8Cache, KvRing
from momij_amd.ops import Context

NQ, NKV, D, BLOCKS, C, M = 10, 2, 128, 6, 200, 3
F16, F32, I32 = torch.float16, torch.float32, torch.int32


class Recorder:
    """Every entry succeeds; what was called with what."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


@pytest.fixture
def ctx():
    c = object.__new__(Context)
    c.lib, c.h, c.device = Recorder(), None, -1
    return c


def cache_of(ctx, nkv=NKV, blocks=BLOCKS):
    c, pages = object.__new__(Kv8Cache), nkv * blocks
    c.ctx, c.n_kv_heads, c.blocks = ctx, nkv, blocks
    c.k_codes, c.v_codes = (z(pages, 8192, dtype=torch.uint8) for _ in range(2))
    c.k_scale, c.v_scale = z(pages, dtype=F32), z(pages, dtype=F32)
    c.k_bounds = z(pages, 2, 128, dtype=torch.int8)
    c.table, c.mass = z(nkv, blocks, dtype=I32), z(nkv, blocks, dtype=F32)
    c._spare = torch.empty_like(c.table), torch.empty_like(c.mass)
    c._bind()
    return c


def cfg(**kw):
    return dict(dict(H=2048, nQ=NQ, nKV=NKV, D=D, rope_dim=64, rope_base=1e6, eps=1e-6, window=0, C=0,
                     gs=64), **kw)


def weights():
    names = ("norm_w", "qkv_w", "qkv_s", "qkv_b", "q_norm_w", "k_norm_w", "o_w", "o_s", "o_b")
    return {n: z(D) for n in names}


def append(ctx, qkv=None, qw=None, kw=None, ring=None, q=None, m=M):
    ctx.qkv_append(cfg(), z(m, (NQ + 2 * NKV) * D) if qkv is None else qkv, z(D) if qw is None else qw,
                   z(D) if kw is None else kw, ring or KvRing(z(NKV, C, D), z(NKV, C, D)), 0, None, m,
                   z(m, NQ * D) if q is None else q)


def attn(ctx, cache=None, ring=None, q=None, out=None, m=M, **kw):
    ctx.kv8_attn(cache or cache_of(ctx), ring or KvRing(z(NKV, C, D), z(NKV, C, D)),
                 z(m, NQ * D) if q is None else q, m, NQ, 4, 256, 260, None,
                 z(m, NQ * D) if out is None else out, **kw)


def seal(ctx, cache=None, ring=None):
    ctx.kv8_seal(cache or cache_of(ctx), ring or KvRing(z(NKV, C, D), z(NKV, C, D)), 0, 1, 0)


def unseal(ctx, cache=None, ring=None):
    ctx.kv8_unseal(cache or cache_of(ctx), 0, 1, ring or KvRing(z(NKV, C, D), z(NKV, C, D)), 0)


def block(ctx, cache=None, ring=None, h=None, m=M, **kw):
    ctx.attn_block_kv8(cfg(), weights(), cache or cache_of(ctx), ring or KvRing(z(NKV, C, D), z(NKV, C, D)),
                       z(m, 2048) if h is None else h, 4, 256, 260, None, m, **kw)


def refused(ctx, f, **kw):
    with pytest.raises(ValueError):
        f(ctx, **kw)
    assert ctx.lib.calls == []


def taken(ctx, f, **kw):
    f(ctx, **kw)
    (name, args), = ctx.lib.calls
    ctx.lib.calls.clear()
    return args


# ------------------------------------------------------------------------------------- rings
def test_ring_tensors():
    for k, v in ((z(NKV, C, D, dtype=F32), z(NKV, C, D, dtype=F32)), (z(NKV, C, D), z(NKV, C, D).bfloat16()),
                 (z(NKV, C, D), z(NKV, C + 1, D)), (z(NKV, C, 64), z(NKV, C, 64)),
                 (z(NKV, 2 * C, D)[:, ::2], z(NKV, C, D)), (z(NKV * C, D), z(NKV * C, D))):
        with pytest.raises(ValueError):
            KvRing(k, v)
    # a capacity beside tensors is theirs
    for k, cap in ((z(NKV, C, D), C + 1), (z(NKV, C, D), C // 2), (z(NKV * C * D), C * NKV + 1),
                   (z(NKV * C * D, dtype=F32), C), (z(2 * NKV * C * D)[::2], C), (z(0), C), (z(NKV * C * D), 0)):
        with pytest.raises(ValueError):
            KvRing(k, k.clone(), capacity=cap)
    with pytest.raises(ValueError):
        KvRing(z(NKV, C, D), z(NKV, C, D), n_kv_heads=NKV + 1)
    r = KvRing(z(NKV * C * D), z(NKV, C, D), capacity=C)
    assert (r.capacity, r.n_kv_heads, r.struct.capacity) == (C, NKV, C)
    r = KvRing(4096, 8192, capacity=7)
    assert (r.capacity, r.n_kv_heads) == (7, None)
    assert KvRing(4096, 8192, capacity=7, n_kv_heads=3).n_kv_heads == 3


@pytest.mark.parametrize("f", [append, attn, seal, unseal, block])
def test_rings_of_other_heads(ctx, f):
    for heads in (1, NKV - 1, NKV + 1, 2 * NKV):
        refused(ctx, f, ring=KvRing(z(heads, C, D), z(heads, C, D)))
        refused(ctx, f, ring=KvRing(4096, 8192, capacity=C, n_kv_heads=heads))
    taken(ctx, f)
    taken(ctx, f, ring=KvRing(4096, 8192, capacity=C))
    taken(ctx, f, ring=KvRing(4096, 8192, capacity=C, n_kv_heads=NKV))


@pytest.mark.parametrize("f", [append, attn, seal, unseal, block])
def test_rings_and_caches_of_another_device(ctx, f):
    cache, ring = cache_of(ctx), KvRing(z(NKV, C, D), z(NKV, C, D))
    other = object.__new__(Context)
    other.lib, other.h, other.device = Recorder(), None, 0
    refused(other, f, ring=ring, **({} if f is append else dict(cache=cache_of(other))))
    if f is not append:
        refused(other, f, cache=cache, ring=KvRing(4096, 8192, capacity=C))


# -------------------------------------------------------------------------------------- rows
def bad_rows(width, m=M):
    """Tensors that do not hold m rows of `width` fp16 values side by side."""
    return [z(m, width, dtype=F32), z(m, width).bfloat16(), z(m - 1, width), z(m, width - 8),
            z(1, width).expand(m, width),          # one row for all: a stride of 0 means packed
            z(width, m).T, z(m, 2 * width)[:, ::2],  # values apart
            z(m * width).as_strided((m, width), (8, 1)),  # rows over each other
            z(m, 2, width)[:, :, : width - 8], z(m, 2, width)[:, :, : width // 2], torch.zeros((), dtype=F16)]


def good_rows(width, m=M):
    """[tensor, stride in halves] (0: packed)"""
    return [(z(m, width), 0), (z(m + 2, width), width), (z(m, width + 64)[:, 8:8 + width], width + 64),
            (z(m, width // 128, 128), 0), (z(m + 1, width // 128, 128), width),
            (z(m, 2, width)[:, 1], 2 * width), (z(1, m, width), 0), (z(1, m, width + 8)[:, :, :width], width + 8)]


@pytest.mark.parametrize("f,name,width,at", [
    (append, "qkv", (NQ + 2 * NKV) * D, 3), (attn, "q", NQ * D, 5), (attn, "out", NQ * D, 14)])
def test_strided_rows(ctx, f, name, width, at):
    """Rows of a stride: the address and the stride come together in the library's arguments."""
    for t in bad_rows(width):
        refused(ctx, f, **{name: t})
    for t, stride in good_rows(width):
        args = taken(ctx, f, **{name: t})
        assert args[at - 1] == t.data_ptr() and args[at] == stride
    # a single row has none: the first of many, a slice, a flat vector, heads by heads
    for t in (z(1, width), z(5, width + 8)[:, :width], z(width), z(width // 128, 128),
              z(1, width // 128, 128), z(1, width).expand(4, width)):
        args = taken(ctx, f, **{name: t, "m": 1})
        assert args[at - 1] == t.data_ptr() and args[at] == 0
    for t in (z(width - 8), z(1, 2 * width)[:, ::2], z(2 * width)[::2], z(width, dtype=F32), z(2, width - 8)):
        refused(ctx, f, **{name: t, "m": 1})


def test_query_rows_of_a_selection(ctx):
    def select(ctx, q, m=M):
        ctx.kv8_select(cache_of(ctx), q, m, NQ, 4, 2, 0, 0, z(m, NKV, 2, dtype=I32))

    for t in bad_rows(NQ * D):
        refused(ctx, select, q=t)
    for t, stride in good_rows(NQ * D):
        args = taken(ctx, select, q=t)
        assert args[3] == t.data_ptr() and args[4] == stride


@pytest.mark.parametrize("f,name,width", [(append, "q", NQ * D), (block, "h", 2048)])
def test_packed_rows(ctx, f, name, width):
    """Rows without a stride in the library's arguments: packed ones only."""
    for t in bad_rows(width) + [z(M, width + 64)[:, :width], z(M, width + 64)]:
        refused(ctx, f, **{name: t})
    for t in (z(M, width), z(M + 1, width), z(M, width // 128, 128), z(M * width), z(M * width // 128, 128)):
        taken(ctx, f, **{name: t})


# ----------------------------------------------------------------- lists, masses, workspaces
def select(ctx, sel=None, m=M, **kw):
    ctx.kv8_select(cache_of(ctx), z(m, NQ * D), m, NQ, 4, 3, 0, 0,
                   z(m, NKV, 3, dtype=I32) if sel is None else sel, **kw)


def listed(ctx, sel, m=M):
    attn(ctx, sel=sel, m=m)


@pytest.mark.parametrize("f", [select, listed])
def test_lists(ctx, f):
    for t in (z(M, NKV, 3, dtype=torch.int64), z(M, NKV, 3), z(M - 1, NKV, 3, dtype=I32),
              z(M, NKV, 6, dtype=I32)[..., :3],
              z(M, NKV, 6, dtype=I32)[..., ::2], z(1, NKV, 3, dtype=I32).expand(M, NKV, 3),
              z(M, 1, 3, dtype=I32).expand(M, NKV, 3), z(NKV, M, 3, dtype=I32).transpose(0, 1),
              z(M, NKV + 1, 3, dtype=I32), z(M, 3, dtype=I32), z(3, dtype=I32), z(NKV, M, 3, dtype=I32)):
        refused(ctx, f, sel=t)
    for t in (z(M, NKV, 3, dtype=I32), z(M + 2, NKV, 3, dtype=I32), z(M * NKV, 3, dtype=I32)):
        taken(ctx, f, sel=t)
    taken(ctx, f, sel=z(1, NKV, 3, dtype=I32), m=1)
    refused(ctx, f, sel=z(1, NKV, 3, dtype=I32), m=2)


def test_lists_of_another_length_than_chosen(ctx):
    for n in (2, 4):
        refused(ctx, select, sel=z(M, NKV, n, dtype=I32))


def bad_masses(t=F32):
    """Not [NKV][BLOCKS] values of type t."""
    return [z(NKV, BLOCKS, dtype=torch.float64), z(NKV, BLOCKS), z(NKV, BLOCKS - 1, dtype=t),
            z(NKV - 1, BLOCKS, dtype=t), z(NKV, BLOCKS + 1, dtype=t)[:, :BLOCKS],
            z(NKV, BLOCKS + 1, dtype=t), z(1, BLOCKS, dtype=t).expand(NKV, BLOCKS),
            z(BLOCKS, NKV, dtype=t).T, z(0, dtype=t)]


@pytest.mark.parametrize("f", [attn, block])
def test_masses(ctx, f):
    good = z(NKV, BLOCKS, dtype=F32)
    for t in bad_masses():
        refused(ctx, f, mass_out=t)
        refused(ctx, f, mass_in=t, mass_out=good)
    taken(ctx, f, mass_out=good)
    taken(ctx, f, mass_in=good, mass_out=z(NKV + 1, BLOCKS, dtype=F32))


def test_eviction(ctx):
    def evict(ctx, mass=z(NKV, BLOCKS, dtype=F32), table=z(NKV, BLOCKS, dtype=I32),
              out=z(NKV, BLOCKS, dtype=F32)):
        ctx.kv8_evict(cache_of(ctx), 4, 2, 0, 0, mass, table, out)

    for t in bad_masses():
        refused(ctx, evict, mass=t)
        refused(ctx, evict, out=t)
    for t in bad_masses(I32):
        refused(ctx, evict, table=t)
    taken(ctx, evict)
    cache = cache_of(ctx)
    table, mass = cache.table, cache.mass
    cache.evict(4, 2)
    assert cache.table is not table and cache.mass is not mass and len(ctx.lib.calls) == 1


@pytest.mark.parametrize("f", [select, attn])
def test_workspaces(ctx, f):
    for t in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 10, dtype=F32)[::2]):
        refused(ctx, f, ws=t)
    for t in (torch.zeros(1 << 10, dtype=torch.uint8), torch.zeros(1 << 8, dtype=F32)):
        args = taken(ctx, f, ws=t)
        assert args[-2:] == (t.data_ptr(), 1 << 10)
    assert taken(ctx, f)[-2:] == (None, 0)


@pytest.mark.parametrize("f,name,width", [(append, "qkv", (NQ + 2 * NKV) * D), (attn, "q", NQ * D),
                                          (attn, "out", NQ * D)])
def test_heads_before_rows(ctx, f, name, width):
    """[heads][M][128] is as large as [M][heads][128] and no rows."""
    for t in (z(width // 128, M, 128), z(width, M), z(M * width // 8, 8), z(1, M * width)):
        refused(ctx, f, **{name: t})


@pytest.mark.parametrize("f,name,width", [(append, "q", NQ * D), (block, "h", 2048)])
def test_heads_before_packed_rows(ctx, f, name, width):
    for t in (z(width // 128, M, 128), z(1, M, width + 8), z(1, M - 1, 2 * width), z(2, M, width)):
        refused(ctx, f, **{name: t})
    for t in (z(1, M, width), z(1, M + 1, width), z(1, M, width // 128, 128)):
        taken(ctx, f, **{name: t})
