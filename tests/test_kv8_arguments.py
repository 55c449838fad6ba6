"""CPU: tensors that the Python calls of the 8-bit KV cache do not take.  A tensor of another type,
layout, size or device than the call reads would be read or written out of range, so each is a
ValueError before the library is reached.  The library is a recorder here and the device is torch's
"none" (-1), which the CPU tensors have."""
import pytest
import torch

from momij_amd.kv8 import Kv8Cache, KvRing
from momij_amd.ops import Context

NQ, NKV, D, BLOCKS, C, M = 8, 2, 128, 6, 200, 3
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
