"""The KV cache in 8 bits as its callers hold it: KvRing (fp16 rows, position p at slot p %
capacity) and Kv8Cache (a pool of pages and each head's list of them), over the mj_kv8_* calls of
Context.

A layer's context in use:

    cache, ring = Kv8Cache(ctx, n_kv_heads, blocks), KvRing(k, v)
    ctx.qkv_append(cfg, qkv, q_norm_w, k_norm_w, ring, L, parents, M, q)   # a pass's rows
    ctx.kv8_attn(cache, ring, q, M, n_heads, n, start, L, parents, out)    # n blocks, then [start, L)
    # 64 committed positions more than the ring should hold: one more block
    ctx.kv8_seal(cache, ring, start, 1, n); n, start = n + 1, start + 64
    # a long context in part: blocks chosen for every row
    ctx.kv8_select(cache, q, M, n_heads, n, n_sel, 1, 2, sel)
    ctx.kv8_attn(cache, ring, q, M, n_heads, n, start, L, parents, out, sel=sel)
    # a bounded cache (of one block more than `keep`): the blocks that got the least attention, of all
    # rows of the passes that were given the masses, go; their pages are used again
    ctx.kv8_attn(..., mass_in=cache.mass, mass_out=cache.mass)
    cache.evict(n, keep, n_first=1, n_last=4); n = keep
    # a rewind into sealed blocks: back to the ring, their weight forgotten
    n, start = n - 1, start - 64; ctx.kv8_unseal(cache, n, 1, ring, start); cache.mass[:, n:] = 0
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import ptr


class KvRing:
    """K and V rows fp16 [n_kv_heads][capacity][128]: torch tensors (flat ones with the capacity
    given), or device addresses (those of VerifyEngine.kv) with the capacity given and, for the
    calls to check, the heads."""

    def __init__(self, k, v, capacity: int | None = None, n_kv_heads: int | None = None):
        self.k, self.v, self.device = k, v, None
        tensors = [t for t in (k, v) if not isinstance(t, int)]
        if capacity is None:
            if len(tensors) < 2:
                raise ValueError("ring addresses need their capacity")
            if k.dim() != 3:
                raise ValueError("ring tensors: two contiguous fp16 [n_kv_heads][capacity][128]")
            capacity = k.shape[1]
        self.capacity, self.n_kv_heads = int(capacity), n_kv_heads
        for t in tensors:
            row = self.capacity * 128
            heads = t.numel() // row if row > 0 else 0
            if heads < 1 or t.numel() != heads * row or (
                    t.dim() > 1 and t.shape != (heads, self.capacity, 128)) or (
                    t.dtype != torch.float16 or not t.is_contiguous()):
                raise ValueError("ring tensors: two contiguous fp16 [n_kv_heads][capacity][128]")
            if self.n_kv_heads not in (heads, None) or self.device not in (t.get_device(), None):
                raise ValueError("ring tensors: of the same heads on one device")
            self.n_kv_heads, self.device = heads, t.get_device()
        addr = [t if isinstance(t, int) else ptr(t) for t in (k, v)]
        self.struct = _lib.KvRingStruct(addr[0], addr[1], self.capacity)

    def of(self, n_kv_heads: int, device: int) -> _lib.KvRingStruct:
        """The struct for a call of n_kv_heads on `device`: a ring of fewer heads would be read and
        written past its end."""
        if (self.n_kv_heads == n_kv_heads or self.n_kv_heads is None) and (
                self.device == device or self.device is None):
            return self.struct
        raise ValueError(f"a ring of {self.n_kv_heads} heads on device {self.device} in a call of "
                         f"{n_kv_heads} on device {device}")


class Kv8Cache:
    """A pool for `blocks` blocks of each head, head g's pages g * blocks .. at first; `mass`
    [n_kv_heads][blocks] holds the blocks' accumulated attention weight."""

    def __init__(self, ctx, n_kv_heads: int, blocks: int):
        device = torch.device("cuda", ctx.device)

        self.ctx, self.n_kv_heads, self.blocks = ctx, n_kv_heads, blocks
        pages = n_kv_heads * blocks

        def zeros(shape, dtype):
            return torch.zeros(shape, dtype=dtype, device=device)

        self.k_codes, self.v_codes = (zeros((pages, 8192), torch.uint8) for _ in range(2))
        self.k_scale, self.v_scale = (zeros(pages, torch.float32) for _ in range(2))
        self.k_bounds = zeros((pages, 2, 128), torch.int8)
        self.table = torch.arange(pages, dtype=torch.int32, device=device).reshape(n_kv_heads, blocks)
        self.mass = zeros((n_kv_heads, blocks), torch.float32)
        self._spare = torch.empty_like(self.table), torch.empty_like(self.mass)
        torch.cuda.synchronize(device)  # the zeros are in place for the context's stream
        self._bind()

    def _bind(self):
        self.struct = _lib.Kv8(self.n_kv_heads, self.n_kv_heads * self.blocks, ptr(self.k_codes),
                               ptr(self.v_codes), ptr(self.k_scale), ptr(self.v_scale),
                               ptr(self.k_bounds), ptr(self.table), self.blocks)

    def on(self, device: int) -> _lib.Kv8:
        """The struct for a call on `device`."""
        if self.ctx.device != device:
            raise ValueError(f"a cache on device {self.ctx.device} in a call on device {device}")
        return self.struct

    def evict(self, n_blocks: int, keep: int, n_first: int = 1, n_last: int = 1):
        """Down to `keep` blocks a head by `mass`; table and mass change places with their spares
        (a captured graph keeps the ones it was captured with)."""
        table, mass = self._spare
        self.ctx.kv8_evict(self, n_blocks, keep, n_first, n_last, self.mass, table, mass)
        self._spare = self.table, self.mass
        self.table, self.mass = table, mass
        self._bind()
