"""The verify step of many requests as its callers hold it: PagedCache (a pool of fp16 pages that all
layers share the numbering of, each sequence's list of them and length) and RowBatch (the rows of a pass
by sequence), over the mj_pages_*, mj_paged_* and mj_accept_rows calls of Context.

A step of a batch in use (row_start int32 [n_seqs + 1], tokens and uniforms on the device):

    cache = PagedCache(ctx, n_seqs, n_pages, n_kv_heads, blocks, n_layers)
    batch = RowBatch(row_start, rows, max_rows, anc)            # anc None: chains
    ctx.pages_reserve(cache, batch, reserved)                   # reserved[:, 0]: who has room; others stay as they are
    for l in range(n_layers):
        ctx.paged_append(cfg, cache, l, batch, qkv, q_norm_w, k_norm_w, q)
        ctx.paged_attn(cache, l, batch, q, n_heads, out, window)
    ctx.accept_rows(batch, logits, tokens, temperature, u_accept, u_sample, accepted, path, token)
    ctx.pages_commit(cache, batch, accepted, path)              # cache.lens advance
    # a request that ends; samples of one prompt that share its pages
    ctx.pages_truncate(cache, lengths)                          # int32 [n_seqs], -1: as it is, 0: freed
    ctx.pages_fork(cache, source)                               # int32 [n_seqs], -1: as it is
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext

import torch

from . import _lib
from .ops import ptr

UNIT = 32  # tokens of a page's units


def tree_masks(parents) -> list[int]:
    """Of each row of a tree (parents[0] = -1, parents[r] < r) the rows that it sees, as RowBatch's anc
    holds them (64-bit masks as signed whole numbers)."""
    out: list[int] = []
    for r, p in enumerate(parents):
        if not (p == -1 if r == 0 else 0 <= p < r) or r > 63:
            raise ValueError(f"parents[{r}] = {p}")
        out.append((out[p] if r else 0) | 1 << r)
    return [m - (1 << 64) if m >> 63 else m for m in out]


class RowBatch:
    """Rows row_start[s] .. row_start[s + 1] - 1 of sequence s (int32 [n_seqs + 1] on the device), at most
    max_rows each, `rows` in all; anc int64 [rows]: the rows of its sequence that a row sees as bits
    (tree_masks; None: chains)."""

    def __init__(self, row_start, rows: int, max_rows: int, anc=None):
        if row_start.dtype != torch.int32 or row_start.dim() != 1 or not row_start.is_contiguous() or (
                row_start.numel() < 2):
            raise ValueError("row_start: contiguous int32 [n_seqs + 1]")
        if anc is not None and (anc.dtype != torch.int64 or not anc.is_contiguous() or anc.numel() < rows or
                                anc.get_device() != row_start.get_device()):
            raise ValueError("anc: contiguous int64 [rows], beside row_start")
        self.row_start, self.anc, self.rows, self.max_rows = row_start, anc, int(rows), int(max_rows)
        self.n_seqs, self.device = row_start.numel() - 1, row_start.get_device()
        self._ref = C.byref(_lib.Batch(ptr(row_start), ptr(anc), self.n_seqs, self.rows, self.max_rows))

    def on(self, device: int):
        """The struct for a call on `device`."""
        if self.device != device:
            raise ValueError(f"a batch on device {self.device} in a call on device {device}")
        return self._ref


class PagedCache:
    """A pool of n_pages pages for n_seqs sequences of at most `blocks` pages each: k and v fp16
    [n_layers][n_pages][n_kv_heads][page_tokens / 32][4096], table int32 [n_seqs][blocks] (-1: none), lens
    int32 [n_seqs], refs int32 [n_pages], served int32 [n_seqs]: whether pages_reserve had room for the
    sequence's rows (1, 0; -1: not known), by which the others are left out of the step.  Views of one pool
    that make a step together share it; who changes the table by hand sets it to -1."""

    def __init__(self, ctx, n_seqs: int, n_pages: int, n_kv_heads: int, blocks: int, n_layers: int = 1,
                 page_tokens: int = 64):
        device = torch.device("cuda", ctx.device)

        def zeros(*shape, dtype=torch.int32):
            return torch.zeros(shape, dtype=dtype, device=device)

        shape = (n_layers, n_pages, n_kv_heads, page_tokens // UNIT, 128 * UNIT)
        k, v = (zeros(*shape, dtype=torch.float16) for _ in range(2))
        table = zeros(n_seqs, blocks).fill_(-1)
        lens, refs, served = zeros(n_seqs), zeros(n_pages), zeros(n_seqs).fill_(-1)
        torch.cuda.synchronize(device)  # they are in place for the context's stream
        self._bind(ctx, k, v, table, lens, refs, served)

    @classmethod
    def over(cls, ctx, k, v, table, lens, refs, served=None):
        """Over tensors that are there already (served None: a new one, not known of any sequence)."""
        self = object.__new__(cls)
        if served is None:
            with torch.cuda.stream(ctx.stream) if lens.is_cuda else nullcontext():
                served = torch.full_like(lens, -1)
        self._bind(ctx, k, v, table, lens, refs, served)
        return self

    def _bind(self, ctx, k, v, table, lens, refs, served):
        if k.dim() < 4 or k.shape != v.shape and k.shape[:3] != v.shape[:3] or k.numel() != v.numel():
            raise ValueError("pages: k and v [n_layers][n_pages][n_kv_heads][page_tokens / 32][4096]")
        self.n_layers, self.n_pages, self.n_kv_heads = (int(x) for x in k.shape[:3])
        heads = self.n_layers * self.n_pages * self.n_kv_heads
        tokens = k.numel() // max(heads * 128, 1)
        shapes = [(k, torch.float16, None), (v, torch.float16, None), (table, torch.int32, 2),
                  (lens, torch.int32, 1), (refs, torch.int32, 1), (served, torch.int32, 1)]
        for t, dtype, dim in shapes:
            if t.dtype != dtype or not t.is_contiguous() or dim not in (None, t.dim()) or (
                    t.get_device() != ctx.device):
                raise ValueError(f"pages: contiguous {dtype} on device {ctx.device}, not {t.dtype} "
                                 f"{tuple(t.shape)} of strides {t.stride()} on {t.device}")
        self.n_seqs, self.blocks = (int(x) for x in table.shape)
        if tokens % UNIT or k.numel() != heads * tokens * 128 or refs.numel() != self.n_pages or (
                lens.numel() != self.n_seqs) or served.numel() != self.n_seqs:
            raise ValueError(f"pages of {tokens} tokens ({k.numel()} halves), {lens.numel()} lengths of {self.n_seqs} sequences, "
                             f"{refs.numel()} counts of {self.n_pages} pages")
        self.ctx, self.device, self.page_tokens = ctx, ctx.device, tokens
        self.k, self.v, self.table, self.lens, self.refs, self.served = k, v, table, lens, refs, served
        self._ref = C.byref(_lib.Pages(self.n_layers, self.n_kv_heads, self.n_pages, tokens, ptr(k), ptr(v),
                                       ptr(table), self.n_seqs, self.blocks, ptr(lens), ptr(refs),
                                       ptr(served)))

    def on(self, device: int):
        """The struct for a call on `device`."""
        if self.device != device:
            raise ValueError(f"pages on device {self.device} in a call on device {device}")
        return self._ref
