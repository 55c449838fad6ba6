"""Python face of the C ABI over torch device tensors.

torch provides device memory and a stream (plumbing only); every computation runs in
libmomij_hip.so.  A Context owns an mj_ctx bound to its own torch stream; call
`torch.cuda.synchronize()` (or run torch work inside `with torch.cuda.stream(ctx.stream)`)
before handing freshly written tensors to it, and `ctx.sync()` before reading results.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import itemgetter

import torch

from . import _lib
from ._lib import AttnConfig, AttnWeights, LayerWeights, MoeWeights, ModelConfig, MomijError


def ptr(t) -> int | None:
    """Device pointer of a torch tensor (None passes a NULL)."""
    if t is None:
        return None
    return t.data_ptr()


_F16 = torch.float16
_CONFIG = itemgetter("H", "nQ", "nKV", "D", "rope_dim", "rope_base", "eps", "window", "C", "gs")


def row_stride(t, M: int, width: int, device: int, what: str) -> int:
    """Halves between M rows of `width` fp16 values side by side, as the library's calls take it (0:
    one row, or packed ones; hence no row that stands for all M)."""
    if t.dtype is _F16 and t.get_device() == device:
        if t.numel() == M * width and t.size(0) == M and t.is_contiguous():
            return 0
        shape, step = t.shape, t.stride()
        if len(shape) == 2 and shape[0] >= M and shape[1] >= width and step[1] == 1:
            if M <= 1:
                return 0
            if step[0] >= width:
                return step[0]
        if M == 1 and t.numel() >= width and t.is_contiguous() and (
                len(shape) == 1 or width % shape[-1] == 0):  # flat, or head by head
            return 0
        if len(shape) > 2 and shape[0] == 1 and M > 1:  # a batch of one
            return row_stride(t[0], M, width, device, what)
        if len(shape) > 2 and shape[0] >= M and (M == 1 or step[0] >= width):
            if t[0].numel() >= width and t[0].is_contiguous():
                return step[0] if M > 1 else 0
    raise ValueError(f"{what}: {M} rows of {width} fp16 values on device {device}, not {t.dtype} "
                     f"{tuple(t.shape)} of strides {t.stride()} on {t.device}")


def packed(t, dtype, rows: int, width: int, device: int, what: str) -> int:
    """Address of `rows` rows of `width` values of a type without gaps."""
    if t.dtype is dtype and t.get_device() == device and t.numel() >= rows * width and t.is_contiguous():
        step = t.stride(0) if rows > 1 else width
        if step == width or step < width and t.dim() < 3:  # (flat, or head by head)
            return t.data_ptr()
        if rows > 1 and t.dim() > 2 and t.size(0) == 1:  # a batch of one
            return packed(t[0], dtype, rows, width, device, what)
    raise ValueError(f"{what}: {rows} packed rows of {width} {dtype} on device {device}, not {t.dtype} "
                     f"{tuple(t.shape)} of strides {t.stride()} on {t.device}")


class Context:
    def __init__(self, device: int = 0):
        self.lib = _lib.load()
        h = C.c_void_p()
        st = self.lib.mj_init(device, C.byref(h))
        if st != 0:
            raise MomijError(st, f"mj_init(device={device}) failed")
        self.h = h
        self.device = device
        self.stream = torch.cuda.Stream(device=device)
        self.check(self.lib.mj_set_stream(self.h, self.stream.cuda_stream))

    def close(self):
        if self.h:
            self.lib.mj_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self, st: int):
        if st != 0:
            msg = self.lib.mj_last_error(self.h)
            raise MomijError(st, msg.decode() if msg else "")

    def sync(self):
        self.check(self.lib.mj_sync(self.h))

    def set_abort(self, flag: bool):
        self.check(self.lib.mj_set_abort(self.h, int(flag)))

    def set_wait_limit(self, polls: int):
        """Bound of the fused MoE launch's waits for its up product, in re-stagings of a
        down item's act rows."""
        self.check(self.lib.mj_set_wait_limit(self.h, int(polls)))

    # ---------------------------------------------------------------- ops
    def gather_qmm2(self, x, w, scales, biases, inds, y, M, ktop, K, N, gs, lhs_per_expert=False,
                    epilogue=_lib.MJ_EPI_STORE):
        self.check(self.lib.mj_gather_qmm2(self.h, ptr(x), ptr(w), ptr(scales), ptr(biases),
                                           ptr(inds), ptr(y), M, ktop, K, N, gs,
                                           int(lhs_per_expert), epilogue))

    @staticmethod
    def moe_struct(mw: dict) -> MoeWeights:
        return MoeWeights(ptr(mw.get("norm_w")), ptr(mw["router_w"]), ptr(mw["up_gate_w"]),
                          ptr(mw["up_gate_s"]), ptr(mw["up_gate_b"]), ptr(mw["down_w"]),
                          ptr(mw["down_s"]), ptr(mw["down_b"]), mw["E"], mw["top_k"], mw["H"],
                          mw["I"], mw["gs"], mw["eps"], ptr(mw.get("up_gate_alpha")),
                          ptr(mw.get("down_alpha")))

    def moe_block(self, mw: dict, x, y, M, flags=0, inds=None, scores=None):
        st = self.moe_struct(mw)
        self.check(self.lib.mj_moe_block(self.h, C.byref(st), ptr(x), ptr(y), M, flags, ptr(inds),
                                         ptr(scores)))

    def moe_block_noalloc(self, mw: dict, x, y, M, flags=0, inds=None, scores=None):
        """mj_moe_block over the library's static per-GPU scratch (no device allocation)."""
        st = self.moe_struct(mw)
        self.check(self.lib.mj_moe_block_noalloc(self.h, C.byref(st), ptr(x), ptr(y), M, flags,
                                                 ptr(inds), ptr(scores)))

    @staticmethod
    def attn_struct(aw: dict) -> AttnWeights:
        return AttnWeights(ptr(aw["norm_w"]), ptr(aw["qkv_w"]), ptr(aw["qkv_s"]), ptr(aw["qkv_b"]),
                           ptr(aw["q_norm_w"]), ptr(aw["k_norm_w"]), ptr(aw["o_w"]),
                           ptr(aw["o_s"]), ptr(aw["o_b"]))

    @staticmethod
    def attn_config(cfg: dict) -> AttnConfig:
        return AttnConfig(*_CONFIG(cfg))

    def attn_block(self, cfg: dict, aw: dict, h, kcache, vcache, L: int, parents, M: int):
        c = self.attn_config(cfg)
        w = self.attn_struct(aw)
        par = None
        if parents is not None:
            par = (C.c_int32 * M)(*[int(p) for p in parents])
        self.check(self.lib.mj_attn_block(self.h, C.byref(c), C.byref(w), ptr(h), ptr(kcache),
                                          ptr(vcache), L, par, M))

    # ------------------------------------------------- a KV cache in 8 bits (kv8.py)
    @staticmethod
    def _parents(parents, M: int):
        if parents is None:
            return None
        if len(parents) != M:
            raise ValueError(f"{len(parents)} parents of {M} rows")
        return (C.c_int32 * M).from_buffer(array("i", parents))

    def _list(self, sel, M: int, n_kv_heads: int, n_sel: int) -> int:
        if (sel.dim() > 1 and sel.shape[-1] != n_sel) or (sel.dim() == 3 and sel.shape[1] != n_kv_heads):
            raise ValueError(f"sel: {tuple(sel.shape)}, not [{M}][{n_kv_heads}][{n_sel}]")
        return packed(sel, torch.int32, M, n_kv_heads * n_sel, self.device, "sel")

    def _mass(self, mass, cache) -> int | None:
        if mass is None:
            return None
        return packed(mass, torch.float32, cache.n_kv_heads, cache.blocks, self.device, "mass")

    def _space(self, ws) -> tuple:
        if ws is None:
            return None, 0
        if not ws.is_contiguous() or ws.get_device() != self.device:
            raise ValueError(f"ws: contiguous memory on device {self.device}")
        return ws.data_ptr(), ws.numel() * ws.element_size()

    def qkv_append(self, cfg: dict, qkv, q_norm_w, k_norm_w, ring, L: int, parents, M: int, q_out):
        """Queries and keys normed and rotated, keys and values appended to the ring; qkv rows may
        be a slice of wider ones."""
        c, dev = self.attn_config(cfg), self.device
        ld = row_stride(qkv, M, (c.n_heads + 2 * c.n_kv_heads) * 128, dev, "qkv")
        self.check(self.lib.mj_qkv_append(self.h, C.byref(c), qkv.data_ptr(), ld,
                                          ptr(q_norm_w), ptr(k_norm_w),
                                          C.byref(ring.of(c.n_kv_heads, dev)), L,
                                          self._parents(parents, M), M,
                                          packed(q_out, _F16, M, c.n_heads * 128, dev, "q_out")))

    def kv8_seal(self, cache, ring, pos: int, count: int, at: int):
        self.check(self.lib.mj_kv8_seal(self.h, C.byref(cache.on(self.device)),
                                        C.byref(ring.of(cache.n_kv_heads, self.device)), pos, count,
                                        at))

    def kv8_unseal(self, cache, at: int, count: int, ring, pos: int):
        self.check(self.lib.mj_kv8_unseal(self.h, C.byref(cache.on(self.device)), at, count,
                                          C.byref(ring.of(cache.n_kv_heads, self.device)), pos))

    def kv8_select(self, cache, q, M: int, n_heads: int, n_blocks: int, n_sel: int, n_first: int,
                   n_last: int, sel, ws=None):
        self.check(self.lib.mj_kv8_select(self.h, C.byref(cache.on(self.device)), n_heads, ptr(q),
                                          row_stride(q, M, n_heads * 128, self.device, "q"), M,
                                          n_blocks, n_sel, n_first, n_last,
                                          self._list(sel, M, cache.n_kv_heads, n_sel),
                                          *self._space(ws)))

    def kv8_attn(self, cache, ring, q, M: int, n_heads: int, n_blocks: int, start: int, L: int,
                 parents, out, sel=None, mass_in=None, mass_out=None, ws=None):
        """sel int32 [M][n_kv_heads][n_sel] (kv8_select's) or None: every block."""
        dev, width, n_sel, lists = self.device, n_heads * 128, 0, None
        if sel is not None:
            n_sel = sel.shape[-1]
            lists = self._list(sel, M, cache.n_kv_heads, n_sel)
        self.check(self.lib.mj_kv8_attn(self.h, C.byref(cache.on(dev)),
                                        C.byref(ring.of(cache.n_kv_heads, dev)), n_heads, ptr(q),
                                        row_stride(q, M, width, dev, "q"), M, n_blocks, lists, n_sel,
                                        start, L, self._parents(parents, M), ptr(out),
                                        row_stride(out, M, width, dev, "out"),
                                        self._mass(mass_in, cache), self._mass(mass_out, cache),
                                        *self._space(ws)))

    def kv8_evict(self, cache, n_blocks: int, keep: int, n_first: int, n_last: int, mass_in,
                  table_out, mass_out):
        self.check(self.lib.mj_kv8_evict(self.h, C.byref(cache.on(self.device)), n_blocks, keep, n_first,
                                         n_last, self._mass(mass_in, cache),
                                         packed(table_out, torch.int32, cache.n_kv_heads, cache.blocks,
                                                self.device, "table_out"),
                                         self._mass(mass_out, cache)))

    def kv8_workspace(self, n_heads: int, n_kv_heads: int, M: int, n_blocks: int, n_sel: int,
                      ring_rows: int, mass: bool = False) -> int:
        return int(self.lib.mj_kv8_workspace(n_heads, n_kv_heads, M, n_blocks, n_sel, ring_rows,
                                             int(mass)))

    def attn_block_kv8(self, cfg: dict, aw: dict, cache, ring, h, n_blocks: int, start: int, L: int,
                       parents, M: int, n_sel: int = 0, n_first: int = 0, n_last: int = 0,
                       mass_in=None, mass_out=None):
        c = self.attn_config(cfg)
        w = self.attn_struct(aw)
        self.check(self.lib.mj_attn_block_kv8(self.h, C.byref(c), C.byref(w),
                                              C.byref(cache.on(self.device)),
                                              C.byref(ring.of(c.n_kv_heads, self.device)),
                                              packed(h, _F16, M, c.H, self.device, "h"),
                                              n_blocks, n_sel, n_first, n_last, start, L,
                                              self._parents(parents, M), M,
                                              self._mass(mass_in, cache), self._mass(mass_out, cache)))

    # ------------------------------------------- the verify step of many requests (paged.py)
    def _ids(self, t, n: int, what: str, dtype=torch.int32) -> int:
        if t.dtype is dtype and t.get_device() == self.device and t.numel() >= n and t.is_contiguous():
            return t.data_ptr()
        raise ValueError(f"{what}: {n} contiguous {dtype} on device {self.device}, not {t.dtype} "
                         f"{tuple(t.shape)} of strides {t.stride()} on {t.device}")

    def _logits(self, t, rows: int, what: str) -> tuple:
        """Address, row stride and width of fp32 rows [rows][V]."""
        if (t.dtype is torch.float32 and t.get_device() == self.device and t.dim() == 2 and
                t.size(0) >= rows and (t.stride(1) == 1 or t.size(1) == 1) and
                (rows <= 1 or t.stride(0) >= t.size(1))):
            return t.data_ptr(), t.stride(0) if rows > 1 else 0, t.size(1)
        raise ValueError(f"{what}: {rows} rows of fp32 values on device {self.device}, not {t.dtype} "
                         f"{tuple(t.shape)} of strides {t.stride()} on {t.device}")

    def pages_reserve(self, cache, batch, out):
        """Room for the batch's rows; out int32 [n_seqs][4]: served, pages taken, page copied from, to."""
        self.check(self.lib.mj_pages_reserve(self.h, cache.on(self.device), batch.on(self.device),
                                             self._ids(out, 4 * cache.n_seqs, "out")))

    def pages_fork(self, cache, source):
        """source int32 [n_seqs]: the sequence that each becomes a branch of (-1: it stays)."""
        self.check(self.lib.mj_pages_fork(self.h, cache.on(self.device),
                                          self._ids(source, cache.n_seqs, "source")))

    def pages_truncate(self, cache, lengths):
        """lengths int32 [n_seqs]: tokens that a sequence keeps at most (-1: it stays)."""
        self.check(self.lib.mj_pages_truncate(self.h, cache.on(self.device),
                                              self._ids(lengths, cache.n_seqs, "lengths")))

    def pages_commit(self, cache, batch, accepted, path=None, lens_out=None):
        """The accepted rows kept (path None: chains, in place already); lens_out None: cache.lens."""
        lens = cache.lens if lens_out is None else lens_out
        self.check(self.lib.mj_pages_commit(
            self.h, cache.on(self.device), batch.on(self.device),
            self._ids(accepted, cache.n_seqs, "accepted"),
            None if path is None else self._ids(path, batch.rows, "path"),
            self._ids(lens, cache.n_seqs, "lens_out")))

    def paged_append(self, cfg: dict, cache, layer: int, batch, qkv, q_norm_w, k_norm_w, q_out):
        c, dev, M = self.attn_config(cfg), self.device, batch.rows
        if M == 0:
            return
        for w in (q_norm_w, k_norm_w):
            if w is not None:
                packed(w, _F16, 1, 128, dev, "norm weight")
        ld = row_stride(qkv, M, (c.n_heads + 2 * c.n_kv_heads) * 128, dev, "qkv")
        self.check(self.lib.mj_paged_append(self.h, C.byref(c), cache.on(dev), layer, batch.on(dev),
                                            qkv.data_ptr(), ld, ptr(q_norm_w), ptr(k_norm_w),
                                            packed(q_out, _F16, M, c.n_heads * 128, dev, "q_out")))

    def paged_attn(self, cache, layer: int, batch, q, n_heads: int, out, window: int = 0, ws=None):
        dev, M, width = self.device, batch.rows, n_heads * 128
        if M == 0:
            return
        self.check(self.lib.mj_paged_attn(self.h, cache.on(dev), layer, batch.on(dev), n_heads, window,
                                          q.data_ptr(), row_stride(q, M, width, dev, "q"), out.data_ptr(),
                                          row_stride(out, M, width, dev, "out"), *self._space(ws)))

    def paged_workspace(self, n_heads: int, n_kv_heads: int, max_rows: int) -> int:
        return int(self.lib.mj_paged_workspace(n_heads, n_kv_heads, max_rows))

    def accept_rows(self, batch, logits, tokens, temperature, u_accept, u_sample, accepted, path, token,
                    q=None, ws=None):
        """Drafts of a batch checked from given random numbers; q fp32 [rows][V]: the distributions that
        the drafts below a row were drawn from (None: drafts that are certain)."""
        R, n, f32 = batch.rows, batch.n_seqs, torch.float32
        x, ld, V = self._logits(logits, R, "logits")
        y, ldq, Vq = (None, 0, V) if q is None else self._logits(q, R, "q")
        if Vq != V:
            raise ValueError(f"q: {Vq} ids, the logits: {V}")
        self.check(self.lib.mj_accept_rows(
            self.h, batch.on(self.device), x, ld, V, self._ids(tokens, R, "tokens"), y, ldq,
            self._ids(temperature, n, "temperature", f32), self._ids(u_accept, R, "u_accept", f32),
            self._ids(u_sample, n, "u_sample", f32), self._ids(accepted, n, "accepted"),
            self._ids(path, R, "path"), self._ids(token, n, "token"), *self._space(ws)))

    def accept_workspace(self, n_seqs: int, rows: int, V: int) -> int:
        return int(self.lib.mj_accept_workspace(n_seqs, rows, V))

    def lm_head_verify(self, x, w, M, K, V, out_argmax, out_max=None, out_logits=None,
                       banned=None, n_banned=0, temperature=1.0, out_lse=None):
        self.check(self.lib.mj_lm_head_verify(self.h, ptr(x), ptr(w), M, K, V, ptr(banned),
                                              n_banned, float(temperature), ptr(out_argmax),
                                              ptr(out_max), ptr(out_lse), ptr(out_logits)))

    def lm_head_verify_q4(self, x, w, scales, biases, M, K, V, out_argmax, out_max=None,
                          out_logits=None, banned=None, n_banned=0, group_size=64,
                          temperature=1.0, out_lse=None):
        self.check(self.lib.mj_lm_head_verify_q4(self.h, ptr(x), ptr(w), ptr(scales),
                                                 ptr(biases), M, K, V, group_size, ptr(banned),
                                                 n_banned, float(temperature), ptr(out_argmax),
                                                 ptr(out_max), ptr(out_lse), ptr(out_logits)))

    def accept_greedy(self, tokens, parents, argmax, n_rows, out):
        par = None
        if parents is not None:
            par = (C.c_int32 * n_rows)(*[int(p) for p in parents])
        self.check(self.lib.mj_accept_greedy(self.h, ptr(tokens), par, ptr(argmax), n_rows,
                                             ptr(out)))

    def accept_sampled(self, logits, rows, V, draft, temperature, q_mode, seed, counter, out,
                       q_point=None):
        self.check(self.lib.mj_accept_sampled(self.h, ptr(logits), rows, V, ptr(draft),
                                              temperature, q_mode, ptr(q_point), seed, counter,
                                              ptr(out)))

    def accept_sampled_ex(self, logits, rows, V, draft, q_mode, seed, counter, out,
                          temperature, top_p=1.0, rep=1.0, pres=0.0, freq=0.0, hist=None,
                          q_point=None):
        """mj_accept_sampled_ex: LogitsProcessor options; hist {token: count}."""
        sp, keep = _lib.sampling(temperature, top_p, rep, pres, freq, hist)
        self.check(self.lib.mj_accept_sampled_ex(self.h, ptr(logits), rows, V, ptr(draft),
                                                 C.byref(sp), q_mode, ptr(q_point), seed,
                                                 counter, ptr(out)))

    def selftest_mfma(self, A, B, D):
        self.check(self.lib.mj_selftest_mfma(self.h, ptr(A), ptr(B), ptr(D)))
