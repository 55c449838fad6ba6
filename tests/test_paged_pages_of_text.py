"""CPU: the example of the verify step of many requests in the project's pages of text and in its module, run
over a model of the calls that knows in which order a step has to make them."""
import glob
import os
import re

import momij_amd.paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
N, LAYERS, STEPS = 3, 4, 20


class Batch:
    def __init__(self, row_start, rows, max_rows, anc=None):
        assert (row_start, rows, max_rows, anc) == ("start", 12, 5, "masks")


class Cache:
    def __init__(self, ctx, n_seqs, n_pages, n_kv_heads, blocks, n_layers=1, page_tokens=64):
        assert (n_seqs, n_pages, n_kv_heads, blocks, n_layers) == (N, 40, 4, 8, LAYERS)


class Calls:
    def __init__(self):
        self.done, self.steps, self.ended = [], 0, []

    def pages_reserve(self, cache, batch, out):
        assert self.done == []
        self.done.append("reserve")

    def paged_append(self, cfg, cache, layer, batch, qkv, qw, kw, q):
        assert self.done[0] == "reserve" and len(self.done) == 1 + 2 * layer and q == "q"
        self.done.append("append")

    def paged_attn(self, cache, layer, batch, q, n_heads, out, window=0, ws=None):
        assert self.done[-1] == "append" and len(self.done) == 2 + 2 * layer and q == "q"
        self.done.append("attn")

    def accept_rows(self, batch, logits, tokens, temperature, ua, us, accepted, path, token, q=None, ws=None):
        assert len(self.done) == 1 + 2 * LAYERS and (accepted, path) == ("accepted", "path")
        self.done.append("accept")

    def pages_commit(self, cache, batch, accepted, path=None, lens_out=None):
        assert self.done[-1] == "accept" and (accepted, path) == ("accepted", "path")
        self.done, self.steps = [], self.steps + 1

    def pages_truncate(self, cache, lengths):
        self.ended.append("truncate")

    def pages_fork(self, cache, source):
        self.ended.append("fork")


def run(code, name, monkeypatch):
    monkeypatch.setattr(momij_amd.paged, "PagedCache", Cache)
    monkeypatch.setattr(momij_amd.paged, "RowBatch", Batch)
    ctx = Calls()
    words = ("q qkv q_norm_w k_norm_w out logits tokens temperature u_accept u_sample accepted path token reserved "
             "lengths source cfg").split()
    names = dict({w: w for w in words}, ctx=ctx, n_seqs=N, n_pages=40, n_kv_heads=4, blocks=8, n_layers=LAYERS,
                 n_heads=16, window=0, row_start="start", rows=12, max_rows=5, anc="masks",
                 project=lambda layer, tokens: "qkv", head=lambda out: "logits",
                 steps=[("tokens", "u_accept", "u_sample")] * STEPS, PagedCache=Cache, RowBatch=Batch)
    exec(compile(code, name, "exec"), names)
    assert ctx.done == [] and ctx.ended == ["truncate", "fork"]
    return ctx.steps


def test_pages(monkeypatch):
    found = [(p, c) for p in glob.glob(os.path.join(ROOT, "*.md"))
             for c in re.findall(r"```python\n(.*?)```", open(p).read(), re.S) if "pages_reserve" in c]
    assert found
    for page, code in found:
        assert run(code, page, monkeypatch) == STEPS


def test_module(monkeypatch):
    code = re.search(r"\n\n((?:    [^\n]*\n)+)", momij_amd.paged.__doc__).group(1)
    assert run(re.sub(r"(?m)^    ", "", code), "paged.py", monkeypatch) == 1
