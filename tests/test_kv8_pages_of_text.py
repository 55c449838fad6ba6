"""CPU: the examples of the 8-bit KV cache in the project's pages of text, run over a model of the cache
that knows which positions it holds: every pass attends each position that was not evicted once."""
import glob
import os
import re

import momij_amd.kv8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Ring:
    def __init__(self, k, v):
        self.capacity = 1 << 30


class Cache:
    def __init__(self, ctx, n_kv_heads, blocks):
        self.blocks, self.mass, self.held, self.gone = blocks, object(), {}, set()

    def evict(self, n, keep, n_first=1, n_last=1):
        assert n_first + n_last <= keep <= n <= self.blocks
        out = list(range(n_first, n_first + n - keep))
        for i in out:
            self.gone |= set(self.held[i])
        self.held = dict(enumerate(self.held[i] for i in range(n) if i not in out))


class Calls:
    def __init__(self):
        self.passes = self.sealed = 0

    def attn_block_kv8(self, cfg, weights, cache, ring, h, n, start, L, parents, M, mass_in=None, mass_out=None):
        seen = [p for i in range(n) for p in cache.held[i]] + list(range(start, L + M))
        assert len(seen) == len(set(seen)), "a position is attended twice"
        assert set(seen) | cache.gone == set(range(L + M)), "a position is left out"
        assert mass_in is mass_out is cache.mass
        self.passes += 1

    def kv8_seal(self, cache, ring, pos, count, at):
        assert 0 <= at and at + count <= cache.blocks
        for i in range(count):
            cache.held[at + i] = range(pos + 64 * i, pos + 64 * (i + 1))
        self.sealed += count


def test_examples(monkeypatch):
    monkeypatch.setattr(momij_amd.kv8, "Kv8Cache", Cache)
    monkeypatch.setattr(momij_amd.kv8, "KvRing", Ring)
    found = 0
    for page in glob.glob(os.path.join(ROOT, "*.md")):
        for code in re.findall(r"```python\n(.*?)```", open(page).read(), re.S):
            if "kv8_seal" not in code:
                continue
            found += 1
            ctx = Calls()
            # the names that an example may use: passes of (hidden rows, parents, rows, rows kept)
            names = dict(ctx=ctx, k=None, v=None, cfg=None, weights=None, blocks=40,
                         passes=[(None, None, 9, 1 + i % 9) for i in range(1200)],
                         h=None, parents=None, M=1, n=0, start=0, L=64)
            exec(compile(code, page, "exec"), names)
            assert ctx.passes >= 1000 and ctx.sealed > 60 and len(names["cache"].gone) > 0
    assert found
