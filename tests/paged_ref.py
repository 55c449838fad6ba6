"""The verify step of many requests in plain Python and torch at 64 bits: what the tests of the pages, the
attention over them and the acceptance compare with."""
import math

import torch

from kv8_ref import D, E16, E32, attention  # noqa: F401


def unit_at(tokens):
    """Half of K and of V, in a head's page, of tokens [T] and all 128 dims: two [T, 128]."""
    t = tokens[:, None]
    d = torch.arange(D, device=tokens.device)[None]
    u, t = t // 32 * 4096, t % 32
    return (u + 2048 * (t // 4 % 2) + 512 * (d // 32) + 128 * (d // 8 % 4) + 32 * (t // 8) + 8 * (t % 4) + d % 8,
            u + 512 * (d // 16) + 128 * (t // 8) + 8 * (d % 16) + t % 8)


def _places(cache, seq, tokens):
    page = cache.page_tokens
    pg = cache.table[seq].long()[tokens // page]
    return pg, unit_at(tokens % page)


def rows_of(cache, layer, seq, tokens):
    """K and V [T, n_kv_heads, 128] (float64) of tokens of a sequence; zeros where there is no page."""
    pg, at = _places(cache, seq, tokens)
    there = (pg >= 0) & (pg < cache.n_pages)
    out = []
    for pool, i in zip((cache.k, cache.v), at):
        flat = pool[layer].reshape(cache.n_pages, cache.n_kv_heads, -1)
        x = flat[pg.clamp(0, cache.n_pages - 1)[:, None], :, i].double()  # [T, 128, n_kv_heads]
        out.append(torch.where(there[:, None, None], x, torch.zeros_like(x)).transpose(1, 2))
    return out


def put(cache, layer, seq, tokens, k, v):
    """K and V [T, n_kv_heads, 128] to tokens of a sequence that has pages for them."""
    pg, at = _places(cache, seq, tokens)
    for pool, i, x in zip((cache.k, cache.v), at, (k, v)):
        flat = pool[layer].view(cache.n_pages, cache.n_kv_heads, -1)
        flat[pg[:, None], :, i] = x.half().transpose(1, 2)


def tree(m, rng=None):
    return [-1] + [i - 1 if rng is None else int(rng.integers(max(0, i - 5), i)) for i in range(1, m)]


def ways(parents):
    """Of each row, the rows it sees."""
    out = []
    for r, p in enumerate(parents):
        out.append((out[p] if r else []) + [r])
    return out


def seen(L, sees, window):
    """Tokens that a row sees of a sequence of L committed ones; sees: rows of its own (in any order)."""
    depth = len([a for a in sees[:-1]])
    first = max(0, L + depth - window + 1) if window else 0
    return list(range(first, L)) + [L + a for a in sorted(sees)]


class Book:
    """Tables, lengths and counts of the pages, as the calls' documentation says them."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens, self.refs, self.page = [list(r) for r in table], list(lens), list(refs), page

    def _valid(self, p):
        return 0 <= p < len(self.refs)

    def _drop(self, s, first):
        for j in range(first, len(self.table[s])):
            if self._valid(self.table[s][j]):
                self.refs[self.table[s][j]] -= 1
            self.table[s][j] = -1

    def blocks(self, n):
        return -(-n // self.page)

    def truncate(self, lens):
        for s, n in enumerate(lens):
            if n >= 0:
                self.lens[s] = min(self.lens[s], n)
                self._drop(s, self.blocks(self.lens[s]))

    def fork(self, source):
        n = len(self.lens)

        def goes(s):
            return 0 <= source[s] < n and source[s] != s

        for s in range(n):
            if goes(s) and not goes(source[s]):
                f = source[s]
                self._drop(s, 0)
                self.lens[s] = self.lens[f]
                for j in range(self.blocks(self.lens[s])):
                    p = self.table[f][j]
                    if self._valid(p):
                        self.table[s][j] = p
                        self.refs[p] += 1

    def reserve(self, rows):
        """The out array; copies: (sequence, from, to, committed tokens of the block)."""
        before = list(self.refs)
        free = [p for p, c in enumerate(before) if c == 0]
        total, out, copies = 0, [], []
        for s, m in enumerate(rows):
            L, row = self.lens[s], [0, 0, -1, -1]
            last = (L + m - 1) // self.page
            if m > 0 and last < len(self.table[s]):
                js = range(L // self.page, last + 1)
                need = [j for j in js if not self._valid(self.table[s][j]) or before[self.table[s][j]] != 1]
                total += len(need)
                if total <= len(free) or not need:
                    row[:2] = 1, len(need)
                    for j, p in zip(need, free[total - len(need):total]):
                        o = self.table[s][j]
                        self.table[s][j] = p
                        self.refs[p] += 1
                        if self._valid(o) and before[o] > 1:
                            self.refs[o] -= 1
                            if j == L // self.page and L % self.page:
                                row[2:] = o, p
                                copies.append((s, o, p, L % self.page))
            out.append(row)
        return out, copies

    def named(self):
        """How often each page is named."""
        c = [0] * len(self.refs)
        for row in self.table:
            for p in row:
                if self._valid(p):
                    c[p] += 1
        return c


def accept(logits, parents, tokens, T, u_accept, u_sample, q=None):
    """Of one sequence: drafts accepted, the path, the token; logits [m, V], q [m, V] or None."""
    m, V = logits.shape
    way, refused = [0], []

    def probabilities(r):
        x = logits[r].double().clone()
        x[x.isnan()] = -math.inf
        top = float(x.max())
        if top == -math.inf:
            return torch.zeros_like(x)
        if not T > 1e-5:
            e = torch.zeros_like(x)
            e[int((x == top).nonzero()[0])] = 1.0
        elif top == math.inf:
            e = (x == math.inf).double()
        else:
            e = torch.exp((x - top) / T)
        return e / e.sum()

    while True:
        p = probabilities(way[-1])
        left, rest, refused, go = p.clone(), float(p.sum()), [], None
        for c in range(1, m):
            if parents[c] != way[-1]:
                continue
            y = int(tokens[c])
            px = float(left[y]) if 0 <= y < V else 0.0
            qx = 1.0 if q is None else float(q[way[-1], y]) if 0 <= y < V else 1.0
            if px > 0 and qx > 0 and float(u_accept[c]) * qx * rest <= px:
                go = c
                break
            refused.append(y)
            if q is None and px > 0:
                rest -= px
                left[y] = 0.0
        if go is None:
            break
        way.append(go)
    if float(p.sum()) <= 0:
        return len(way) - 1, way + [-1] * (m - len(way)), -1
    if q is not None and refused:
        y = q[way[-1]].double()
        left = (p - torch.where(y > 0, y, torch.zeros_like(y))).clamp_min(0)
    if float(left.sum()) <= 0:
        left = p
    cum = torch.cumsum(left, 0)
    over = (cum > float(u_sample) * cum[-1]).nonzero()
    token = int(over[0]) if len(over) else int((left > 0).nonzero()[-1])
    return len(way) - 1, way + [-1] * (m - len(way)), token
