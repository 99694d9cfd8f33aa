"""CPU oracle of the paged K/V cache: the operations of include/kb200.h by loops over Python lists, values in float64.

TEST INFRASTRUCTURE ONLY.  Nothing in the product (package kiln_b200) imports this file.  The rules are restated from
their definitions: a sequence is a list of pages, a page a block of rows, a holder count a number of lists that name the page.
"""

from __future__ import annotations

import numpy as np
import torch

NO_PAGES, TOO_LONG, BAD_INDEX, NO_ROOM, SHARED = 1, 2, 4, 8, 16


def rounded(x, dtype):
    """float64 values of ``x`` in ``dtype`` (x: float32 or of that type)."""
    return x.detach().cpu().to(dtype).double().numpy()


class Oracle:
    def __init__(self, layers, sequences, max_pages, pages, kv_heads, head_dim, page_tokens, dtype):
        self.max_pages, self.P, self.dtype = max_pages, page_tokens, dtype
        self.pool = np.zeros((layers, 2, pages, kv_heads, page_tokens, head_dim))
        self.rows = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.refs = [0] * pages
        self.faults = 0

    @classmethod
    def of(cls, cache):
        """With the state of a PagedCache."""
        o = cls(cache.layers, cache.sequences, cache.max_pages, cache.pages, cache.kv_heads, cache.head_dim, cache.page_tokens, cache.dtype)
        o.pool = cache.pool.cpu().double().numpy()
        table, held = cache.table.cpu().tolist(), cache.held.cpu().tolist()
        o.rows = [row[:n] for row, n in zip(table, held)]
        o.lengths, o.refs = cache.lengths.cpu().tolist(), cache.refs.cpu().tolist()
        return o

    def table(self):
        return [row + [-1] * (self.max_pages - len(row)) for row in self.rows]

    def fork(self, sources):
        rows, lengths = [list(r) for r in self.rows], list(self.lengths)
        for s, source in enumerate(sources):
            if not -1 <= source < len(rows):
                self.faults |= BAD_INDEX
                continue
            for page in (rows[source] if source >= 0 else []):
                self.refs[page] += 1
            for page in rows[s]:
                self.refs[page] -= 1
            self.rows[s], self.lengths[s] = (list(rows[source]), lengths[source]) if source >= 0 else ([], 0)

    def reserve(self, counts):
        spans = {}
        bad = (BAD_INDEX if min(counts) < 0 else 0)
        for s, c in enumerate(counts):
            if c > 0:
                spans[s] = range(self.lengths[s] // self.P, -(-(self.lengths[s] + c) // self.P))
                bad |= TOO_LONG if spans[s].stop > self.max_pages else 0
        if bad:
            self.faults |= bad
            return
        writers = {}
        for s, span in spans.items():
            for page in self.rows[s][span.start:span.stop]:
                writers.setdefault(page, []).append(s)
        wanted = [(s, k) for s, span in spans.items() for k in span
                  if k >= len(self.rows[s]) or (self.refs[self.rows[s][k]] > 1
                                                and not (len(writers[self.rows[s][k]]) == self.refs[self.rows[s][k]] and writers[self.rows[s][k]][0] == s))]
        free = [page for page, n in enumerate(self.refs) if n == 0]
        if len(wanted) > len(free):
            self.faults |= NO_PAGES
            return
        for (s, k), page in zip(wanted, free):
            self.refs[page] = 1
            if k < len(self.rows[s]):
                old, self.rows[s][k] = self.rows[s][k], page
                self.refs[old] -= 1
                if k == self.lengths[s] // self.P:
                    n = self.lengths[s] % self.P
                    self.pool[:, :, page, :, :n] = self.pool[:, :, old, :, :n]
            else:
                self.rows[s].append(page)

    def _cut(self, s, length):
        self.lengths[s] = length
        keep = -(-length // self.P)
        for page in self.rows[s][keep:]:
            self.refs[page] -= 1
        del self.rows[s][keep:]

    def truncate(self, lengths):
        for s, length in enumerate(lengths):
            if length >= 0:
                self._cut(s, min(length, self.lengths[s]))

    def _place(self, s, at):
        return self.rows[s][at // self.P], at % self.P

    def append(self, layer, k, v, counts=None, slots=None):
        rows, tokens = k.shape[:2]
        k, v = rounded(k, self.dtype), rounded(v, self.dtype)
        seen = set()
        for b in range(rows):
            s, n = (b if slots is None else slots[b]), (tokens if counts is None else counts[b])
            if not 0 <= s < len(self.rows) or s in seen:
                self.faults |= BAD_INDEX
                continue
            seen.add(s)
            if not 0 <= n <= tokens:
                self.faults |= BAD_INDEX
            for i in range(min(max(n, 0), tokens)):
                if (self.lengths[s] + i) // self.P >= len(self.rows[s]):
                    self.faults |= NO_ROOM
                    continue
                page, row = self._place(s, self.lengths[s] + i)
                if self.refs[page] > 1:
                    self.faults |= SHARED
                    continue
                self.pool[layer, 0, page, :, row], self.pool[layer, 1, page, :, row] = k[b, i], v[b, i]

    def accept(self, counts, kept=None):
        refs = list(self.refs)                 # pages are shared or not as they were before the call
        for s, n in enumerate(counts):
            mine = list(range(max(n, 0))) if kept is None else list(kept[s])[:max(n, 0)]
            room = len(self.rows[s]) * self.P - self.lengths[s]
            fault = BAD_INDEX if n < 0 or len(mine) < n or any(b <= a for a, b in zip([-1] + mine, mine)) else 0
            fault |= NO_ROOM if any(x >= room for x in mine) else 0
            if not fault and any(i != x for i, x in enumerate(mine)):
                fault = SHARED if any(refs[self._place(s, self.lengths[s] + i)[0]] > 1 for i in range(n)) else 0
            if fault:
                self.faults |= fault
                continue
            for i, x in enumerate(mine):
                (page, row), (from_page, from_row) = self._place(s, self.lengths[s] + i), self._place(s, self.lengths[s] + x)
                self.pool[:, :, page, :, row] = self.pool[:, :, from_page, :, from_row]
            self._cut(s, self.lengths[s] + n)

    def compact(self):
        used = [page for page, n in enumerate(self.refs) if n]
        holes = [page for page in range(len(used)) if not self.refs[page]]
        to = dict(zip([page for page in used if page >= len(used)], holes))
        for page, hole in to.items():
            self.pool[:, :, hole] = self.pool[:, :, page]
            self.refs[hole], self.refs[page] = self.refs[page], 0
        self.rows = [[to.get(page, page) for page in row] for row in self.rows]

    def attend(self, layer, q, mask=None, counts=None, slots=None, scale=None):
        """(out, weight, sizes): the attention; per element the sum of p |v|, by which a kernel's roundings of p count; per row the
        largest sum of |q k| of a score, by which the roundings of its sum count."""
        rows, tokens, heads, dim = q.shape
        q = rounded(q, self.dtype)
        mask = np.tril(np.ones((tokens, tokens), bool)) if mask is None else mask.cpu().numpy()
        out, weight, sizes = np.zeros(q.shape), np.zeros(q.shape), np.zeros((*q.shape[:3], 1))
        group = heads // self.pool.shape[3]
        for b in range(rows):
            s, n = (b if slots is None else slots[b]), (tokens if counts is None else counts[b])
            if n <= 0 or not 0 <= s < len(self.rows):
                continue
            length = self.lengths[s]
            places = [self._place(s, at) for at in range(length + n)]
            pages, at = np.array([p for p, _ in places]), np.array([r for _, r in places])
            for h in range(heads):
                keys, values = (self.pool[layer, i][pages, h // group, at] for i in range(2))
                for i in range(n):
                    sees = np.concatenate([np.ones(length, bool), (mask if mask.ndim == 2 else mask[b])[i, :n]])
                    if not sees.any():
                        continue
                    factor = dim ** -0.5 if scale is None else scale
                    x = keys[sees] @ q[b, i, h] * factor
                    sizes[b, i, h] = (np.abs(keys[sees]) @ np.abs(q[b, i, h])).max() * factor
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[b, i, h], weight[b, i, h] = p @ values[sees], p @ np.abs(values[sees])
        return out, weight, sizes
