"""CPU oracle of what a sequence gives up before its end, and of drafted tokens' verification: by loops, in float64.

TEST INFRASTRUCTURE ONLY.  Nothing in the product (package kiln_b200) imports this file.  A page that was released is -1 in its sequence's list.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle.cache_oracle import BAD_INDEX, NO_ROOM, SHARED, Oracle, rounded

BAD_VALUE = 32


class Steps(Oracle):
    def fork(self, sources):
        rows, lengths = [list(r) for r in self.rows], list(self.lengths)
        for s, source in enumerate(sources):
            for page in rows[source] if source >= 0 else []:
                if page >= 0:
                    self.refs[page] += 1
            for page in rows[s]:
                if page >= 0:
                    self.refs[page] -= 1
            self.rows[s], self.lengths[s] = (list(rows[source]), lengths[source]) if source >= 0 else ([], 0)

    def _cut(self, s, length):
        self.lengths[s] = length
        keep = -(-length // self.P)
        for page in self.rows[s][keep:]:
            if page >= 0:
                self.refs[page] -= 1
        del self.rows[s][keep:]

    def compact(self):
        used = [page for page, n in enumerate(self.refs) if n]
        holes = [page for page in range(len(used)) if not self.refs[page]]
        to = dict(zip([page for page in used if page >= len(used)], holes))
        for page, hole in to.items():
            self.pool[:, :, hole] = self.pool[:, :, page]
            self.refs[hole], self.refs[page] = self.refs[page], 0
        self.rows = [[to.get(page, page) for page in row] for row in self.rows]

    def release(self, window, sinks=0):
        for s, row in enumerate(self.rows):
            for k, page in enumerate(row):
                if all(sinks <= j <= self.lengths[s] - window for j in range(k * self.P, (k + 1) * self.P)):
                    row[k] = -1
                    if page >= 0:
                        self.refs[page] -= 1

    def sees(self, b, s, n, tokens, mask, window, sinks, places):
        """Which keys each of a row's tokens sees: [n, length + n]."""
        length = self.lengths[s]
        shows = np.zeros((n, length + n), bool)
        for i in range(n):
            at = length + (i if places is None else min(max(int(places[b][i]), 0), tokens - 1))
            for j in range(length + n):
                near = window is None or j < sinks or j > at - window
                if j < length:
                    shows[i, j] = near
                elif mask is None:
                    shows[i, j] = j - length <= i and near
                else:
                    shows[i, j] = (mask if mask.ndim == 2 else mask[b])[i, j - length]
        return shows

    def look(self, layer, q, mask=None, counts=None, slots=None, scale=None, window=None, sinks=0, places=None):
        """(out, weight, sizes, lse): as Oracle.attend, and the logarithms of the sums."""
        rows, tokens, heads, dim = q.shape
        q = rounded(q, self.dtype)
        mask = None if mask is None else np.asarray(mask)
        factor = dim ** -0.5 if scale is None else scale
        out, weight, sizes, lse = np.zeros(q.shape), np.zeros(q.shape), np.zeros((*q.shape[:3], 1)), np.full(q.shape[:3], -np.inf)
        group = heads // self.pool.shape[3]
        for b in range(rows):
            s, n = (b if slots is None else slots[b]), (tokens if counts is None else counts[b])
            if n <= 0 or not 0 <= s < len(self.rows):
                continue
            shows = self.sees(b, s, n, tokens, mask, window, sinks, places)
            places_of = [self._place(s, at) for at in range(self.lengths[s] + n)]
            pages, at = np.array([p for p, _ in places_of]), np.array([r for _, r in places_of])
            for h in range(heads):
                keys, values = (self.pool[layer, i][pages, h // group, at] for i in range(2))
                for i in range(n):
                    see = shows[i]
                    if not see.any():
                        continue
                    x = keys[see] @ q[b, i, h] * factor
                    sizes[b, i, h] = (np.abs(keys[see]) @ np.abs(q[b, i, h])).max() * factor
                    p = np.exp(x - x.max())
                    lse[b, i, h] = x.max() + math.log(p.sum())
                    p /= p.sum()
                    out[b, i, h], weight[b, i, h] = p @ values[see], p @ np.abs(values[see])
        return out, weight, sizes, lse

    def weigh(self, layer, q, lse, weights, mask=None, counts=None, slots=None, scale=None):
        """(weights, allowed): the sums, and what float32's arithmetic may be off by.

        A score is off by (D / 8 + 8) 2^-23 of its products' sizes, and by 2^-21 of them where the products are float32's; it, lse and their difference are rounded (and scaled by a
        rounded log2 e) to 2^-22 of their sizes together; the exponential is off by 2^-21, and the sum of R weights by R 2^-23."""
        weights = np.array(weights, np.float64)
        rows, tokens, heads, dim = q.shape
        q, lse = rounded(q, self.dtype), np.asarray(lse, np.float64)
        mask = None if mask is None else np.asarray(mask)
        factor, group, allowed = dim ** -0.5 if scale is None else scale, heads // self.pool.shape[3], np.abs(weights) * 2.0**-23
        for b in range(rows):
            s, n = (b if slots is None else slots[b]), (tokens if counts is None else counts[b])
            shows = self.sees(b, s, n, tokens, mask, None, 0, None)
            places = [self._place(s, at) for at in range(self.lengths[s] + n)]
            pages, at = np.array([p for p, _ in places]), np.array([r for _, r in places])
            for h in range(heads):
                keys = self.pool[layer, 0][pages, h // group, at]
                for i in range(n):
                    if lse[b, i, h] == -np.inf:
                        continue
                    x = keys[shows[i]] @ q[b, i, h] * factor
                    size = np.abs(keys[shows[i]]) @ np.abs(q[b, i, h]) * factor
                    w = np.exp(x - lse[b, i, h])
                    weights[s, :len(pages)][shows[i]] += w
                    wide = size * ((dim / 8 + 8) * 2.0**-23 + (2.0**-21 if self.dtype == torch.float32 else 0.0))
                    allowed[s, :len(pages)][shows[i]] += w * (wide + (np.abs(x) + abs(lse[b, i, h])) * 2.0**-22 + 2.0**-21 + tokens * heads * 2.0**-23)
        return weights, allowed

    def evict(self, weights, keep, recent=0, sinks=0):
        refs = list(self.refs)                 # pages are shared or not as they were before the call
        after = np.zeros_like(weights)
        for s, want in enumerate(keep):
            length = self.lengths[s]
            after[s, :length] = weights[s, :length]
            if want < 0 or want >= length:
                continue
            kept = list(range(min(sinks, want)))
            last = min(recent, want - len(kept))
            middle = range(len(kept), length - last)
            order = sorted(middle, key=lambda j: (0 if math.isnan(weights[s, j]) else 1, 0.0 if math.isnan(weights[s, j]) else -weights[s, j], j))
            kept = sorted(kept + order[:want - len(kept) - last] + list(range(length - last, length)))
            moved = [i for i, j in enumerate(kept) if i != j]
            fault = 0
            if any(self.rows[s][j // self.P] < 0 for j in kept):
                fault |= NO_ROOM
            for k in range(moved[0] // self.P, (want - 1) // self.P + 1) if moved else []:
                fault |= NO_ROOM if self.rows[s][k] < 0 else SHARED if refs[self.rows[s][k]] > 1 else 0
            if fault:
                self.faults |= fault
                continue
            for i in moved:
                (page, row), (from_page, from_row) = self._place(s, i), self._place(s, kept[i])
                self.pool[:, :, page, :, row] = self.pool[:, :, from_page, :, from_row]
            after[s] = 0
            after[s, :want] = weights[s, kept]
            self._cut(s, want)
        return after


def verify(sequences, logits, tokens, uniform, draft=None, parents=None, counts=None, slots=None, temperature=None):
    """(n_accepted, accepted, following, faults), by the rules of kb200_cache_verify."""
    logits = logits.cpu().double().numpy()
    rows, width, vocab = logits.shape
    draft = None if draft is None else draft.cpu().double().numpy()
    tokens, uniform = tokens.cpu().numpy(), uniform.cpu().double().numpy()
    n_accepted, accepted, following, faults, named = [0] * sequences, [[-1] * width for _ in range(sequences)], [-1] * sequences, 0, set()
    for b in range(rows):
        s, n = (b if slots is None else slots[b]), (width if counts is None else counts[b])
        t = 1.0 if temperature is None else float(temperature[b])
        if not 0 <= s < sequences or s in named or not (t >= 0 and math.isfinite(t)) or not 0 <= n <= width:
            faults |= BAD_INDEX
        again = s in named
        named.add(s)
        n = min(max(n, 0), width)
        if not 0 <= s < sequences or again or not (t >= 0 and math.isfinite(t)) or n == 0:
            continue
        parent = [i - 1 if parents is None else int(parents[i] if parents.dim() == 1 else parents[b, i]) for i in range(n)]
        for i in range(1, n):
            if not -1 <= parent[i] < i or not 0 <= tokens[b, i] < vocab:
                faults |= BAD_INDEX
                parent[i] = -1

        def after(i):
            x = logits[b, i]
            if np.isnan(x).any() or x.max() == -np.inf or (t > 0 and x.max() == np.inf):
                return None
            if t == 0:
                return (np.arange(vocab) == np.argmax(x)).astype(float)
            e = np.exp((x - x.max()) / t)
            return e / e.sum()

        path, r, left = [0], after(0), 1.0
        for c in range(1, n):
            if parent[c] != path[-1] or r is None:
                continue
            q, x = None, tokens[b, c]
            if draft is not None and t > 0:
                q = draft[b, path[-1]]
            if uniform[b, c] * (1.0 if q is None else q[x]) * left < r[x]:
                path.append(c)
                r, left = after(c), 1.0
                continue
            rest = np.maximum(r / left - q, 0.0) if q is not None else np.where(np.arange(vocab) == x, 0.0, r)
            if rest.sum() > 0:
                r, left = rest, rest.sum()
        n_accepted[s], accepted[s] = len(path), path + [-1] * (width - len(path))
        if r is None:
            faults |= BAD_VALUE
            continue
        sums = np.cumsum(r)
        over = np.nonzero(sums > uniform[b, 0] * sums[-1])[0]
        following[s] = int(over[0] if len(over) else np.nonzero(r)[0][-1])
    return n_accepted, accepted, following, faults
