"""What the calls on a cache's pages and on beams do, step by step on the host."""
import math

import numpy as np


def need(tokens, page):
    return (tokens + page - 1) // page


class Cache:
    """Tables, lengths and counts as lists; a page outside the cache or a length that does not fit is a mistake of the test."""

    def __init__(self, pages, page, table, lens):
        self.page, self.table, self.lens = page, [list(map(int, r)) for r in table], [int(n) for n in lens]
        self.refs = [0] * pages
        for row, n in zip(self.table, self.lens):
            for p in row[:need(n, page)]:
                self.refs[p] += 1

    def free(self):
        return [p for p, c in enumerate(self.refs) if c == 0]

    def fork(self, parents, release=True):
        """-> table, lens, moves [(from, to, tokens)], rows that lost their last page's tokens"""
        width = len(self.table[0]) if self.table else 0
        new, lens = [], []
        for p in parents:
            n = need(self.lens[p], self.page) if p >= 0 else 0
            new.append((self.table[p][:n] if n else []) + [-1] * (width - n))
            lens.append(self.lens[p] if p >= 0 else 0)
        for row, n in zip(new, lens):
            for p in row[:need(n, self.page)]:
                self.refs[p] += 1
        if release:
            for row, n in zip(self.table, self.lens):
                for p in row[:need(n, self.page)]:
                    self.refs[p] -= 1
        writers = {}
        for i, n in enumerate(lens):
            if n % self.page:
                writers.setdefault(new[i][n // self.page], []).append(i)
        keep = {w[0] for p, w in writers.items() if self.refs[p] == len(w)}
        free, moves, lost = self.free(), [], []
        for i, n in enumerate(lens):
            if n % self.page == 0 or i in keep:
                continue
            at = n // self.page
            self.refs[new[i][at]] -= 1
            if free:
                to = free.pop(0)
                moves.append((new[i][at], to, n % self.page))
                self.refs[to], new[i][at] = 1, to
            else:
                new[i][at], lens[i] = -1, n - n % self.page
                lost.append(i)
        return new, lens, moves, lost

    def give_back(self, rows):
        for r in rows:
            if r < 0:
                continue
            for j in range(need(self.lens[r], self.page)):
                self.refs[self.table[r][j]] -= 1
                self.table[r][j] = -1
            self.lens[r] = 0

    def extend(self, counts, starts, tokens):
        """-> slots, rows that found no place"""
        slots, without, free = [-1] * tokens, [], self.free()
        wants = []
        for r, c in enumerate(counts):
            after = need(self.lens[r] + c, self.page)
            fits = after <= len(self.table[r])
            wants.append(after - need(self.lens[r], self.page) if fits else 0)
            if not fits:
                without.append(r)
        for r, c in enumerate(counts):
            rank = sum(wants[:r])
            if wants[r] and rank + wants[r] > len(free):
                without.append(r)
            if r in without:
                continue
            before = need(self.lens[r], self.page)
            for j in range(wants[r]):
                self.table[r][before + j] = free[rank + j]
                self.refs[free[rank + j]] = 1
            for i in range(c):
                place = self.lens[r] + i
                slots[starts[r] + i] = self.table[r][place // self.page] * self.page + place % self.page
            self.lens[r] += c
        return slots, without

    def compact(self):
        """-> places, moves [(from, to)]"""
        n = sum(c != 0 for c in self.refs)
        holes = [p for p in range(n) if self.refs[p] == 0]
        places, moves, refs = [-1] * len(self.refs), [], [0] * len(self.refs)
        for p, c in enumerate(self.refs):
            if c:
                places[p] = p if p < n else holes.pop(0)
                if p >= n:
                    moves.append((p, places[p]))
                refs[places[p]] = c
        self.refs = refs
        for row, m in zip(self.table, self.lens):
            row[:need(m, self.page)] = [places[p] for p in row[:need(m, self.page)]]
        return places, moves


def best(logits, scores, k):
    """logits [requests * beams, vocabulary], scores [requests, beams] as numpy arrays -> scores (64 bits), tokens, parents [requests, k]"""
    B, K = scores.shape
    out = np.full((B, k), -np.inf), np.full((B, k), -1, dtype=np.int32), np.full((B, k), -1, dtype=np.int32)
    for b in range(B):
        found = []
        for i in range(K):
            score, x = float(scores[b, i]), logits[b * K + i].astype(np.float64)
            if not math.isfinite(score):
                continue
            x = np.where(np.isnan(x), -np.inf, x)
            top = x.max(initial=-np.inf)
            if top == -np.inf:
                continue
            x = np.where(x == np.inf, 0.0, -np.inf) if top == np.inf else x - top
            p = score + (x - np.log(np.exp(x).sum()))
            # of one beam by the logits: what they differ by may be lost in the sum with the score, even in 64 bits
            for rank, t in enumerate(np.lexsort((np.arange(len(p)), -logits[b * K + i].astype(np.float64), -p))[:k]):
                if p[t] > -np.inf:
                    found.append((-p[t], i, rank, int(t)))
        for place, (p, i, _, t) in enumerate(sorted(found)[:k]):
            out[0][b, place], out[1][b, place], out[2][b, place] = -p, t, b * K + i
    return out
