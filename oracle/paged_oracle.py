"""CPU oracle of the paged-serving calls (include/llx.h) in plain 64-bit integers -- TEST
INFRASTRUCTURE ONLY.  Row by row and key by key from the definitions, on numpy arrays; the norm,
the rotation, the requantization and the table exponentials are golden_oracle's."""
from __future__ import annotations

import math

import numpy as np

from . import golden_oracle as O

I64 = np.int64


def rows_of(q_start, length, seqs, rows):
    """(row, slot, position) of every row of a launch; behind the last sequence: absent."""
    out = []
    for i in range(len(q_start) - 1):
        slot = int(seqs[i]) if seqs is not None else i
        for r in range(int(q_start[i]), int(q_start[i + 1])):
            if r < rows:
                out.append((r, slot, int(length[slot]) - (int(q_start[i + 1]) - r)))
    return out


def append(q, k, v, k_pages, v_pages, table, length, q_start, cos, sin, q_rq, k_rq, q_norm, k_norm, seqs, out):
    """In place on out, k_pages, v_pages."""
    R, H, D = q.shape
    n_pages, Hkv, P, _ = k_pages.shape
    for r, slot, pos in rows_of(q_start, length, seqs, R):
        page = table[slot, pos // P] if 0 <= pos < table.shape[1] * P else -1
        if not 0 <= pos < len(cos) or not 0 <= page < n_pages:
            out[r] = 0
            continue
        for x, norm, rq, heads, dst in ((q[r], q_norm, q_rq, H, out[r]), (k[r], k_norm, k_rq, Hkv, k_pages[page, :, pos % P])):
            y = O.rmsnorm(x, norm[0], *norm[1:]) if norm is not None else x.astype(I64)
            z = O.rope(y.reshape(1, heads * D), heads, D, cos, sin, pos)
            dst[:] = O.vquant(z, *rq).reshape(heads, D)
        v_pages[page, :, pos % P] = v[r]


def attention(q8, k_pages, v_pages, table, length, q_start, score_rq, out_rq, bits, seqs, max_rows, max_len, out):
    R, H, D = q8.shape
    n_pages, Hkv, P, _ = k_pages.shape
    first = {}
    for i in range(len(q_start) - 1):
        for r in range(int(q_start[i]), int(q_start[i + 1])):
            first[r] = int(q_start[i])
    for r, slot, pos in rows_of(q_start, length, seqs, R):
        if r - first[r] >= max_rows:
            continue
        T = max(0, min(pos + 1, max_len, table.shape[1] * P))
        t = np.arange(T)
        page = table[slot][t // P]
        ok = (page >= 0) & (page < n_pages)
        page, row = page[ok], (t % P)[ok]
        for h in range(H):
            if not len(page):
                out[r, h] = 0
                continue
            kv = h * Hkv // H
            out[r, h] = O.attention_head(q8[r, h], k_pages[page, kv, row], v_pages[page, kv, row], *score_rq, *out_rq, bits)


class Pages:
    """Tables, lengths and counts of a paged cache, and the page copies each call makes."""

    def __init__(self, table, length, refs, P):
        self.table, self.length, self.refs, self.P = table.copy(), length.copy(), refs.copy(), P

    def _slots_fine(self, once, others=()):
        S = len(self.table)
        return all(0 <= s < S for s in (*once, *others)) and len(set(once)) == len(once) and not set(once) & set(others)

    def _release(self, s):
        for j, p in enumerate(self.table[s]):
            if 0 <= p < len(self.refs):
                self.refs[p] -= 1

    def reserve(self, slots, counts):
        """Status code."""
        if not self._slots_fine(slots):
            return 16
        P, code, want = self.P, 0, []
        for s, c in zip(slots, counts):
            n = int(self.length[s])
            if n < 0 or c < 0 or n + c > min(self.table.shape[1] * P, 2 ** 31 - 1):
                code |= 2
                continue
            if c and n % P:
                p = self.table[s][n // P]
                code |= 1 if not 0 <= p < len(self.refs) else 32 if self.refs[p] > 1 else 0
            want += [(s, j) for j in range(-(-n // P), -(-(n + c) // P))]
        if code:
            return code
        free = np.flatnonzero(self.refs <= 0)
        if len(free) < len(want):
            return 8
        for (s, j), p in zip(want, free):
            self.table[s][j] = p
            self.refs[p] = 1
        for s, c in zip(slots, counts):
            self.length[s] += c
        return 0

    def free(self, slots):
        for s in dict.fromkeys(slots):
            if 0 <= s < len(self.table):
                self._release(s)
                self.table[s] = -1
                self.length[s] = 0

    def fork(self, parents, children, share):
        """(status code, [(source page, new page, rows)])"""
        if not self._slots_fine(children, parents):
            return 16, []
        P, keep = self.P, self.refs.copy()
        for p in parents:  # what is to be copied has to be there
            n = max(0, min(int(self.length[p]), self.table.shape[1] * P))
            if any(not 0 <= self.table[p][j] < len(keep) for j in range(n // P if share else 0, -(-n // P))):
                return 1, []
        for c in children:
            self._release(c)
        free = np.flatnonzero(self.refs <= 0)
        sizes = [max(0, min(int(self.length[p]), self.table.shape[1] * P)) for p in parents]
        need = sum(-(-n // P) - (n // P if share else 0) for n in sizes)
        if need > len(free):
            self.refs = keep
            return 8, []
        copies, nxt = [], 0
        for p, c, n in zip(parents, children, sizes):
            row = np.full(self.table.shape[1], -1)
            for j in range(-(-n // P)):
                src = self.table[p][j]
                if share and (j + 1) * P <= n:
                    row[j] = src
                    if 0 <= src < len(self.refs):
                        self.refs[src] += 1
                else:
                    row[j] = free[nxt]
                    self.refs[free[nxt]] = 1
                    if 0 <= src < len(self.refs):
                        copies.append((int(src), int(free[nxt]), min(P, n - j * P)))
                    nxt += 1
            self.table[c] = row
            self.length[c] = n
        return 0, copies

    def compact(self):
        """[(from page, to page)]"""
        used = self.refs > 0
        n = int(used.sum())
        src = [p for p in range(n, len(used)) if used[p]]
        dst = [p for p in range(n) if not used[p]]
        name = np.arange(len(used))
        name[src] = dst
        ok = (self.table >= 0) & (self.table < len(used))
        self.table = np.where(ok, name[np.where(ok, self.table, 0)], self.table)
        refs = np.zeros_like(self.refs)
        refs[name[used]] = self.refs[used]
        self.refs = refs
        return list(zip(src, dst))


POW2 = [round(2.0 ** 31 * 2.0 ** (-j / 1024.0)) for j in range(1024)]


def weight(gap: int, step: int) -> int:
    e = (gap * step) >> 12
    b = POW2[(e >> 10) & 1023]
    return (b - ((b * ((e & 1023) * 2839)) >> 32)) >> (e >> 20)


def sample(row, u, exponent, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row of logits; float settings are float32 values."""
    V = len(row)
    greedy = not temperature > 0
    step = 0 if greedy or math.isinf(temperature) else min(round(1.4426950408889634 * 2.0 ** (32 + exponent) / temperature), 1 << 47)
    top = int(row.max())
    gaps = top - row.astype(I64)
    memo = {}
    w = [memo.setdefault(g, weight(g, step)) if g in memo else memo.setdefault(g, weight(g, step)) for g in gaps.tolist()]
    order = np.lexsort((np.arange(V), gaps)).tolist()
    n = 1 if greedy else V if top_k <= 0 or top_k > V else int(top_k)
    order = order[:n]
    if top_p < 1:
        part = math.floor(max(0.0, top_p) * 2 ** 31) if top_p > 0 else 0
        need = max(1, -(-sum(w[i] for i in order) * part // 2 ** 31))
        got = 0
        for j, i in enumerate(order):
            got += w[i]
            if got >= need:
                order = order[: j + 1]
                break
    least = math.ceil(min(1.0, min_p) * 2 ** 31) if min_p > 0 else 0
    order = [i for i in order if w[i] >= least]
    kept = sorted(order)
    total = sum(w[i] for i in kept)
    target = total * (math.floor(min(max(u, 0.0), 1 - 2.0 ** -31) * 2 ** 31) if u > 0 else 0) >> 31
    run = 0
    for i in kept:
        run += w[i]
        if run > target:
            return i, w[i] / total
    raise AssertionError("the running weight ends above every target")
