"""Oracle: attention of packed sequences, the paged cache's contents, what tokens receive, eviction.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

Not in the reference; plain numpy in float64 from the definitions.  Pinning
(tests/test_oracle_paged.py): attention against ``oracle.streaming.attention``, an eviction
worked out by hand.
"""
from __future__ import annotations

import math

import numpy as np

from .streaming import attention


def seen_by_frame(n: int, frame: int | None) -> np.ndarray:
    """(n, n) booleans: query i sees the keys below (i // frame + 1) * frame."""
    i = np.arange(n)
    limit = np.full(n, n) if frame is None else (i // frame + 1) * frame
    return i[None] < limit[:, None]


def packed(q, k, v, lens, scale: float, frame: int | None) -> np.ndarray:
    """q (T, H, D), k, v (T, Hk, D): float64 (sum(lens), H, D)."""
    out, at = [], 0
    for n in lens:
        s = slice(at, at + n)
        out.append(attention(q[s], k[s], v[s], scale, seen_by_frame(n, frame)))
        at += n
    return np.concatenate(out) if out else np.zeros((0,) + np.shape(q)[1:])


def received(q, k, scale: float, keep=None) -> np.ndarray:
    """(Hk, Lk): the probabilities that each key gets, over the queries and the heads of its key head."""
    q, k = np.asarray(q, np.float64), np.asarray(k, np.float64)
    n, heads, m, hk = q.shape[0], q.shape[1], k.shape[0], k.shape[1]
    keep = np.ones((n, m), bool) if keep is None else np.broadcast_to(keep, (n, m))
    out = np.zeros((hk, m))
    for h in range(heads):
        for i in range(n):
            on = keep[i]
            if on.any():
                s = k[on, h // (heads // hk)] @ q[i, h] * scale
                p = np.exp(s - s.max())
                out[h // (heads // hk), on] += p / p.sum()
    return out


class Sequence:
    """One sequence of a paged cache: rows[0], rows[1] (capacity, Hk, D) by slot, weights and positions (Hk, capacity)."""

    def __init__(self, capacity: int, heads: int, dim: int):
        self.rows = np.zeros((2, capacity, heads, dim))
        self.weights = np.zeros((heads, capacity))
        self.positions = np.zeros((heads, capacity), np.int64)
        self.len = self.evicted = 0

    def append(self, k, v, start: int | None = None):
        start = self.len if start is None else start
        start = min(start, self.rows.shape[1])
        end = min(start + len(k), self.rows.shape[1])
        for r, x in zip(self.rows, (k, v)):
            r[start:end] = x[:end - start]
        self.weights[:, start:end] = 0
        self.positions[:, start:end] = np.arange(start, end) + self.evicted
        self.len = end

    def evict(self, keep: int, recent: int = 0, first: int = 0):
        if self.len <= keep:
            return
        seen = self.len + self.evicted
        for h in range(len(self.weights)):
            def rank(s):
                p, w = self.positions[h, s], self.weights[h, s]
                if p < first or p >= seen - recent:
                    return (0, 0.0, s)
                return (2, 0.0, s) if math.isnan(w) else (1, -w, s)
            kept = set(sorted(range(self.len), key=rank)[:keep])
            holes = [s for s in range(keep) if s not in kept]
            behind = [s for s in range(keep, self.len) if s in kept]
            for to, frm in zip(holes, behind):
                self.rows[:, to, h] = self.rows[:, frm, h]
                self.weights[h, to] = self.weights[h, frm]
                self.positions[h, to] = self.positions[h, frm]
        self.evicted += self.len - keep
        self.len = keep
