"""Oracle: rotary positions of several axes, the 8-bit key / value cache, attention of two lengths.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

Not in the reference; plain numpy in float64 from the definitions.  Pinning
(tests/test_oracle_streaming.py): a quarter turn, the (32, 32) block layout
against ``oracle.rope.rope2d``, scales and codes worked out by hand, attention
against ``oracle.attention.attention_ref``.
"""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np

BLOCK = 64


def rope_pairs(sections, layout: str, base: float = 100.0):
    """[(lo, hi, axis, radians per position)] of every rotated pair."""
    rot, at, out = sum(sections), 0, []
    for axis, n in enumerate(sections):
        for i in range(n // 2):
            if layout == "block":
                out.append((at + i, at + n // 2 + i, axis, base ** (-2.0 * i / n)))
            else:
                j = at // 2 + i
                out.append((j, rot // 2 + j, axis, base ** (-2.0 * j / rot)))
        at += n
    return out


def rope_axes(x, positions, pairs) -> np.ndarray:
    """x (T, H, D), positions (T, axes): float64 result."""
    x = np.asarray(x, np.float64)
    y = x.copy()
    for lo, hi, axis, theta in pairs:
        a = (np.asarray(positions)[:, axis].astype(np.float64) * theta)[:, None]
        y[..., lo] = x[..., lo] * np.cos(a) - x[..., hi] * np.sin(a)
        y[..., hi] = x[..., hi] * np.cos(a) + x[..., lo] * np.sin(a)
    return y


def scale_of(amax: float) -> float:
    """The smallest number of four significant bits >= amax / 127, at least 2^-120; 0 for 0."""
    if amax == 0:
        return 0.0
    need = Fraction(float(amax)) / 127
    step = Fraction(2) ** (math.frexp(float(amax) / 127)[1] - 4)
    return max(float(math.ceil(need / step) * step), 2.0 ** -120)


class Cache:
    """One tensor (keys or values) of one sequence: codes (tokens, H, D), scales (blocks, H)."""

    def __init__(self, capacity: int, heads: int, dim: int):
        self.codes = np.zeros((capacity, heads, dim), np.int64)
        self.scales = np.zeros((capacity // BLOCK, heads))
        self.len = 0

    def append(self, x, start: int | None = None):
        """x (n, H, D)."""
        x = np.asarray(x, np.float64)
        start = self.len if start is None else start
        end = min(start + len(x), len(self.codes))
        for base in range(start // BLOCK * BLOCK, end, BLOCK):
            lo, hi = max(base, start), min(base + BLOCK, end)
            if lo >= hi:
                continue
            new = x[lo - start:hi - start]
            for h in range(x.shape[1]):
                was = self.scales[base // BLOCK, h] if base < start else 0.0
                bad = not np.isfinite(new[:, h]).all()
                s = math.nan if bad or math.isnan(was) else max(scale_of(np.abs(new[:, h]).max()), was)
                if base < start and s > was:
                    self.codes[base:start, h] = np.rint(self.codes[base:start, h] * was / s)
                self.codes[lo:hi, h] = np.rint(new[:, h] / s) if s > 0 else 0
                self.scales[base // BLOCK, h] = s
        self.len = end

    def values(self) -> np.ndarray:
        """(len, H, D)."""
        return (self.codes * np.repeat(self.scales, BLOCK, 0)[..., None])[:self.len]


def attention(q, k, v, scale: float, keep=None) -> np.ndarray:
    """q (Lq, H, D), k and v (Lk, Hk, D), keep (Lk,) or (Lq, Lk) booleans: float64
    (Lq, H, D); a query that keeps no key gives zeros, and what is not kept is not read."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    out = np.zeros(q.shape)
    group = q.shape[1] // k.shape[1]
    keep = np.ones((len(q), len(k)), bool) if keep is None else np.broadcast_to(keep, (len(q), len(k)))
    some = keep.any(0)                       # keys that some query sees
    k, v, keep = k[some], v[some], keep[:, some]
    if not some.any():
        return out
    rows = keep.any(1)
    for h in range(q.shape[1]):
        s = np.where(keep, q[:, h] @ k[:, h // group].T * scale, -np.inf)[rows]
        p = np.exp(s - s.max(1, keepdims=True))
        out[rows, h] = p / p.sum(1, keepdims=True) @ v[:, h // group]
    return out
