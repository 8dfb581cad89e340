"""The text-decoding operators in 64 bits, one row at a time, for the tests.

A cache is held as Python dictionaries {(page, head, line): ...}-like numpy arrays; nothing here calls
the package."""

import math
from decimal import Decimal, localcontext

import numpy as np


def angles(rotary, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """Rad per position of each pair and the magnitude, in 64 bits."""
    i = np.arange(rotary // 2, dtype=np.float64)
    b = base * factor ** (rotary / (rotary - 2)) if scaling == "ntk" else base
    f = 1.0 / b ** (2 * i / rotary)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        # number of the pair that makes n turns within the original length: f_i * original = 2 pi n
        lo, hi = (rotary * math.log(original / (n * 2 * math.pi)) / (2 * math.log(b)) for n in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rotary - 1)
        t = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f * (t / factor + (1 - t)), 0.1 * math.log(factor) + 1
    return f, 1.0


def rotate(x, positions, rotary, layout="half", back=False, **kw):
    """x [tokens, heads, dim] float64; also the sums of magnitudes that errors are relative to."""
    f, mag = angles(rotary, **kw)
    a = np.asarray(positions, dtype=np.float64)[:, None] * f
    c, s = (mag * np.cos(a))[:, None], (mag * np.sin(a))[:, None] * (-1 if back else 1)
    y, size = x.copy(), np.zeros_like(x)
    lo, hi = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if layout == "half" else (
        slice(0, rotary, 2), slice(1, rotary, 2))
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    size[..., lo] = size[..., hi] = mag * (np.abs(x[..., lo]) + np.abs(x[..., hi]))
    return y, size


def turns_of(rotary, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """Turns per position of each pair, to some 45 digits: exp(-2 i ln(base) / rotary) / (2 pi)."""
    with localcontext() as context:
        context.prec = 50
        pi, b, f = _pi(), Decimal(base), Decimal(factor)
        if scaling == "ntk":
            b *= (f.ln() * rotary / (rotary - 2)).exp()
        w = [(b.ln() * -2 * i / rotary).exp() / (2 * pi) for i in range(rotary // 2)]
        if scaling == "linear":
            w = [x / f for x in w]
        if scaling == "yarn":
            lo, hi = (rotary * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rotary - 1)
            t = [min(max((i - lo) / max(Decimal(hi - lo), Decimal("0.001")), 0), 1) for i in range(rotary // 2)]
            w = [x * (y / f + (1 - y)) for x, y in zip(w, t)]
        return w


def _pi():
    """By Machin's formula, 16 arctan(1/5) - 4 arctan(1/239)."""
    def arctan(n):
        x, total, k = Decimal(1) / n, Decimal(0), 0
        while abs(x) > Decimal(10) ** -55:
            total += x / (2 * k + 1) * (-1) ** k
            x, k = x / (n * n), k + 1
        return total

    return 16 * arctan(5) - 4 * arctan(239)


class Cache:
    def __init__(self, k, v, table, counts, weight=None, pos=None):
        self.k, self.v, self.table, self.counts = k, v, table, counts
        self.weight, self.pos = weight, pos
        self.pages, self.heads, self.page, self.dim = k.shape

    def capacity(self):
        return self.table.shape[1] * self.page

    def at(self, b, r):
        """(page, line) of row r, or None for a page that is none."""
        p = int(self.table[b, r // self.page])
        return (p, r % self.page) if 0 <= p < self.pages else None

    def append(self, k, v, cu, weight=None):
        """k, v [tokens, heads, dim]; k already rotated."""
        for b in range(self.table.shape[0]):
            n = int(cu[b + 1] - cu[b])
            for j in range(n):
                r = int(self.counts[0, b]) + j
                where = self.at(b, r) if r < self.capacity() else None
                if where is None:
                    continue
                p, line = where
                self.k[p, :, line], self.v[p, :, line] = k[cu[b] + j], v[cu[b] + j]
                if self.pos is not None:
                    self.pos[p, :, line] = self.counts[1, b] + j
                if self.weight is not None:
                    self.weight[p, :, line] = 0 if weight is None else weight[cu[b] + j]
            self.counts[0, b] = max(self.counts[0, b], min(self.counts[0, b] + n, self.capacity()))
            self.counts[1, b] += n

    def rows(self, b, valid=None):
        """(rows that count, their pages, their lines)."""
        out = []
        for r in range(min(int(self.counts[0, b]), self.capacity())):
            if valid is not None and r < valid.shape[1] and not valid[b, r]:
                continue
            where = self.at(b, r)
            if where is not None:
                out.append((r, *where))
        return np.array(out, dtype=np.int64).reshape(-1, 3).T

    def attend(self, q, scale, valid=None, track=False):
        """out, lse, and for the tolerances: sum of p |v|, the largest sum of |q| |k| of a row, rows."""
        batch, heads, dim = q.shape
        g = heads // self.heads
        out, size = np.zeros(q.shape), np.zeros(q.shape)
        lse, reach = np.full((batch, heads), -np.inf), np.zeros((batch, heads))
        for b in range(batch):
            _, p, line = self.rows(b, valid)
            if p.size == 0:
                continue
            for h in range(self.heads):
                k, v = self.k[p, h, line], self.v[p, h, line]
                hs = slice(h * g, (h + 1) * g)
                s = scale * q[b, hs] @ k.T
                m = s.max(1, keepdims=True)
                e = np.exp(s - m)
                prob = e / e.sum(1, keepdims=True)
                out[b, hs], size[b, hs] = prob @ v, prob @ np.abs(v)
                lse[b, hs] = (m + np.log(e.sum(1, keepdims=True)))[:, 0]
                reach[b, hs] = abs(scale) * (np.abs(q[b, hs]) @ np.abs(k).T).max(1)
                if track:
                    np.add.at(self.weight, (p, h, line), prob.sum(0))
        return out, lse, size, reach

    def evict(self, budget, recent=0, sinks=0):
        for b in range(self.table.shape[0]):
            n = min(int(self.counts[0, b]), self.capacity())
            where = [self.at(b, r) for r in range(n)]
            if n <= budget or None in where:
                continue
            for h in range(self.heads):
                def rank(r):
                    p, line = where[r]
                    pos, w = self.pos[p, h, line], self.weight[p, h, line]
                    if pos >= self.counts[1, b] - recent or pos < sinks:
                        return (2, 0.0, r)
                    return (0, 0.0, r) if np.isnan(w) else (1, float(w), r)

                gone = set(sorted(range(n), key=rank)[: n - budget])
                holes = [r for r in range(budget) if r in gone]
                stay = [r for r in range(budget, n) if r not in gone]
                assert len(holes) == len(stay)
                for dst, src in zip(holes, stay):
                    (pd, ld), (ps, ls) = where[dst], where[src]
                    for x in (self.k, self.v, self.weight, self.pos):
                        x[pd, h, ld] = x[ps, h, ls]
            self.counts[0, b] = budget
