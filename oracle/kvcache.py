"""8-bit key/value cache oracle: E4M3 by arithmetic in float64, one power-of-two scale per page,
head and side.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). torch-CPU.
"""
from __future__ import annotations

import math

import torch

LEAST = -100


def nearest(x):
    """float64 -> the nearest E4M3 value (ties to even, largest 448); nonfinite -> NaN."""
    x = x.double()
    finite = torch.isfinite(x)
    y = torch.where(finite, x, 0.0)
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    y = torch.round(y / step) * step
    assert float(y.abs().max() if y.numel() else 0.0) <= 448
    return torch.where(finite, y, math.nan)


def exponent(amax):
    """The least e >= LEAST with amax <= 448 * 2^e, of one number."""
    if amax == 0:
        return LEAST
    m, e = math.frexp(amax / 448)                       # amax / 448 = m 2^e, m in [1/2, 1)
    return max(e - 1 if m == 0.5 else e, LEAST)


class Cache:
    """Values (float64) and exponents of the pages, written as the product's cache is."""

    def __init__(self, pages, kv_heads, page, dim):
        self.values = [torch.zeros(pages, kv_heads, page, dim, dtype=torch.float64) for _ in range(2)]
        self.exponents = [torch.zeros(pages, kv_heads, dtype=torch.int64) for _ in range(2)]
        self.page = page

    def write(self, key, value, table, starts, sizes):
        at = 0
        for i, n in enumerate(sizes):
            for side, x in enumerate((key, value)):
                self._append(side, x[at:at + n].double(), table[i], starts[i])
            at += n

    def _append(self, side, x, pages, place):
        while x.shape[0]:
            inside = place % self.page
            n = min(self.page - inside, x.shape[0])
            p = int(pages[place // self.page])
            for h in range(x.shape[1]):
                new = x[:n, h].clamp(-1.875 * 2.0 ** 127, 1.875 * 2.0 ** 127)
                new = torch.where(torch.isfinite(x[:n, h]), new, math.nan)
                finite = new[torch.isfinite(new)]
                e = exponent(float(finite.abs().max()) if finite.numel() else 0.0)
                if inside:
                    e = max(e, int(self.exponents[side][p, h]))
                    held = self.values[side][p, h, :inside]
                    self.values[side][p, h, :inside] = nearest(held / 2.0 ** e) * 2.0 ** e
                self.exponents[side][p, h] = e
                self.values[side][p, h, inside:inside + n] = nearest(new / 2.0 ** e) * 2.0 ** e
            x, place = x[n:], place + n

    def tokens(self, side, pages, start, stop):
        """[stop - start, heads, dim]"""
        return torch.stack([self.values[side][int(pages[t // self.page]), :, t % self.page]
                            for t in range(start, stop)]) if stop > start else \
            self.values[side][0, :, :0].transpose(0, 1)
