"""Mean keys of pages, the selection by them and attention over it, in float64.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). torch-CPU.
"""
from __future__ import annotations

import math

import torch


def to_bf16(x):
    """float64 -> the nearest BF16 value (ties to even, normal range), NaN kept, in float64."""
    finite = torch.isfinite(x)
    y = torch.where(finite, x, 0.0)
    m, e = torch.frexp(y)                                   # y = m 2^e, |m| in [1/2, 1)
    y = torch.ldexp(torch.round(m * 256), e - 8)
    return torch.where(finite, y, x)


def mean(values, n):
    """The first n of a page's keys [kv_heads, page, dim] (float64)."""
    return to_bf16(values[:, :n].sum(1) / n)


def select(q, means, row, length, page, count, first, last):
    """q [Q, H, D], means [pages, kv_heads, D], row: the sequence's page ids. Returns for each query the
    page ids of every K/V head, and the tokens in them."""
    tokens, heads, _ = q.shape
    kv_heads = means.shape[1]
    group = heads // kv_heads
    out = []
    for i in range(tokens):
        sees = max(0, length - tokens + 1 + i)
        have = -(-sees // page)
        ids = [int(p) for p in row[:have]]
        picked = []
        for u in range(kv_heads):
            score = []
            for at, p in enumerate(ids):
                s = (q[i, u * group:(u + 1) * group].double() @ means[p, u].double()).tolist()
                s = max(math.inf if math.isnan(x) else x for x in s)
                score.append((0 if at < first or at >= have - last else 1, -s, at))
            picked.append([ids[at] for at in sorted(t[2] for t in sorted(score)[:count])])
        taken = min(have, count)
        out.append((picked, sees - (have - taken) * page if have else 0))
    return out
