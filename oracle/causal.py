"""Causal attention oracle in float64, with a bound on what a 16-bit kernel may differ by.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). torch-CPU.
"""
from __future__ import annotations

import torch


def attention(q, k, v, first, scale):
    """q [m, H, D] over k, v [n, Hkv, D]: query i sees the keys j <= first + i. Returns the output,
    the log-sum-exp [m, H], A = sum_j w_j |v_j|, and the largest sum_c |q_c k_c| scale of a row."""
    group = q.shape[1] // k.shape[1]
    q = q.double().transpose(0, 1)
    k = k.double().repeat_interleave(group, 1).transpose(0, 1)
    v = v.double().repeat_interleave(group, 1).transpose(0, 1)
    i, j = torch.arange(q.shape[1])[:, None], torch.arange(k.shape[1])[None]
    seen = j <= i + first
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -float("inf"))
    lse = torch.logsumexp(s, -1) if k.shape[1] else torch.full(s.shape[:2], -float("inf")).double()
    w = torch.where(seen, torch.exp(s - lse.clamp_min(-1e300)[..., None]), 0.0)
    size = torch.where(seen, q.abs() @ k.abs().transpose(1, 2) * scale, 0.0)
    size = size.amax(-1) if k.shape[1] else torch.zeros_like(lse)
    return ((w @ v).transpose(0, 1), lse.T, (w @ v.abs()).transpose(0, 1), size.T)


def packed(q, k, v, lengths, scale):
    """attention() of each sequence of packed rows, results packed alike."""
    parts, start = [], 0
    for n in lengths:
        rows = slice(start, start + n)
        parts.append(attention(q[rows], k[rows], v[rows], 0, scale))
        start += n
    return tuple(torch.cat(p) for p in zip(*parts))


def bounds(out, mass, size, v, dtype, head_dim, keys):
    """How far a kernel's output and log-sum-exp may be from attention()'s.

    Output: each probability is rounded to `dtype` (half a step of it, relative; fp16 rounds
    those under its normal range, relative to a largest of at least 1, to within 2^-25), the
    output once. A score is an fp32 sum of head_dim products, scaled: its error is at most
    (head_dim + 2) half steps of the sum of their magnitudes, and moves weights and sum by as
    much, relative; the hardware exp2 adds at most 2^-21, and the sums over the keys one half step
    for each addition of a chain: of at most 64 keys in a lane, and of a partial sum per 16 keys.
    """
    half = torch.finfo(dtype).eps / 2
    score = (head_dim + 2) * 2.0 ** -24 * size
    extra = 2.0 ** -21 + (min(keys, 64) + keys / 16 + 4) * 2.0 ** -24
    tiny = keys * 2.0 ** -25 * v.double().abs().max() if dtype == torch.float16 and v.numel() else 0.0
    o = half * (mass + out.abs()) * 1.01 + (2 * score[..., None] + extra) * mass + tiny
    return o + torch.finfo(dtype).tiny, score + extra + 2.0 ** -23 * size + 2.0 ** -23
