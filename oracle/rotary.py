"""Rotation of heads by their positions in float64, with the RMSNorm in front of it.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). torch-CPU.
"""
from __future__ import annotations

import math

import torch


def rotate(x, positions, frequencies, layout="half", amplitude=1.0, weight=None, eps=1e-6):
    """x [tokens, heads, dim] -> (value, what its products add up to without their signs)."""
    y = x.double()
    if weight is not None:
        y = y * weight.double() / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    half = len(frequencies)
    angle = positions.double()[:, None, None] * torch.tensor(frequencies, dtype=torch.float64)
    c, s = amplitude * torch.cos(angle), amplitude * torch.sin(angle)
    first = torch.arange(half) * (1 if layout == "half" else 2)
    second = first + (half if layout == "half" else 1)
    a, b = y[..., first], y[..., second]
    out, size = y.clone(), y.abs()
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    # |cos|, |sin| <= amplitude: an error of the angle moves the product that is zero, too
    size[..., first] = size[..., second] = abs(amplitude) * (a.abs() + b.abs())
    return out, size


def tolerance(value, size, dtype):
    """The output's rounding by half a step, and 32 roundings of fp32 of the products: the sum of squares
    (8 in a lane, 5 across, halved by the root), root, weight and two products make 12, an angle
    that is off by 4 roundings and the sum the rest."""
    half = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
    off = 32 * 2.0 ** -24 * size
    return half * (value.abs() + off) + off + least


def bands(base, dim, factor, original, low, high):
    """Frequencies scaled by how often a pair turns in the original context."""
    out = []
    for j in range(dim // 2):
        f = base ** (-2 * j / dim)
        turns = original * f / (2 * math.pi)
        w = 0.0 if turns <= low else 1.0 if turns >= high else (turns - low) / (high - low)
        out.append((1 - w) * f / factor + w * f)
    return out
