"""Rotation of queries and keys by their positions, with the RMSNorm of each head in the same pass.

The token-sequence companion of window.paper_qk_rmsnorm_rope, which takes the angles of a frame
grid as full tables: here a token has one position, the angles are made on the device from it
and a plan of frequencies, query and key may have different head counts (grouped heads), and the rounding to the
activation dtype comes once, at the end. What it returns goes into causal.causal_attention,
kvcache.write_cache and the cache's attentions.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from fractions import Fraction

import torch

from . import _lib

HEAD_DIMS = (64, 128, 256)
LAYOUTS = ("half", "interleaved")
SCALINGS = (None, "linear", "base", "parts")
_DTYPES = (torch.bfloat16, torch.float16)
# 2 pi to 50 digits: the angles are exact fractions of a turn
_TURN = Fraction("6.28318530717958647692528676655900576839433879875021")


@dataclass(frozen=True, eq=False)
class RotaryPlan:
    """Frequencies of the rotated channel pairs: `steps` int64 [rotary_dim / 2] on the device, the
    turns that a pair makes from one position to the next, times 2^64 (modulo 2^64)."""
    head_dim: int
    rotary_dim: int
    layout: str
    amplitude: float
    steps: torch.Tensor

    @property
    def device(self):
        return self.steps.device


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original=None,
                       parts=(1.0, 32.0)):
    """(radians per position of each of the rotary_dim / 2 pairs, amplitude).

    f_j = base ** (-2 j / rotary_dim), scaled for contexts `factor` times as long:
      None      not at all (factor 1)
      "linear"  f_j / factor: positions are interpolated
      "base"    base * factor ** (rotary_dim / (rotary_dim - 2)): the slowest pair by factor, the fastest kept
      "parts"   by how often a pair turns within the `original` context: at most parts[0] times,
                f_j / factor; at least parts[1] times, f_j; in between, a mixture that is linear in
                the turns. The amplitude is 0.1 ln(factor) + 1 for it, 1 otherwise."""
    if type(rotary_dim) is not int or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    base, factor = float(base), float(factor)
    if not math.isfinite(base) or base <= 1:
        raise ValueError("base must be finite and above 1")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if not math.isfinite(factor) or factor < 1 or (scaling is None and factor != 1):
        raise ValueError("factor must be finite and at least 1, and 1 without scaling")
    if (scaling == "parts") != (original is not None):
        raise ValueError("original is the trained context of the scaling by parts")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling the base needs more than one pair")
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    steps = [math.pow(base, -2 * j / rotary_dim) for j in range(rotary_dim // 2)]
    if scaling == "linear":
        steps = [f / factor for f in steps]
    if scaling != "parts":
        return steps, 1.0
    low, high = (float(p) for p in parts)
    if not 0 <= low < high < math.inf or not 0 < original < math.inf:
        raise ValueError("parts must rise from 0 on, original must be positive")
    keep = [min(1.0, max(0.0, (original * f / math.tau - low) / (high - low))) for f in steps]
    return [f * (w + (1 - w) / factor) for f, w in zip(steps, keep)], 0.1 * math.log(factor) + 1.0


def prepare_rotary_plan(head_dim, *, rotary_dim=None, base=10000.0, layout="half", scaling=None,
                        factor=1.0, original=None, parts=(1.0, 32.0), amplitude=None, device):
    """The plan of rotate_qk, once per model.

    The first rotary_dim channels (all of head_dim 64, 128 or 256 without it; a multiple of 8) turn in pairs:
    (j, j + rotary_dim / 2) in layout "half", (2 j, 2 j + 1) in "interleaved". base, scaling, factor, original
    and parts as rotary_frequencies; `amplitude` takes the place of its value."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be in {HEAD_DIMS}")
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    if type(rotary_dim) is not int or not 8 <= rotary_dim <= head_dim or rotary_dim % 8:
        raise ValueError("rotary_dim must be a multiple of 8 up to head_dim")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}")
    frequencies, own = rotary_frequencies(rotary_dim, base, scaling=scaling, factor=factor,
                                          original=original, parts=parts)
    amplitude = own if amplitude is None else float(amplitude)
    if not math.isfinite(amplitude):
        raise ValueError("amplitude must be finite")
    turns = [round(Fraction(f) / _TURN * 2 ** 64) % 2 ** 64 for f in frequencies]
    steps = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64,
                         device=device)
    return RotaryPlan(head_dim, rotary_dim, layout, amplitude, steps)


def _check_weight(name, w, dim, dtype, index):
    if w.ndim != 1 or w.shape[0] != dim or w.dtype not in (dtype, torch.float32) or w.get_device() != index \
            or not w.is_contiguous():
        raise ValueError(f"{name} must be contiguous [head_dim] of the activation dtype or FP32, on the "
                         "query's device")


def _check_out(name, out, x, others):
    if out.shape != x.shape or out.dtype is not x.dtype or out.get_device() != x.get_device() \
            or out.stride(-1) != 1:
        raise ValueError(f"out's {name} must be like the input, with unit channel stride")
    if not out.is_contiguous() and _lib.overlaps_itself(out):
        raise ValueError("out must not overlap itself")
    if (out.data_ptr() != x.data_ptr() or out.stride() != x.stride()) and _lib.overlap(out, x) \
            or any(_lib.overlap(out, y) for y in others):
        raise ValueError("out may be query and key themselves, but must not overlap them otherwise")


def rotate_qk(query, key, positions, plan: RotaryPlan, q_weight=None, k_weight=None, eps=1e-6, *, out=None):
    """Turns each head of query [tokens, H, D] and key [tokens, H_kv, D] by its token's position.

    BF16 or FP16, unit channel stride, rows and `out`'s 8-byte aligned; positions int32 or int64 [tokens], any values. With q_weight (k_weight),
    [D] of the activation dtype or FP32, a query (key) head is first divided by the root of its
    mean square plus eps and multiplied by the weight (its squares have to be within fp32's range). All in
    fp32, rounded once. Channels from
    plan.rotary_dim on are not turned; plan.amplitude multiplies the turned ones only.

    Returns two fresh contiguous tensors, or `out`, a pair of views to write to: these may be query and key
    themselves (in place), and must not overlap them, each other or themselves otherwise."""
    if torch.is_grad_enabled():
        raise RuntimeError("rotate_qk is inference-only; use no_grad/inference_mode")
    if not isinstance(plan, RotaryPlan):
        raise TypeError("plan must be a RotaryPlan")
    dtype, index = query.dtype, query.get_device()
    if query.ndim != 3 or key.ndim != 3:
        raise ValueError("query must be [tokens, H, D] and key [tokens, H_kv, D]")
    (tokens, heads, dim), (k_tokens, kv_heads, k_dim) = query.shape, key.shape
    (q_st, q_sh, q_sd), (k_st, k_sh, k_sd) = query.stride(), key.stride()
    if dim != plan.head_dim or k_dim != dim or k_tokens != tokens or heads == 0 or kv_heads == 0:
        raise ValueError("query and key must have the same tokens, at least one head and the plan's D")
    if dtype not in _DTYPES or key.dtype is not dtype or q_sd != 1 or k_sd != 1:
        raise ValueError("query and key must share BF16 or FP16, with unit innermost stride")
    if index < 0:
        raise ValueError("query must be on a CUDA (HIP) device")
    steps = plan.steps
    if key.get_device() != index or steps.get_device() != index or positions.get_device() != index:
        raise ValueError("query, key, positions and the plan must be on one device")
    if positions.ndim != 1 or positions.shape[0] != tokens or not positions.is_contiguous() \
            or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be contiguous int32 or int64 [tokens]")
    q_w = k_w = None
    wide = 0
    if q_weight is not None:
        _check_weight("q_weight", q_weight, dim, dtype, index)
        q_w, wide = q_weight.data_ptr(), int(q_weight.dtype is torch.float32)
    if k_weight is not None:
        _check_weight("k_weight", k_weight, dim, dtype, index)
        k_w, wide = k_weight.data_ptr(), int(k_weight.dtype is torch.float32)
        if q_weight is not None and q_weight.dtype is not k_weight.dtype:
            raise ValueError("q_weight and k_weight must share a dtype")
    eps = float(eps)
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be finite and not negative")
    if steps.numel() * 2 != plan.rotary_dim or steps.dtype is not torch.int64 or not steps.is_contiguous():
        raise ValueError("the plan's steps are not those that it was made with")
    if out is None:
        q_out, k_out = query.new_empty((tokens, heads, dim)), query.new_empty((tokens, kv_heads, dim))
        qo_st, ko_st, qo_sh, ko_sh = heads * dim, kv_heads * dim, dim, dim
    else:
        q_out, k_out = out
        _check_out("query", q_out, query, (key,))
        _check_out("key", k_out, key, (query, q_out))
        (qo_st, qo_sh, _), (ko_st, ko_sh, _) = q_out.stride(), k_out.stride()
    _lib.call_on(index, "vdn_rotary", query.data_ptr(), q_st, q_sh, key.data_ptr(), k_st, k_sh, q_w, k_w, wide,
                 eps, positions.data_ptr(), int(positions.dtype is torch.int64), steps.data_ptr(),
                 plan.rotary_dim, int(plan.layout == "interleaved"), plan.amplitude, tokens, heads, kv_heads, dim,
                 int(dtype is torch.float16), q_out.data_ptr(), qo_st, qo_sh, k_out.data_ptr(), ko_st, ko_sh,
                 _lib.raw_stream(index))
    return q_out, k_out
