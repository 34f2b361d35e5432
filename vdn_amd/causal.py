"""Causal attention over packed prompts: grouped heads, sequences of different lengths.

The companion of window.paper_window_attention for token sequences (a prompt in front of the
block, a causal decoder's prefill): each token sees itself and the tokens before it in its own
sequence. Device work runs in libvdnmi.so; the host prepares a plan of row blocks once per
batch of lengths. What a prompt leaves for later steps goes into the 8-bit cache (kvcache.py).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib

_DTYPES = (torch.bfloat16, torch.float16)
MAX_ROWS = 2 ** 31 - 512   # rows (tokens x query heads of a K/V head) of one sequence


@dataclass(frozen=True, eq=False)
class CausalPlan:
    """Blocks of the packed sequences: `blocks` int32 [n, 4] on the device = (first packed row of
    the sequence, its tokens, first row of the block among the sequence's tokens x heads /
    kv_heads rows, 0), 128 rows each, the blocks with most keys first; `wide_blocks` the same of
    256 rows, or None where they would be slower. `rows` counts the packed rows."""
    lengths: tuple
    heads: int
    kv_heads: int
    rows: int
    blocks: torch.Tensor
    wide_blocks: torch.Tensor | None

    @property
    def device(self):
        return self.blocks.device


def _launch(plan, head_dim):
    """The entry point's block arguments, from the tensors that the plan holds now (a copied or
    unpickled plan has its own), and their device index (-1 off the GPU)."""
    wide = head_dim == 128 and plan.wide_blocks is not None
    blocks = plan.wide_blocks if wide else plan.blocks
    return (blocks.data_ptr(), blocks.shape[0], 256 if wide else 128), blocks.get_device()


# When head dim 128 takes 256-row blocks (8 waves, one workgroup a CU) instead of 128-row ones (two
# of 4 waves): a K/V tile then serves twice the rows, which pays where rows see many keys, and a
# block takes the CU to itself, so that there have to be enough of them. Microseconds of 256 and
# 128 rows, 32 heads and 8 K/V heads: 32768 tokens 7285, 7630; 8192: 485, 485; 4096: 131, 138 (the
# mean row sees 2048 keys); 4 x 2048: 151, 142; 2048: 55, 45; 24 prompts of 77 - 1200 with 56 heads
# 140, 111. 8 heads that share one K/V head: 16384 tokens, 512 blocks: 467, 519; 8192, 256 blocks:
# 186, 160.
WIDE_MEAN_KEYS = 2048
WIDE_LEAST_BLOCKS = 512    # two for each of 256 CUs


def _blocks(lengths, group, block_rows):
    """[nblocks, 4] of all sequences, by falling number of keys (a host tensor)."""
    n = np.array(lengths, dtype=np.int64)
    first = n.cumsum() - n
    count = (n * group + block_rows - 1) // block_rows
    seq = np.repeat(np.arange(len(lengths)), count)
    r0 = (np.arange(seq.size) - (count.cumsum() - count)[seq]) * block_rows
    keys = np.minimum(r0 + block_rows, n[seq] * group)
    blocks = np.zeros((seq.size, 4), dtype=np.int32)
    order = np.argsort(-keys, kind="stable")
    for column, values in enumerate((first[seq], n[seq], r0)):
        blocks[:, column] = values[order]
    return torch.from_numpy(blocks)


def prepare_causal_plan(lengths, heads, kv_heads=None, *, device="cpu"):
    """Plan of sequences of `lengths` tokens (ints >= 0), packed in that order from row 0, for
    `heads` query heads that share `kv_heads` K/V heads (all of their own by default)."""
    kv_heads = heads if kv_heads is None else kv_heads
    lengths = tuple(lengths)
    if any(type(n) is not int or n < 0 for n in lengths):
        raise ValueError("lengths must be non-negative integers")
    if any(type(h) is not int or h <= 0 for h in (heads, kv_heads)) or heads % kv_heads:
        raise ValueError("heads must be a positive multiple of kv_heads")
    group = heads // kv_heads
    if sum(lengths) * group > MAX_ROWS:
        raise ValueError("too many rows for one plan")
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    rows = sum(lengths)
    blocks = _blocks(lengths, group, 128)
    if sum(n * (n + 1) // 2 for n in lengths) >= WIDE_MEAN_KEYS * rows > 0:
        wide = _blocks(lengths, group, 256)
        if wide.shape[0] * kv_heads >= WIDE_LEAST_BLOCKS:
            both = torch.cat((blocks, wide)).to(device)     # one transfer
            return CausalPlan(lengths, heads, kv_heads, rows, both[:blocks.shape[0]],
                              both[blocks.shape[0]:])
    return CausalPlan(lengths, heads, kv_heads, rows, blocks.to(device), None)


def causal_attention(query, key, value, plan: CausalPlan, scale=None, *, return_lse=False,
                     out=None):
    """softmax(scale Q Kᵀ) V over each token's own sequence up to itself.

    query [rows, H, D], key and value [rows, Hkv, D] (BF16 or FP16, D 64, 128 or 256, unit
    channel stride, rows >= plan.rows; any token and head strides that keep 16-byte alignment);
    query head h reads K/V head h // (H / Hkv). Returns [rows, H, D] of the same dtype, scores
    and sums in fp32 (within whose range |V| times 256 times the tokens has to stay), probabilities
    rounded to the activation dtype before the product with V;
    with return_lse also the natural-log sum of exp of the scaled scores, fp32 [rows, H].
    Rows behind the plan's last sequence are zero (LSE -inf); in a caller's `out` they are left
    as they were. `out` may be the query itself; it must not overlap it otherwise, nor key, value or
    itself. Values of tokens that a row does not see never reach it, nonfinite ones included; a
    nonfinite value that it sees makes its channel nonfinite."""
    if torch.is_grad_enabled():
        raise RuntimeError("causal attention is inference-only; use no_grad/inference_mode")
    if not isinstance(plan, CausalPlan):
        raise TypeError("plan must be prepared with prepare_causal_plan")
    if query.ndim != 3:
        raise ValueError("Q/K/V must be [rows, heads, D]")
    rows, heads, d = query.shape
    kv_heads, dtype = plan.kv_heads, query.dtype
    if (heads != plan.heads or key.shape != (rows, kv_heads, d) or value.shape != key.shape
            or rows < plan.rows or d not in (64, 128, 256)):
        raise ValueError("Q/K/V do not match the plan's heads and rows, or D is not 64, 128 or 256")
    q_st, q_sh, q_sd = query.stride()
    k_st, k_sh, k_sd = key.stride()
    v_st, v_sh, v_sd = value.stride()
    if dtype not in _DTYPES or key.dtype is not dtype or value.dtype is not dtype \
            or q_sd != 1 or k_sd != 1 or v_sd != 1:
        raise ValueError("Q/K/V must share BF16 or FP16 and have unit innermost stride")
    index = query.get_device()
    launch, plan_index = _launch(plan, d)
    if index < 0 or key.get_device() != index or value.get_device() != index \
            or plan_index != index:
        raise ValueError("Q/K/V and prepared plan must be on the same CUDA device")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        o_st, o_sh = heads * d, d
        if rows > plan.rows:
            out[plan.rows:].zero_()
    elif (out.shape != query.shape or out.dtype is not dtype or out.device != query.device
          or out.stride(2) != 1 or 0 in out.stride()):
        raise ValueError("out must be a [rows, H, D] view like the queries, unit channel stride, "
                         "no broadcast")
    else:
        _lib.check_attention_out(out, query, key, value)
        o_st, o_sh, _ = out.stride()
    lse = lse_ptr = None
    if return_lse:
        lse = torch.empty((rows, heads), dtype=torch.float32, device=query.device)
        lse_ptr = lse.data_ptr()
        if rows > plan.rows:
            lse[plan.rows:].fill_(-math.inf)
    _lib.call_on(index, "vdn_causal_attention", query.data_ptr(), q_st, q_sh, key.data_ptr(),
                 k_st, k_sh, value.data_ptr(), v_st, v_sh,
                 *launch, kv_heads, heads // kv_heads, d,
                 1 if dtype is torch.float16 else 0, scale, out.data_ptr(), o_st, o_sh, lse_ptr,
                 heads, 1, _lib.raw_stream(index))
    return (out, lse) if return_lse else out
