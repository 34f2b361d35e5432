"""Attention of sequences that share prefixes in the 8-bit cache (kvcache.py): each prefix is read once for
all sequences behind it.

A batch that asks about one document, or several samples of each of several prompts: the prompt's tokens
are in the cache once, in pages that the row of a prefix table names, and each sequence has pages of its own
for its tail. kvcache.cache_attention over tables that repeat the prefix's pages gives the same result,
but reads them again for every sequence.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from functools import lru_cache

import numpy as np
import torch

from . import _lib
from .kvcache import HEAD_DIMS, KVCache, _check_cache, _check_table, _check_vector
from .sparse import _check_query

BLOCK_ROWS = 128   # query rows of a prefix that a workgroup takes
TILE = 64          # tokens of its step
LEAST_TILES = 2    # of a piece, where the prefix has more
FEW_ROWS = 16      # so many rows are taken otherwise: the workgroup's waves divide the tiles, not the rows
FEW_STEP = 4       # its tiles at once
FEW_COST = 0.55    # time of a tile, of that of a block of rows (4.5 us for four with 128 channels, and 2.0 for one)
# The pieces leave an eighth of the card's places to the tails, or half of them where even so the longest
# is shorter than this: the tails then take as long as the pieces. 46 sequences behind 12 prompts of up
# to 4097 tokens: 21.3 us against 23.7, 36 behind 8 of up to 2000, 40 heads: 23.0, 27.4; with 16, 16
# sequences behind 4 prompts of 8000 - 16384: 39.3 against 28.5.
SHORT_TILES = 8
_WORKGROUPS_PER_CU = {64: 2, 128: 2, 256: 1}


@dataclass(frozen=True, eq=False)
class PrefixPlan:
    """Prefixes of `lengths` tokens with `counts` sequences each, and how their attention is cut up:
    `items` int32 [n, 8] on the device, a piece of a prefix for a block of query rows each, and
    `sequences` int32 [batch, 8], where each sequence finds its own (the rows of the C entry point);
    `slot_rows`: query rows of all pieces, each of which leaves a partial result for every K/V head."""
    lengths: tuple
    counts: tuple
    heads: int
    kv_heads: int
    head_dim: int
    tokens: int
    longest: int
    piece_tiles: int
    slot_rows: int
    items: torch.Tensor
    sequences: torch.Tensor

    @property
    def device(self):
        return self.sequences.device

    @property
    def batch(self):
        return self.sequences.shape[0]


def _cut(tiles, step, units, slots):
    """Pieces of each prefix (tiles of tokens, of which a workgroup takes `step` at once, and units that walk
    them): as long ones as fill the slots once."""
    def pieces(most):
        return -(-tiles // (-(-most // step) * step))
    lo, hi = min(LEAST_TILES, int(tiles.max())), int(tiles.max())
    while lo < hi:                                      # the least length whose pieces fit
        mid = (lo + hi) // 2
        if int((pieces(mid) * units).sum()) <= slots:
            hi = mid
        else:
            lo = mid + 1
    return pieces(lo)


def prepare_prefix_plan(lengths, counts, heads, kv_heads, head_dim, *, tokens=1, device):
    """Plan of prefixes of `lengths` tokens (ints >= 0) with `counts` sequences each (ints >= 0, in the
    order of the batch), for `tokens` queries of each sequence of `heads` query heads that share `kv_heads`
    K/V heads of head_dim 64, 128 or 256. Once per composition of the batch; the tails may grow."""
    lengths, counts = tuple(lengths), tuple(counts)
    if len(lengths) != len(counts) or any(type(n) is not int or n < 0 for n in lengths + counts):
        raise ValueError("lengths and counts must be non-negative integers, as many of each")
    if any(type(n) is not int or n <= 0 for n in (heads, kv_heads, tokens)) or heads % kv_heads:
        raise ValueError("heads must be a positive multiple of kv_heads, tokens positive")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be in {HEAD_DIMS}")
    if max(lengths, default=0) > 2 ** 31 - 1024 or sum(counts) * tokens * (heads // kv_heads) > 2 ** 31 - 512:
        raise ValueError("too many tokens or rows for one plan")
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    cus = torch.cuda.get_device_properties(device).multi_processor_count if device.type == "cuda" else 256
    n = np.array(lengths, dtype=np.int64)
    count = np.array(counts, dtype=np.int64)
    first = count.cumsum() - count
    rows = count * tokens * (heads // kv_heads)
    blocks = np.where(n > 0, -(-rows // BLOCK_ROWS), 0)
    tiles = -(-n // TILE)
    step = np.where(rows <= FEW_ROWS, FEW_STEP, 1)
    pieces = np.zeros_like(n)
    if int((blocks * tiles).sum()):
        places = cus * _WORKGROUPS_PER_CU[head_dim]
        for share in (7 / 8, 1 / 2):
            pieces = np.where(blocks > 0, _cut(tiles, step, blocks * kv_heads, int(places * share)), 0)
            if int((-(-tiles // np.maximum(pieces, 1)))[blocks > 0].max()) >= SHORT_TILES:
                break
    made = pieces * blocks
    base = made.cumsum() - made
    if int(made.sum()) * kv_heads >= 2 ** 24 - 2 ** 16:
        raise ValueError("too many rows for one plan")
    in_slots = pieces * rows                            # partial results of a prefix's rows
    slot = in_slots.cumsum() - in_slots
    # a prefix's items, piece by piece; its tiles are spread evenly over the pieces
    p = np.repeat(np.arange(len(lengths)), made)
    at = np.arange(p.size) - base[p]
    items = np.zeros((p.size, 8), dtype=np.int32)
    if p.size:
        piece, block = at // blocks[p], at % blocks[p]
        steps = -(-tiles // step)
        cuts = [np.minimum(steps[p] * at // pieces[p] * step[p], tiles[p]) for at in (piece, piece + 1)]
        for column, values in enumerate((p, first[p], block * BLOCK_ROWS, rows[p], *cuts, n[p],
                                         slot[p] + piece * rows[p])):
            items[:, column] = values
    owner = np.repeat(np.arange(len(lengths)), count)
    sequences = np.zeros((owner.size, 8), dtype=np.int32)
    for column, values in enumerate((first, base, pieces, blocks, n, slot, rows)):
        sequences[:, column] = values[owner]
    both = torch.from_numpy(np.concatenate((items, sequences))).to(device)      # one transfer
    # the longest piece's time, in tiles of a block of rows
    tiles_of_one = int(np.ceil((items[:, 5] - items[:, 4]) * np.where(step[p] > 1, FEW_COST, 1)).max()) if p.size else 0
    return PrefixPlan(lengths, counts, heads, kv_heads, head_dim, tokens, max(lengths, default=0), tiles_of_one,
                      int(in_slots.sum()), both[:p.size], both[p.size:])


def prefix_attention(query, cache: KVCache, prefix_table, plan: PrefixPlan, table, lengths, scale=None, *,
                     return_lse=False, out=None):
    """Softmax attention of each sequence's newest tokens over its prefix and its own tail.

    query [batch, Q, H, D] or [batch, H, D] (Q = 1), BF16 or FP16, rows and `out`'s 16-byte aligned, batch =
    plan.batch and Q = plan.tokens, the sequences of the first prefix in front; prefix_table int32 [prefixes, width] names the pages of each
    prefix in order (unit inner stride), table and lengths the tails' pages and tokens, as
    cache_attention's do: the Q queries' own tokens are the tail's newest. Query i of sequence b sees all
    tokens of its prefix, and the tail's tokens j < lengths[b] - Q + 1 + i: a tail may be empty.

    Output, return_lse, out and faults as in cache_attention; a bad page id of a prefix makes all its
    sequences NaN. The result is that of cache_attention over both parts, to its accuracy."""
    index, args = _check_cache(cache, "prefix_attention")
    if not isinstance(plan, PrefixPlan):
        raise TypeError("plan must be prepared with prepare_prefix_plan")
    batch, tokens, heads, d, q_sb, q_st, q_sh = _check_query(query, cache, index)
    _, kv_heads, page, _ = cache._geometry
    if (batch, tokens, heads, kv_heads, d) != (plan.batch, plan.tokens, plan.heads, plan.kv_heads, plan.head_dim):
        raise ValueError("query and cache do not match the plan's batch, tokens, heads and head_dim")
    items, sequences = plan.items, plan.sequences
    if items.get_device() != index or sequences.get_device() != index:
        raise ValueError("the plan must be on the cache's device")
    prefixes, prefix_width, p_st = _check_table(prefix_table, index)
    if prefixes != len(plan.lengths) or plan.longest > prefix_width * page:
        raise ValueError("prefix_table must name every prefix's pages")
    table_batch, width, t_st = _check_table(table, index)
    _check_vector("lengths", lengths, batch, index)
    if table_batch != batch or width <= 0:
        raise ValueError("table must name at least one page for each sequence of the query")
    if max(width, prefix_width) * page > 2 ** 31 - 1024:
        raise ValueError("the table is too wide")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    dtype = query.dtype
    if out is None:
        out, o_sb, o_st, o_sh = query.new_empty(query.shape), tokens * heads * d, heads * d, d
    elif (out.shape != query.shape or out.dtype is not dtype or out.get_device() != index
          or out.stride(-1) != 1 or 0 in out.stride()):
        raise ValueError("out must be a view like the query, unit channel stride, no broadcast")
    else:
        _lib.check_attention_out(out, query)
        o_sb, o_sh, o_st = out.stride(0), out.stride(-2), out.stride(1) if out.ndim == 4 else 0
    lse = lse_ptr = None
    if return_lse:
        lse = query.new_empty(query.shape[:-1], dtype=torch.float32)
        lse_ptr = lse.data_ptr()
    group = heads // kv_heads
    workspace, nbytes = None, 0
    if batch:
        # from the allocator in stream order: calls on other streams and captured graphs have their own
        nbytes = _workspace_bytes(index, -(-plan.slot_rows // BLOCK_ROWS), batch, width, page, tokens, group, kv_heads, d)
        workspace = query.new_empty(nbytes // 2)
    _lib.call_on(index, "vdn_prefix_attention", query.data_ptr(), q_sb, q_st, q_sh, *args,
                 prefix_table.data_ptr(), p_st, prefix_width, items.data_ptr(), items.shape[0],
                 plan.piece_tiles, sequences.data_ptr(), table.data_ptr(), t_st, batch, width, lengths.data_ptr(),
                 tokens, group,
                 int(dtype is torch.float16), scale, out.data_ptr(), o_sb, o_st, o_sh, lse_ptr,
                 _lib.ptr(workspace), nbytes, _lib.raw_stream(index))
    return (out, lse) if return_lse else out


@lru_cache(maxsize=4096)
def _workspace_bytes(device_index, blocks, batch, width, page, tokens, group, kv_heads, head_dim):
    nbytes = ctypes.c_int64(0)
    _lib.call_on(device_index, "vdn_prefix_attention_workspace", blocks, batch, width, page, tokens, group,
                 kv_heads, head_dim, ctypes.addressof(nbytes))
    return nbytes.value
