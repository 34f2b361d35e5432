"""The 8-bit key/value cache: pages of E4M3 codes with one E8M0 scale per page, head and side.

The block format is that of the MXFP8 operands (mxfp8.py) with another block: a page of one
sequence's tokens and one K/V head shares a power-of-two scale 2^e, the least e >= -100 with
max |x| <= 448 * 2^e over the page's finite values. K codes are [pages, kv_heads, page, D]; V
codes [pages, kv_heads, D, page], the order in which the attention reads them.

The caller owns the pool's bookkeeping: an int32 table [batch, width] names each sequence's pages
in order, an int32 tensor the tokens that it holds. Both stay on the device, so that a decode step
can be captured into a graph and replayed as they change. A page id outside the pool, a
length that the table cannot hold, offsets that fall or do not fit the rows: kernels follow none of
them; they raise the cache's `faults` word, and KVCache.check() reports it. Around bad offsets
other sequences of that call may be left out too, or, among more than 64, rows that falling offsets
name twice moved twice.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib

PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
_DTYPES = (torch.bfloat16, torch.float16)
WHOLE_TOKENS = 512   # tokens of a sequence that are never split: no workspace for shorter tables


@dataclass(frozen=True, eq=False)
class KVCache:
    """k_codes uint8 [pages, kv_heads, page, D], k_scales uint8 [pages, kv_heads] (e + 127), v_codes
    uint8 [pages, kv_heads, D, page], v_scales like k_scales, faults int32 [1]; all contiguous.

    copy.deepcopy and pickle give a pool of its own. Each call takes the tensors as they are then:
    their storage may be exchanged (moved to the host and back) for one of the same size."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    faults: torch.Tensor

    def __post_init__(self):
        k, v = self.k_codes, self.v_codes
        if k.ndim != 4 or k.shape[0] <= 0 or k.shape[1] <= 0 or k.shape[2] not in PAGES \
                or k.shape[3] not in HEAD_DIMS:
            raise ValueError(f"K codes must be [pages, kv_heads, page in {PAGES}, D in {HEAD_DIMS}]")
        if v.shape != (*k.shape[:2], k.shape[3], k.shape[2]) or \
                any(s.shape != k.shape[:2] for s in (self.k_scales, self.v_scales)) or \
                self.faults.shape != (1,):
            raise ValueError("V codes, scales and faults do not match the K codes")
        if any(t.dtype != torch.uint8 for t in (k, v, self.k_scales, self.v_scales)) or \
                self.faults.dtype != torch.int32:
            raise ValueError("codes and scales must be uint8, faults int32")
        if any(t.device != k.device or not t.is_contiguous()
               for t in (k, v, self.k_scales, self.v_scales, self.faults)):
            raise ValueError("the cache's tensors must be contiguous and on one device")
        # sizes only: a copied handle has tensors of its own, so addresses are read at each call
        object.__setattr__(self, "_nbytes", tuple(
            t.nbytes for t in (k, self.k_scales, v, self.v_scales)))
        object.__setattr__(self, "_geometry", tuple(k.shape))
        object.__setattr__(self, "_row", (k.shape[1], k.shape[3]))

    @property
    def pages(self):
        return self.k_codes.shape[0]

    @property
    def kv_heads(self):
        return self.k_codes.shape[1]

    @property
    def page(self):
        return self.k_codes.shape[2]

    @property
    def head_dim(self):
        return self.k_codes.shape[3]

    @property
    def device(self):
        return self.k_codes.device

    def check(self):
        """Reads the fault word on the host (waits for the current stream) and raises if it is set."""
        if int(self.faults.item()):
            self.faults.zero_()
            raise RuntimeError("a table, length or offset named what the cache does not have")


def empty_cache(pages, kv_heads, head_dim, page=64, *, device):
    """A pool of `pages` pages of `page` tokens (16 .. 256, a power of two)."""
    if any(type(x) is not int or x <= 0 for x in (pages, kv_heads)):
        raise ValueError("pages and kv_heads must be positive integers")
    if page not in PAGES or head_dim not in HEAD_DIMS:
        raise ValueError(f"page must be in {PAGES} and head_dim in {HEAD_DIMS}")

    def codes(*shape):
        return torch.empty((pages, kv_heads, *shape), dtype=torch.uint8, device=device)

    return KVCache(codes(page, head_dim), codes(), codes(head_dim, page), codes(),
                   torch.zeros(1, dtype=torch.int32, device=device))


def _check_cache(cache, what):
    """(device index, the entry points' arguments) of a cache."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} is inference-only; use no_grad/inference_mode")
    if not isinstance(cache, KVCache):
        raise TypeError("cache must be a KVCache")
    index, args = _cache_args(cache)
    if index < 0:
        raise ValueError("the cache must be on a CUDA (HIP) device")
    return index, args


def _cache_args(cache):
    """The device index (-1 off the GPU) and the entry points' arguments, from the tensors that the
    handle holds now: one that was copied, unpickled or given other storage follows its own."""
    k, ks, v, vs, faults = cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.faults
    index = k.get_device()
    if ks.get_device() != index or v.get_device() != index or vs.get_device() != index \
            or faults.get_device() != index:
        raise ValueError("the cache's tensors must be on one device")
    if (k.nbytes, ks.nbytes, v.nbytes, vs.nbytes) != cache._nbytes:
        raise ValueError("the cache's tensors are not of the size that the handle was made for")
    return index, (k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), faults.data_ptr(),
                   *cache._geometry)


def _check_table(table, index):
    """(batch, width, row stride) of a page table."""
    if table.ndim != 2 or table.dtype is not torch.int32 or table.get_device() != index:
        raise ValueError("table must be int32 [batch, width] on the cache's device, unit inner stride")
    batch, width = table.shape
    row, inner = table.stride()
    if inner != 1 and width > 1:
        raise ValueError("table must be int32 [batch, width] on the cache's device, unit inner stride")
    return batch, width, row


def _check_vector(name, t, n, index):
    if t.ndim != 1 or t.shape[0] != n or t.dtype is not torch.int32 or t.get_device() != index \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{n}] on the cache's device")


def _move(name, index, args, key, value, rows, dtype, table, starts, offsets):
    batch, width, t_st = _check_table(table, index)
    _check_vector("starts", starts, batch, index)
    if offsets is not None:
        _check_vector("offsets", offsets, batch + 1, index)
        offsets = offsets.data_ptr()
    elif rows != batch:
        raise ValueError("without offsets there is one row for each sequence")
    if rows > 2 ** 31 - 1:
        raise ValueError("too many rows")
    k_st, k_sh, k_sd = key.stride()
    v_st, v_sh, v_sd = value.stride()
    if k_sd != 1 or v_sd != 1:
        raise ValueError("key and value must have unit innermost stride")
    _lib.call_on(index, name, *args, table.data_ptr(), t_st, batch, width,
                 starts.data_ptr(), offsets, key.data_ptr(), k_st, k_sh, value.data_ptr(), v_st,
                 v_sh, rows, 1 if dtype is torch.float16 else 0, _lib.raw_stream(index))


def write_cache(cache: KVCache, key, value, table, starts, offsets=None):
    """Appends packed rows to their sequences.

    key, value [rows, kv_heads, D] (BF16 or FP16, unit channel stride); rows offsets[i] ..
    offsets[i + 1] - 1 (int32 [batch + 1], rising from 0; one row each without it) become
    the tokens starts[i], starts[i] + 1, ... of sequence i, in the pages that table[i] names.
    Rows from offsets[batch] on are not written.

    A page that holds earlier tokens of the sequence (the first one, if starts[i] is not a multiple
    of the page) keeps the larger of its scale and the new tokens' one; if that is the new
    tokens', the held codes are rounded once more. A nonfinite value becomes the NaN code and
    leaves the scale alone. No page may be written twice in one call, by two sequences or by a table
    that names it twice."""
    index, args = _check_cache(cache, "write_cache")
    shape, dtype = key.shape, key.dtype
    if len(shape) != 3 or shape[1:] != cache._row or value.shape != shape:
        raise ValueError("key and value must be [rows, kv_heads, D] of the cache")
    if dtype not in _DTYPES or value.dtype is not dtype or key.get_device() != index \
            or value.get_device() != index:
        raise ValueError("key and value must share BF16 or FP16 and the cache's device")
    _move("vdn_cache_write", index, args, key, value, shape[0], dtype, table, starts, offsets)


def read_cache(cache: KVCache, table, starts, offsets, rows, *, dtype=torch.bfloat16):
    """The values of cached tokens, packed: rows offsets[i] .. offsets[i + 1] - 1 of the two
    fresh [rows, kv_heads, D] tensors (keys, values) are the tokens starts[i], ... of sequence i
    (arguments as write_cache). Exact in BF16; FP16 rounds what is under its normal range and
    saturates at 65504. Rows of a page that is not there are NaN, rows from offsets[batch] on
    zero; rows of offsets that are not followed may hold anything."""
    index, args = _check_cache(cache, "read_cache")
    if type(rows) is not int or rows < 0:
        raise ValueError("rows must be a non-negative integer")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be BF16 or FP16")
    key = torch.empty((rows, *cache._row), dtype=dtype, device=cache.k_codes.device)
    value = torch.empty_like(key)
    _move("vdn_cache_read", index, args, key, value, rows, dtype, table, starts, offsets)
    return key, value


def cache_attention(query, cache: KVCache, table, lengths, scale=None, *, return_lse=False,
                    out=None):
    """Softmax attention of each sequence's newest tokens over all its cached ones.

    query [batch, Q, H, D] or [batch, H, D] (Q = 1), BF16 or FP16, H a multiple of the cache's
    kv_heads (query head h reads K/V head h // (H / kv_heads)); lengths int32 [batch] counts
    the tokens that the cache holds, the Q queries' own among them: query i sees the tokens j <
    lengths - Q + 1 + i. A row that sees none is zero, one
    whose scores are all -inf NaN (LSE -inf). Returns a tensor like the query,
    with return_lse also the natural-log sum of exp of the scaled scores, fp32 [batch, Q, H]
    (or [batch, H]). Scores, sums and the output are accumulated in fp32; probabilities are
    rounded to the query's dtype before the product with V, the codes' values are exact.

    `out` may be the query itself; it must not overlap it otherwise, nor itself, nor the cache.

    A sequence with a bad page id or length gets NaN (see KVCache.check). For FP16 queries
    the cached values must be within FP16's range; an output that E4M3's rounding takes over its
    largest value is that value."""
    index, args = _check_cache(cache, "cache_attention")
    if query.ndim not in (3, 4):
        raise ValueError("query must be [batch, Q, H, D] or [batch, H, D]")
    dtype = query.dtype
    _, kv_heads, page, dim = cache._geometry
    if query.ndim == 4:
        batch, tokens, heads, d = query.shape
        q_sb, q_st, q_sh, q_sd = query.stride()
    else:
        batch, heads, d = query.shape
        q_sb, q_sh, q_sd = query.stride()
        tokens, q_st = 1, 0
    if d != dim or heads <= 0 or heads % kv_heads or tokens <= 0:
        raise ValueError("query heads must be a multiple of the cache's, D the same, Q positive")
    if dtype not in _DTYPES or q_sd != 1 or query.get_device() != index:
        raise ValueError("query must be BF16 or FP16 with unit innermost stride, on the cache's device")
    table_batch, width, t_st = _check_table(table, index)
    _check_vector("lengths", lengths, batch, index)
    if table_batch != batch or width <= 0:
        raise ValueError("table must name at least one page for each sequence of the query")
    if width * page > 2 ** 31 - 1024:
        raise ValueError("the table is too wide")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif (out.shape != query.shape or out.dtype is not dtype or out.get_device() != index
          or out.stride(-1) != 1 or 0 in out.stride()):
        raise ValueError("out must be a view like the query, unit channel stride, no broadcast")
    else:
        _lib.check_attention_out(out, query)
    o_sb, o_sh, o_st = out.stride(0), out.stride(-2), out.stride(1) if out.ndim == 4 else 0
    lse = torch.empty(query.shape[:-1], dtype=torch.float32, device=query.device) if return_lse else None
    group = heads // kv_heads
    workspace, nbytes = None, 0
    if width * page > WHOLE_TOKENS:
        # from the allocator in stream order: calls on other streams and captured graphs have their own
        nbytes = _workspace_bytes(index, tokens, group, d)
        workspace = query.new_empty(nbytes // 2)   # 2-byte elements
    _lib.call_on(index, "vdn_cache_attention", query.data_ptr(), q_sb, q_st, q_sh,
                 *args, table.data_ptr(), t_st, batch, width,
                 lengths.data_ptr(), tokens, group, int(dtype is torch.float16), scale,
                 out.data_ptr(), o_sb, o_st, o_sh, _lib.ptr(lse), _lib.ptr(workspace), nbytes,
                 _lib.raw_stream(index))
    return (out, lse) if return_lse else out


@lru_cache(maxsize=None)
def _workspace_bytes(device_index, tokens, group, head_dim):
    nbytes = ctypes.c_int64(0)
    _lib.call_on(device_index, "vdn_cache_attention_workspace", tokens, group,
                 head_dim, ctypes.addressof(nbytes))
    return nbytes.value
