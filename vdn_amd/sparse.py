"""Attention of each query over the pages of the 8-bit cache (kvcache.py) that a cheap score selects for it.

Three calls beside the cache's own: write_means keeps the mean key of every page as the cache
grows, select_pages scores the pages of a sequence by their means and names the best ones for each
query and K/V head, selected_attention attends over those:

    write_cache(cache, k, v, table, lengths); write_means(cache, means, table, lengths, lengths + 1)
    lengths += 1
    pages, tokens = select_pages(q, cache, means, table, lengths, 32)
    out = selected_attention(q, cache, pages, tokens)

Table, lengths and the selection stay on the device, so that a captured step may change them between
replays. Bad page ids and lengths raise the cache's fault word, as in kvcache.py.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch

from . import _lib
from .kvcache import (KVCache, WHOLE_TOKENS, _DTYPES, _check_cache, _check_table, _check_vector,
                      _workspace_bytes)


MOST_PAGES = 65536   # of a table that pages are selected from


def empty_means(cache: KVCache):
    """BF16 [pages, kv_heads, D] for write_means: the mean keys of the cache's pages, not yet set."""
    return torch.empty((*cache.k_scales.shape, cache.head_dim), dtype=torch.bfloat16, device=cache.device)


def _check_means(cache, means, index):
    pages, kv_heads, _, dim = cache._geometry
    if means.shape != (pages, kv_heads, dim) or means.dtype is not torch.bfloat16 \
            or means.get_device() != index or not means.is_contiguous():
        raise ValueError("means must be contiguous BF16 [pages, kv_heads, D] on the cache's device")


def write_means(cache: KVCache, means, table, starts, lengths):
    """Sets the mean key of every page that holds tokens starts[i] .. lengths[i] - 1 of a sequence (int32
    [batch] each): over all the page's tokens in front of lengths[i], from the codes that the cache holds,
    rounded once to BF16. Call it after write_cache, with its starts and the new lengths. A NaN key
    makes its channel's mean NaN. Other pages' means stay as they are. Sequences may share full pages, but
    not one that is partly filled to different lengths in the same call."""
    index, args = _check_cache(cache, "write_means")
    _check_means(cache, means, index)
    batch, width, t_st = _check_table(table, index)
    _check_vector("starts", starts, batch, index)
    _check_vector("lengths", lengths, batch, index)
    if width <= 0:
        raise ValueError("table must name at least one page for each sequence")
    k, ks, _, _, faults, *geometry = args
    _lib.call_on(index, "vdn_cache_means", k, ks, faults, *geometry, table.data_ptr(), t_st, batch, width,
                 starts.data_ptr(), lengths.data_ptr(), means.data_ptr(), _lib.raw_stream(index))


def _check_query(query, cache, index):
    """(batch, Q, H, D, strides of the first three)"""
    if query.ndim == 4:
        batch, tokens, heads, d = query.shape
        q_sb, q_st, q_sh, q_sd = query.stride()
    elif query.ndim == 3:
        batch, heads, d = query.shape
        q_sb, q_sh, q_sd = query.stride()
        tokens, q_st = 1, 0
    else:
        raise ValueError("query must be [batch, Q, H, D] or [batch, H, D]")
    _, kv_heads, _, dim = cache._geometry
    if d != dim or heads <= 0 or heads % kv_heads or tokens <= 0:
        raise ValueError("query heads must be a multiple of the cache's, D the same, Q positive")
    if query.dtype not in _DTYPES or q_sd != 1 or query.get_device() != index:
        raise ValueError("query must be BF16 or FP16 with unit innermost stride, on the cache's device")
    return batch, tokens, heads, d, q_sb, q_st, q_sh


def select_pages(query, cache: KVCache, means, table, lengths, count, *, first=1, last=1):
    """The `count` pages of its sequence that each query and K/V head attends over.

    query [batch, Q, H, D] or [batch, H, D] (Q = 1), BF16 or FP16, rows 16-byte aligned: the newest tokens of each sequence, as
    in cache_attention; means as write_means left them. Query i sees the pages with tokens in front of
    lengths - Q + 1 + i (tables of up to 65536 pages; batch x Q x kv_heads below 2^22, and where the table is wider than
    4096 pages, that times its width in whole 64 pages below 2^30); a page's score is the largest q . mean over the query heads of the K/V head, in 64 bits.
    The first `first` pages and the last `last` (at least 1) that the query sees are always taken; of equal
    scores the page in front. A NaN score counts as +inf.

    Returns (pages, tokens): int32 [batch, Q, kv_heads, count] (or [batch, kv_heads, count]) page ids in the
    table's order, -1 behind the last one where the sequence has fewer, and int32 [batch, Q] (or
    [batch]) the tokens in them: what selected_attention takes. A bad length gives -1 tokens; a page id that
    the pool does not have is selected before scored ones, so that the attention reports it."""
    index, args = _check_cache(cache, "select_pages")
    _check_means(cache, means, index)
    batch, tokens, heads, d, q_sb, q_st, q_sh = _check_query(query, cache, index)
    table_batch, width, t_st = _check_table(table, index)
    _check_vector("lengths", lengths, batch, index)
    _, kv_heads, page, _ = cache._geometry
    if table_batch != batch or width <= 0:
        raise ValueError("table must name at least one page for each sequence of the query")
    if width > MOST_PAGES or width * page > 2 ** 31 - 1024:
        raise ValueError(f"the table must not be wider than {MOST_PAGES} pages or 2^31 tokens")
    units = batch * tokens * kv_heads
    if units >= 2 ** 22 or (width > 4096 and units * -(-width // 64) >= 2 ** 24):
        raise ValueError("too many queries and pages for one call")
    if any(type(n) is not int for n in (count, first, last)) or first < 0 or last < 1 or count < first + last:
        raise ValueError("count must be at least first + last, first >= 0, last >= 1")
    lead = query.shape[:-2]
    pages = lengths.new_empty((*lead, kv_heads, count))
    seen = lengths.new_empty(lead)
    nbytes = _select_bytes(index, batch, tokens, kv_heads, width) if batch else 0
    workspace = query.new_empty(nbytes // 2) if nbytes else None
    faults, geometry = args[4], args[5:]
    _lib.call_on(index, "vdn_cache_select", query.data_ptr(), q_sb, q_st, q_sh, means.data_ptr(), faults,
                 *geometry, table.data_ptr(), t_st, batch, width, lengths.data_ptr(), tokens,
                 heads // kv_heads, int(query.dtype is torch.float16), count, first, last, pages.data_ptr(),
                 seen.data_ptr(), _lib.ptr(workspace), nbytes, _lib.raw_stream(index))
    return pages, seen


def _merged(x, tokens, what):
    """Strides of [batch * Q, heads] of a [batch, Q, heads, ..] or [batch, heads, ..] tensor."""
    if x.ndim == 3:
        return x.stride()[:2]
    s_b, s_t, s_h, _ = x.stride()
    if tokens == 1:
        return s_b, s_h
    if x.shape[0] > 1 and s_b != tokens * s_t:
        raise ValueError(f"{what}'s tokens must follow each other at one stride")
    return s_t, s_h


def selected_attention(query, cache: KVCache, pages, tokens, scale=None, *, return_lse=False, out=None):
    """Softmax attention of each query over its selected pages.

    query [batch, Q, H, D] or [batch, H, D] as in select_pages, its Q tokens at one stride; pages int32 [batch, Q,
    kv_heads, count] (or [batch, kv_heads, count]; unit inner stride) and tokens int32 [batch, Q] (or
    [batch]) as that returns them: query head h attends over the first `tokens` tokens of the pages that
    pages[..., h // (H / kv_heads), :] names, in that order, all of them full but the last one. A caller's
    own selection may name any pages of the pool; one that is named twice counts twice.

    Output, return_lse, out and faults as in cache_attention: a query with no tokens is zero, LSE -inf."""
    index, args = _check_cache(cache, "selected_attention")
    batch, q_tokens, heads, d, *_ = _check_query(query, cache, index)
    _, kv_heads, page, _ = cache._geometry
    shape, lead, dtype = query.shape, query.shape[:-2], query.dtype
    if pages.shape[:-1] != (*lead, kv_heads) or pages.dtype is not torch.int32 or pages.get_device() != index \
            or pages.shape[-1] == 0 or pages.stride(-1) != 1:
        raise ValueError("pages must be int32 [batch, Q, kv_heads, count] for the query, unit inner stride, on "
                         "the cache's device")
    if tokens.shape != lead or tokens.dtype is not torch.int32 or tokens.get_device() != index \
            or not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous int32 [batch, Q] for the query, on the cache's device")
    count = pages.shape[-1]
    if count * page > 2 ** 31 - 1024:
        raise ValueError("too many pages")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    if out is None:
        out, o_sb, o_sh = query.new_empty(shape), heads * d, d
    elif (out.shape != shape or out.dtype is not dtype or out.get_device() != index
          or out.stride(-1) != 1 or 0 in out.stride()):
        raise ValueError("out must be a view like the query, unit channel stride, no broadcast")
    else:
        _lib.check_attention_out(out, query)
        o_sb, o_sh = _merged(out, q_tokens, "out")
    q_sb, q_sh = _merged(query, q_tokens, "query")
    p_sb, p_sh = _merged(pages, q_tokens, "pages")
    lse = lse_ptr = None
    if return_lse:
        lse = query.new_empty(shape[:-1], dtype=torch.float32)
        lse_ptr = lse.data_ptr()
    group = heads // kv_heads
    workspace, nbytes = None, 0
    if count * page > WHOLE_TOKENS:
        # from the allocator in stream order: calls on other streams and captured graphs have their own
        nbytes = _workspace_bytes(index, 1, group, d)
        workspace = query.new_empty(nbytes // 2)   # 2-byte elements
    _lib.call_on(index, "vdn_cache_attention_heads", query.data_ptr(), q_sb, q_sh, *args, pages.data_ptr(), p_sb, p_sh,
                 batch * q_tokens, count, tokens.data_ptr(), group, int(dtype is torch.float16), scale,
                 out.data_ptr(), o_sb, o_sh, lse_ptr, _lib.ptr(workspace), nbytes, _lib.raw_stream(index))
    return (out, lse) if return_lse else out


@lru_cache(maxsize=4096)
def _select_bytes(device_index, batch, tokens, kv_heads, width):
    nbytes = ctypes.c_int64(0)
    _lib.call_on(device_index, "vdn_cache_select_workspace", batch, tokens, kv_heads, width,
                 ctypes.addressof(nbytes))
    return nbytes.value
