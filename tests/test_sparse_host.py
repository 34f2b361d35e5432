"""CPU: the refusals of the page selection's calls, and the oracle's pins."""
import ctypes
import math

import pytest
import torch

from oracle import sparse as osp
from vdn_amd import _lib
from vdn_amd import kvcache as kv
from vdn_amd import sparse as sp

P = 1 << 20


def test_oracle_rounds_as_torch():
    x = torch.randn(2000, dtype=torch.float64).float()
    assert torch.equal(osp.to_bf16(x.double()).float(), x.bfloat16().float())
    ties = torch.tensor([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -1 - 2.0 ** -8, math.inf, 0.0], dtype=torch.float64)
    assert osp.to_bf16(ties).tolist() == [1.0, 1 + 2.0 ** -6, -1.0, math.inf, 0.0]
    assert osp.to_bf16(torch.tensor([1 + 2.0 ** -8 + 2.0 ** -40], dtype=torch.float64)).item() == 1 + 2.0 ** -7


def test_oracle_selection():
    means = torch.tensor([[[3.0]], [[1.0]], [[math.nan]], [[5.0]], [[5.0]], [[0.0]]])
    q = torch.ones(1, 1, 1)
    for count, first, last, want in ((2, 0, 1, [2, 5]), (3, 0, 1, [2, 3, 5]), (4, 1, 1, [0, 2, 3, 5]),
                                     (9, 0, 1, [0, 1, 2, 3, 4, 5])):
        (picked, tokens), = osp.select(q, means, range(6), 95, 16, count, first, last)
        assert picked == [want] and tokens == 16 * (len(want) - 1) + 15


def test_calls_need_a_device_and_no_grad():
    c = kv.empty_cache(2, 1, 64, 16, device="cpu")
    m = sp.empty_means(c)
    assert m.shape == (2, 1, 64) and m.dtype is torch.bfloat16
    x, t, n = torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, 1).int(), torch.zeros(1).int()
    calls = (lambda: sp.write_means(c, m, t, n, n), lambda: sp.select_pages(x, c, m, t, n, 1, first=0),
             lambda: sp.selected_attention(x, c, torch.zeros(1, 1, 1).int(), n))
    for call in calls:
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call()


def test_entry_points_validate_before_launching():
    lib = _lib.load()

    def means(codes=P, pages=4, heads=2, page=16, dim=64, table=P, batch=2, width=2, starts=P, out=P):
        return lib.vdn_cache_means(codes, P, P, pages, heads, page, dim, table, 2, batch, width, starts, P, out,
                                   None)

    for bad in (dict(pages=0), dict(page=48), dict(dim=96), dict(width=0), dict(batch=-1), dict(codes=None),
                dict(table=None), dict(starts=None), dict(out=None), dict(out=P + 8), dict(codes=P + 8)):
        assert means(**bad) != 0, bad
    assert means(batch=0, table=None) == 0

    def select(q=P, q_sh=64, m=P, pages=4, heads=2, page=16, dim=64, batch=2, width=2, tokens=1, group=1, dtype=0,
               count=2, first=1, last=1, out=P, ws=P, nbytes=1 << 40):
        return lib.vdn_cache_select(q, 128, 128, q_sh, m, P, pages, heads, page, dim, P, 2, batch, width, P, tokens,
                                    group, dtype, count, first, last, out, P, ws, nbytes, None)

    for bad, said in ((dict(page=8), b"geometry"), (dict(width=1 << 30), b"geometry"), (dict(group=0), b"geometry"),
                      (dict(tokens=0), b"geometry"), (dict(dtype=2), b"dtype"), (dict(count=1), b"count"),
                      (dict(last=0), b"last"), (dict(first=-1), b"first"), (dict(first=2 ** 31 - 1), b"count"),
                      (dict(q=None), b"null"), (dict(m=None), b"null"), (dict(out=None), b"null"),
                      (dict(q_sh=60), b"alignment"), (dict(q=P + 8), b"alignment"),
                      (dict(batch=1 << 30), b"too many"), (dict(width=1 << 17), b"geometry"), (dict(width=1 << 16, ws=None), b"workspace"),
                      (dict(width=1 << 16, nbytes=1000), b"workspace")):
        assert select(**bad) != 0, bad
        assert said in lib.vdn_last_error(), (bad, lib.vdn_last_error())
    assert select(batch=0, q=None) == 0
    n = ctypes.c_int64(0)
    assert lib.vdn_cache_select_workspace(1, 1, 0, 4, ctypes.addressof(n)) != 0
    assert lib.vdn_cache_select_workspace(1, 1, 1, 4, None) != 0

    def heads(q=P, q_sh=64, tables=P, batch=2, width=2, group=1, dim=64, scale=0.1, ws=P, nbytes=1 << 30):
        return lib.vdn_cache_attention_heads(q, 128, q_sh, P, P, P, P, P, 4, 2, 16, dim, tables, 4, 2, batch, width,
                                             P, group, 0, scale, P, 128, 64, None, ws, nbytes, None)

    for bad in (dict(q=None), dict(tables=None), dict(width=0), dict(group=0), dict(dim=32), dict(scale=0.0),
                dict(q_sh=60), dict(width=64, ws=None)):
        assert heads(**bad) != 0, bad
    assert b"vdn_cache_attention_heads" in lib.vdn_last_error()
    assert heads(batch=0) == 0


def test_limits_of_a_selection():
    """A grid has fewer than 2^32 threads: 1024 for a unit, and 256 for 64 of its pages where a workspace holds them."""
    lib = _lib.load()

    def select(batch, tokens, heads, width):
        return lib.vdn_cache_select(P, 128, 128, 64, P, P, 4, heads, 16, 64, P, 2, batch, width, P, tokens, 1, 0, 2, 1, 1,
                                    P, P, None, 0, None)

    # (no workspace: what is within the limits is refused for that)
    for sizes, said in (((511, 1, 32, 65536), b"workspace"), ((512, 1, 32, 65536), b"too many"),
                        ((512, 1, 8, 65536), b"workspace"), ((513, 4, 8, 65472), b"too many"),
                        ((2 ** 19, 1, 8, 16), b"too many"), ((1000, 4, 8, 4097), b"workspace")):
        assert select(*sizes) != 0 and said in lib.vdn_last_error(), (sizes, lib.vdn_last_error())
