"""GPU: the 8-bit cache at the edges of its types, against the formula in 64 bits."""
import math

import pytest
import torch

from oracle import causal as oc
from oracle import kvcache as ok
from vdn_amd import kvcache as kv

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def in_order(n, page):
    """The table of one sequence of n tokens whose pages lie in order."""
    return torch.arange(-(-n // page), dtype=torch.int32)[None]


@pytest.mark.parametrize("n", [1, 300, 3000])          # one token, a whole unit, a split one
@pytest.mark.parametrize("dim", [64, 128, 256])
@torch.no_grad()
def test_fp16_outputs_next_to_the_largest_value(device, n, dim):
    """65504 and 63488 are stored as 65536: an output of theirs is 65504. (The rounded weights sum
    to within 2^-11 of 1, and from 65536 (1 - 2^-11) on fp16 gives 65504.)"""
    cache = kv.empty_cache(-(-n // 16), 2, dim, 16, device=device)
    table = in_order(n, 16).cuda()
    v = torch.full((n, 2, dim), 65504.0)
    v[..., 1::4], v[..., 2::4], v[..., 3::4] = -65504.0, 63488.0, -1.0
    k = torch.randn(n, 2, dim, generator=torch.Generator().manual_seed(n))
    kv.write_cache(cache, k.to(FP16).cuda(), v.to(FP16).cuda(), table, ints(0), ints(0, n))
    q = torch.randn(1, 6, dim, generator=torch.Generator().manual_seed(1)).to(FP16).cuda()
    out, lse = kv.cache_attention(q, cache, table, ints(n), return_lse=True)
    assert (out[..., 0::4] == 65504).all() and (out[..., 1::4] == -65504).all()
    assert (out[..., 2::4] == 65504).all() and torch.isfinite(lse).all()
    assert torch.isfinite(out).all()
    cache.check()
