"""GPU: handles that were copied, unpickled or moved work on their own memory."""
import copy
import io

import pytest
import torch

from vdn_amd import causal as vc
from vdn_amd import kvcache as kv

pytestmark = pytest.mark.gpu

PARTS = ("k_codes", "k_scales", "v_codes", "v_scales", "faults")


def small_cache(device):
    """A pool of 3 pages with 20 tokens, its table, the tokens' count and a query."""
    g = torch.Generator().manual_seed(0)
    cache = kv.empty_cache(3, 2, 64, 16, device=device)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=device)
    x = torch.randn(20, 2, 64, generator=g).bfloat16().to(device)
    zero, held = (torch.tensor([n], dtype=torch.int32, device=device) for n in (0, 20))
    kv.write_cache(cache, x, -x, table, zero, torch.tensor([0, 20], dtype=torch.int32, device=device))
    return cache, table, held, torch.randn(1, 4, 64, generator=g).bfloat16().to(device)


def forks(cache):
    stream = io.BytesIO()
    torch.save(cache, stream)
    stream.seek(0)
    # a file that this test has just written
    return copy.deepcopy(cache), torch.load(stream, weights_only=False)


@torch.no_grad()
def test_a_forked_cache_is_a_pool_of_its_own(device):
    cache, table, held, q = small_cache(device)
    want = kv.cache_attention(q, cache, table, held)
    loud = torch.full((1, 2, 64), 50.0, dtype=torch.bfloat16, device=device)
    for fork in forks(cache):
        assert torch.equal(kv.cache_attention(q, fork, table, held), want)
        codes = [getattr(cache, p).clone() for p in PARTS]
        kv.write_cache(fork, loud, loud, table, held)
        assert all(torch.equal(getattr(cache, p), c) for p, c in zip(PARTS, codes))
        k, _ = kv.read_cache(fork, table, held, None, 1)
        assert (k == 48).all() or (k == 52).all()       # E4M3: steps of 4 from 32 on
        assert torch.equal(kv.cache_attention(q, cache, table, held), want)
        kv.cache_attention(q, fork, table, -held)
        cache.check()                                   # the fork's fault, not this pool's
        with pytest.raises(RuntimeError):
            fork.check()


@torch.no_grad()
def test_a_cache_that_goes_to_the_host_and_back(device):
    cache, table, held, q = small_cache(device)
    want = kv.cache_attention(q, cache, table, held)
    for parts in (("v_codes",), ("faults",), PARTS):
        for p in parts:
            getattr(cache, p).data = getattr(cache, p).data.cpu()
        with pytest.raises(ValueError, match="device"):
            kv.cache_attention(q, cache, table, held)
        filler = [torch.full((1 << 20,), 127, dtype=torch.uint8, device=device)]
        for p in parts:
            getattr(cache, p).data = getattr(cache, p).data.to(device)
        assert torch.equal(kv.cache_attention(q, cache, table, held), want)
        del filler
    cache.check()


@torch.no_grad()
def test_a_forked_plan_outlives_the_first_one(device):
    x = torch.randn(150, 6, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    q, k, v = x[:, :4], x[:, 4:5], x[:, 5:]
    plan = vc.prepare_causal_plan([100, 50], 4, 1, device=device)
    want = vc.causal_attention(q, k, v, plan)
    fork, loaded = forks(plan)
    plan.blocks.copy_(vc.prepare_causal_plan([50, 100], 4, 1).blocks)
    assert not torch.equal(vc.causal_attention(q, k, v, plan), want)
    for own in (fork, loaded):
        assert torch.equal(vc.causal_attention(q, k, v, own), want)
    loaded.blocks.data = loaded.blocks.data.cpu()
    with pytest.raises(ValueError, match="device"):
        vc.causal_attention(q, k, v, loaded)
