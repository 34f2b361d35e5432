"""CPU: handles that were copied, unpickled or given other storage name their own tensors."""
import copy
import pickle

import pytest
import torch

from vdn_amd import causal as vc
from vdn_amd import kvcache as kv

PARTS = ("k_codes", "k_scales", "v_codes", "v_scales", "faults")


def addresses(handle, parts):
    return tuple(getattr(handle, p).data_ptr() for p in parts)


def test_cache_copies_name_their_own_tensors():
    cache = kv.empty_cache(4, 2, 64, 16, device="cpu")
    index, args = kv._cache_args(cache)
    assert index == -1 and args == (*addresses(cache, PARTS), 4, 2, 16, 64)
    for fork in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        _, own = kv._cache_args(fork)
        assert own == (*addresses(fork, PARTS), 4, 2, 16, 64)
        assert not set(own[:5]) & set(args[:5])
        assert kv._cache_args(cache)[1] == args
    same = copy.copy(cache)                        # a shallow copy shares the tensors
    assert kv._cache_args(same)[1] == args


@pytest.mark.parametrize("part", PARTS)
def test_cache_follows_exchanged_storage(part):
    cache = kv.empty_cache(4, 2, 64, 16, device="cpu")
    before = addresses(cache, PARTS)
    fresh = getattr(cache, part).clone()
    getattr(cache, part).data = fresh
    args = kv._cache_args(cache)[1]
    assert args[:5] == addresses(cache, PARTS) != before
    assert args[PARTS.index(part)] == fresh.data_ptr()


@pytest.mark.parametrize("part", PARTS[:4])
def test_cache_refuses_storage_of_another_size(part):
    cache = kv.empty_cache(4, 2, 64, 16, device="cpu")
    tensor = getattr(cache, part)
    tensor.data = tensor[:3].clone()
    with pytest.raises(ValueError, match="size"):
        kv._cache_args(cache)


@pytest.mark.parametrize("lengths,heads,kv_heads,block_rows", [([40, 3], 4, 2, 128), ([4096], 32, 8, 256)])
def test_plan_copies_name_their_own_blocks(lengths, heads, kv_heads, block_rows):
    plan = vc.prepare_causal_plan(lengths, heads, kv_heads)
    for fork in (plan, copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        own = fork.blocks if block_rows == 128 else fork.wide_blocks
        assert fork is plan or own.data_ptr() not in (plan.blocks.data_ptr(), plan.blocks.data_ptr() + 16 * len(
            plan.blocks))
        assert vc._launch(fork, 128) == ((own.data_ptr(), own.shape[0], block_rows), -1)
        assert vc._launch(fork, 64) == ((fork.blocks.data_ptr(), fork.blocks.shape[0], 128), -1)
    plan.blocks.data = plan.blocks.clone()
    assert vc._launch(plan, 256)[0][0] == plan.blocks.data_ptr()
