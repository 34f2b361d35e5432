"""CPU: the causal plan's blocks, its refusals, and the oracle's closed forms."""
import ctypes

import pytest
import torch

from oracle import causal as oc
from vdn_amd import _lib
from vdn_amd import causal as vc


@pytest.mark.parametrize("block_rows", [128, 256])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([5, 0, 700, 1], 6, 2), ([1], 1, 1), ([300] * 3, 7, 1),
                                                    ([], 2, 1), ([0], 2, 2)])
def test_blocks_cover_every_row_once(lengths, heads, kv_heads, block_rows):
    plan = vc.prepare_causal_plan(lengths, heads, kv_heads)
    group, seen = heads // kv_heads, set()
    blocks = vc._blocks(tuple(lengths), group, block_rows)
    assert block_rows == 256 or torch.equal(blocks, plan.blocks)
    first = {sum(lengths[:i]): n for i, n in enumerate(lengths) if n}
    keys = []
    for row0, n, r0, _ in blocks.tolist():
        assert first[row0] == n and r0 % block_rows == 0 and 0 <= r0 < n * group
        for r in range(r0, min(r0 + block_rows, n * group)):
            assert (row0, r) not in seen
            seen.add((row0, r))
        keys.append((min(r0 + block_rows, n * group) - 1) // group)
    assert len(seen) == sum(lengths) * group == plan.rows * group
    assert keys == sorted(keys, reverse=True)


def test_wide_blocks_where_rows_see_many_keys():
    assert vc.prepare_causal_plan([4096], 32, 8).wide_blocks.shape == (64, 4)
    assert vc.prepare_causal_plan([4094], 32, 8).wide_blocks is None     # 2047.5 keys
    assert vc.prepare_causal_plan([8192], 8, 1).wide_blocks is None      # 256 blocks
    assert vc.prepare_causal_plan([2048] * 4, 32, 8).wide_blocks is None


def test_plan_refusals():
    for lengths in ([-1], [2.0], [True, "a"]):
        with pytest.raises(ValueError, match="lengths"):
            vc.prepare_causal_plan(lengths, 4)
    for heads in ((0, 1), (4, 3), (4, 0), (4.0, 2)):
        with pytest.raises(ValueError, match="heads"):
            vc.prepare_causal_plan([3], *heads)
    with pytest.raises(ValueError, match="too many"):
        vc.prepare_causal_plan([2 ** 31], 1)


def test_calls_that_need_a_device():
    plan = vc.prepare_causal_plan([3], 2)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with torch.no_grad():
        with pytest.raises(ValueError, match="CUDA"):
            vc.causal_attention(x, x, x, plan)
        with pytest.raises(TypeError, match="prepare_causal_plan"):
            vc.causal_attention(x, x, x, None)
    with pytest.raises(RuntimeError, match="inference-only"):
        vc.causal_attention(x, x, x, plan)


def test_entry_point_validates_before_launching():
    lib, fake = _lib.load(), 1 << 20

    def call(q=fake, k_st=256, blocks=fake, nblocks=1, rows=256, dim=128, dtype=0, scale=0.1, out=fake):
        return lib.vdn_causal_attention(q, 256, 128, fake, k_st, 128, fake, 256, 128, blocks, nblocks,
                                        rows, 2, 1, dim, dtype, scale, out, 256, 128, None, 0, 0, None)
    for change, word in ((dict(q=None), b"null"), (dict(out=None), b"null"), (dict(nblocks=-1), b"geometry"),
                         (dict(rows=64), b"block_rows"), (dict(rows=256, dim=64), b"block_rows"),
                         (dict(dim=96), b"head_dim"),
                         (dict(dtype=2), b"dtype"), (dict(scale=0.0), b"scale"),
                         (dict(q=fake + 8), b"16-byte"), (dict(k_st=252), b"16-byte"),
                         (dict(k_st=1 << 23), b"strides")):
        assert call(**change) != 0, change
        assert word in lib.vdn_last_error(), change
    assert call(nblocks=0, blocks=None) == 0
    assert isinstance(lib.vdn_causal_attention, ctypes._CFuncPtr)


def test_oracle_closed_forms():
    """Equal scores: the running mean of V and log(i + 1)."""
    n = 9
    v = torch.randn(n, 2, 64).double()
    z = torch.zeros(n, 2, 64)
    out, lse, mass, size = oc.attention(z, z, v, 0, 0.125)
    count = torch.arange(1, n + 1).double()
    torch.testing.assert_close(out, v.cumsum(0) / count[:, None, None])
    torch.testing.assert_close(lse, count.log()[:, None].expand(n, 2))
    torch.testing.assert_close(mass, v.abs().cumsum(0) / count[:, None, None])
    assert not size.any()
    out, lse, _, _ = oc.attention(z, z, v, -3, 0.125)     # the first three rows see nothing
    assert not out[:3].any() and torch.isneginf(lse[:3]).all()
    torch.testing.assert_close(out[3], v[0])
