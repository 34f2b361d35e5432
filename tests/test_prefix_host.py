"""CPU: plans of shared prefixes, and what is refused."""
import ctypes
import math
import random

import pytest
import torch

from vdn_amd import _lib
from vdn_amd import kvcache as kv
from vdn_amd import prefix as vp

P = 1 << 20


def test_every_row_and_tile_is_in_one_item():
    r = random.Random(3)
    for _ in range(200):
        n = r.randint(1, 6)
        lengths = [r.choice((0, 1, 63, 64, 65, r.randint(1, 70000))) for _ in range(n)]
        counts = [r.choice((0, 1, 2, r.randint(1, 200))) for _ in range(n)]
        heads, kv_heads = r.choice(((1, 1), (40, 8), (12, 2), (16, 16), (24, 1)))
        dim, tokens = r.choice((64, 128, 256)), r.choice((1, 1, 4))
        plan = vp.prepare_prefix_plan(lengths, counts, heads, kv_heads, dim, tokens=tokens, device="cpu")
        assert plan.batch == sum(counts) and plan.items.dtype is plan.sequences.dtype is torch.int32
        items, seqs = plan.items.tolist(), plan.sequences.tolist()
        assert len(seqs) == plan.batch
        b = 0
        for p, (length, count) in enumerate(zip(lengths, counts)):
            first, rows, tiles = b, count * tokens * heads // kv_heads, -(-length // vp.TILE)
            for _ in range(count):
                f, base, pieces, blocks, n_tokens = seqs[b][:5]
                assert (f, n_tokens) == (first, length)
                assert blocks == (-(-rows // vp.BLOCK_ROWS) if length else 0) and (pieces > 0) == (length > 0)
                b += 1
            if not count or not length:
                assert all(it[0] != p for it in items)
                continue
            at = 0
            for piece in range(pieces):
                ends = set()
                for block in range(blocks):
                    it = items[base + piece * blocks + block]
                    assert it[:4] == [p, first, block * vp.BLOCK_ROWS, rows] and it[6] == length
                    assert it[4] == at and it[5] > it[4]
                    ends.add(it[5])
                at, = ends
            assert at == tiles
        assert len(items) == sum(1 for it in items)


def test_pieces_fill_the_card_once():
    plan = vp.prepare_prefix_plan([65536], [128], 40, 8, 128, device="cpu")
    assert 0.8 * 512 <= plan.items.shape[0] * 8 <= 448     # an eighth is left for the tails
    many = vp.prepare_prefix_plan([300] * 500, [2] * 500, 16, 16, 128, device="cpu")
    assert many.items.shape[0] == 500                    # more units than workgroups: none is cut
    assert vp.prepare_prefix_plan([], [], 2, 1, 64, device="cpu").batch == 0


def test_pieces_of_few_rows_are_whole_steps():
    """16 rows and fewer: four tiles at a time, of which only a prefix's last may be missing."""
    for lengths, counts in (([5000, 64, 1, 700, 65], [2, 1, 4, 2, 3]), ([100000], [4]), ([9000, 9000], [4, 30])):
        plan = vp.prepare_prefix_plan(lengths, counts, 32, 8, 128, device="cpu")
        seen = [0] * len(lengths)
        for p, first, row, rows, tile, end, tokens, _ in plan.items.tolist():
            assert rows == counts[p] * 4 and tokens == lengths[p] and tile < end
            if rows <= vp.FEW_ROWS:
                last = -(-tokens // vp.TILE)
                assert row == 0 and tile == seen[p] and tile % vp.FEW_STEP == 0
                assert end == last or end % vp.FEW_STEP == 0
                seen[p] = end
        assert all(n == -(-length // vp.TILE) for n, length, c in zip(seen, lengths, counts) if c * 4 <= vp.FEW_ROWS)


@pytest.mark.parametrize("args", [
    ([1], [1, 2], 2, 1, 64), ([-1], [1], 2, 1, 64), ([1.0], [1], 2, 1, 64), ([1], [-1], 2, 1, 64),
    ([1], [1], 3, 2, 64), ([1], [1], 0, 1, 64), ([1], [1], 2, 0, 64), ([1], [1], 2, 1, 96),
    ([2 ** 31], [1], 2, 1, 64), ([1], [2 ** 31], 2, 1, 64)])
def test_plans_refuse(args):
    with pytest.raises(ValueError):
        vp.prepare_prefix_plan(*args, device="cpu")


def test_tokens_refused():
    with pytest.raises(ValueError):
        vp.prepare_prefix_plan([1], [1], 2, 1, 64, tokens=0, device="cpu")


def test_calls_need_a_device_and_no_grad():
    c = kv.empty_cache(2, 1, 64, 16, device="cpu")
    plan = vp.prepare_prefix_plan([16], [1], 1, 1, 64, device="cpu")
    x, t, n = torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, 1).int(), torch.zeros(1).int()
    with pytest.raises(RuntimeError, match="inference-only"):
        vp.prefix_attention(x, c, t, plan, t, n)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        vp.prefix_attention(x, c, t, plan, t, n)


def test_entry_point_validates_before_launching():
    lib = _lib.load()

    def call(q=P, q_st=64, pages=4, page=16, dim=64, p_table=P, p_width=2, items=P, n=3, seqs=P, batch=2, width=2,
             tokens=1, group=1, dtype=0, scale=0.1, out=P, ws=P, nbytes=1 << 40):
        return lib.vdn_prefix_attention(q, 128, q_st, 64, P, P, P, P, P, pages, 2, page, dim, p_table, 2, p_width,
                                        items, n, 1, seqs, P, 2, batch, width, P, tokens, group, dtype, scale, out, 128,
                                        64, 64, None, ws, nbytes, None)

    for bad, said in ((dict(pages=0), b"geometry"), (dict(page=24), b"geometry"), (dict(dim=32), b"geometry"),
                      (dict(width=0), b"geometry"), (dict(p_width=0), b"geometry"), (dict(n=-1), b"geometry"),
                      (dict(p_width=1 << 28), b"geometry"), (dict(dtype=3), b"dtype"), (dict(scale=math.nan), b"scale"),
                      (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(seqs=None), b"null"),
                      (dict(items=None), b"null"), (dict(p_table=None), b"null"), (dict(q_st=4), b"alignment"),
                      (dict(items=P + 8), b"alignment"), (dict(seqs=P + 8), b"alignment"), (dict(out=P + 2), b"alignment"),
                      (dict(ws=None), b"workspace"), (dict(nbytes=1000), b"workspace"), (dict(ws=P + 8), b"workspace"),
                      (dict(batch=1 << 24), b"too many"), (dict(n=1 << 24), b"too many")):
        assert call(**bad) != 0, bad
        assert said in lib.vdn_last_error(), (bad, lib.vdn_last_error())
    assert call(batch=0, q=None) == 0
    n = ctypes.c_int64(0)
    assert lib.vdn_prefix_attention_workspace(3, 2, 2, 16, 1, 1, 2, 64, ctypes.addressof(n)) == 0
    assert n.value == 4 * 68 * (3 * 2 * 128 + 4)
    assert lib.vdn_prefix_attention_workspace(3, 2, 0, 16, 1, 1, 2, 64, ctypes.addressof(n)) != 0
    assert lib.vdn_prefix_attention_workspace(3, 2, 2, 16, 1, 1, 2, 64, None) != 0


def test_items_and_slots_of_a_plan_are_its_own():
    """Items: as many as pieces x blocks of the prefixes in order, none between them. Partial results: each row of each
    piece has a place, once, and nothing more is asked for."""
    r = random.Random(4)
    for _ in range(100):
        n = r.randint(1, 6)
        lengths = [r.choice((0, 1, 64, 65, r.randint(1, 70000))) for _ in range(n)]
        counts = [r.choice((0, 1, 2, r.randint(1, 200))) for _ in range(n)]
        heads, kv_heads = r.choice(((1, 1), (40, 8), (12, 2), (16, 16), (24, 1)))
        plan = vp.prepare_prefix_plan(lengths, counts, heads, kv_heads, r.choice((64, 128, 256)),
                                      tokens=r.choice((1, 1, 4)), device="cpu")
        items, seqs = plan.items.tolist(), plan.sequences.tolist()
        at_item = at_row = b = 0
        for length, count in zip(lengths, counts):
            if not count:
                continue
            first, base, pieces, blocks, _, slot, rows, _ = seqs[b]
            assert all(s == seqs[b] for s in seqs[b:b + count]) and first == b and rows == count * plan.tokens * heads // kv_heads
            b += count
            assert base == at_item and slot == at_row
            for piece in range(pieces):
                for it in items[base + piece * blocks:base + (piece + 1) * blocks]:
                    assert it[7] == at_row and it[3] == rows
                at_row += rows
            at_item += pieces * blocks
        assert len(items) == at_item and plan.slot_rows == at_row and b == len(seqs)


@pytest.mark.parametrize("prefixes,count,heads,kv_heads,dim", [(500, 2, 16, 16, 128), (2000, 1, 40, 8, 128),
                                                               (2000, 4, 32, 8, 256)])
def test_workspace_of_many_small_prefixes(prefixes, count, heads, kv_heads, dim):
    """What the rows need, not a block of 128 of them for each prefix."""
    plan = vp.prepare_prefix_plan([300] * prefixes, [count] * prefixes, heads, kv_heads, dim, device="cpu")
    rows = prefixes * count * heads                        # a piece each, and the tails' own
    n = ctypes.c_int64(0)
    assert _lib.load().vdn_prefix_attention_workspace(-(-plan.slot_rows // vp.BLOCK_ROWS), plan.batch, 2, 16, 1,
                                                      heads // kv_heads, kv_heads, dim, ctypes.addressof(n)) == 0
    assert 2 * rows <= n.value / (4 * (dim + 4)) < 2 * rows + vp.BLOCK_ROWS * kv_heads
