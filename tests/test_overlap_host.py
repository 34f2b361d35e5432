"""CPU: which outputs of an attention share memory with themselves or its inputs, against the
elements' addresses one by one."""
import itertools
import random

import pytest
import torch

from vdn_amd import _lib


def addresses(t):
    base = t.data_ptr() // t.element_size()
    return [base + sum(i * s for i, s in zip(at, t.stride()))
            for at in itertools.product(*(range(n) for n in t.shape))]


def test_against_every_address():
    r = random.Random(1)
    said = [0, 0]
    for _ in range(4000):
        buffer, dim = torch.empty(700, dtype=torch.bfloat16), r.choice((2, 4))

        def view(row):
            heads = r.choice((0, dim, dim + 1, 2 * dim, 40))
            return buffer.as_strided((r.randint(1, 4), r.randint(1, 3), dim), (row, heads, 1), r.randint(0, 99))
        row = r.choice((0, dim, 9, 24, 60))
        a, b = view(row), view(row)
        mine = addresses(a)
        assert _lib.overlaps_itself(a) == (len(set(mine)) < len(mine))
        if row:
            share = bool(set(mine) & set(addresses(b)))
            assert _lib.overlap(a, b) == share
            said[share] += 1
        c = view(r.choice((7, 50)))
        assert not _lib.overlap(a, c) or set(mine) & set(addresses(c))
    assert min(said) > 500


def test_outputs_of_an_attention():
    fused = torch.zeros(9, 4 + 2 + 2 + 4, 64)
    q, k, v, rest = fused.split((4, 2, 2, 4), 1)
    for out in (torch.empty(9, 4, 64), rest, q, torch.empty(4, 9, 64).transpose(0, 1), fused[:, :4]):
        _lib.check_attention_out(out, q, k, v)
    turns = torch.zeros(9, 4, 3, 64)                    # q, k, v of a head beside each other
    _lib.check_attention_out(turns[:, :, 0], *(turns[:, :, i] for i in range(3)))
    _lib.check_attention_out(torch.zeros(9, 4, 80)[..., 8:72], q, k, v)
    for out in (fused[:, 2:6], fused[:, 3:7], fused[:, 5:9]):
        with pytest.raises(ValueError, match="key or value"):
            _lib.check_attention_out(out, q, k, v)
    with pytest.raises(ValueError, match="query itself"):
        _lib.check_attention_out(fused[:, 1:5], q)
    with pytest.raises(ValueError, match="query itself"):
        _lib.check_attention_out(fused[:8, :4], fused[1:, :4])
    with pytest.raises(ValueError, match="query itself"):
        _lib.check_attention_out(torch.as_strided(q, (9, 4, 64), (768, 64, 1), 64), q)
    with pytest.raises(ValueError, match="key or value"):
        _lib.check_attention_out(turns[:, :, 1], *(turns[:, :, i] for i in range(3)))
    for strides in ((64, 64, 1), (256, 32, 1), (200, 64, 1)):
        with pytest.raises(ValueError, match="itself"):
            _lib.check_attention_out(torch.zeros(9000).as_strided((9, 4, 64), strides), q)
    steps = torch.zeros(2, 3, 4, 64)
    _lib.check_attention_out(steps, steps)
    _lib.check_attention_out(steps[:, :, :2], steps[:, :, 2:])
    with pytest.raises(ValueError, match="query itself"):
        _lib.check_attention_out(steps[:, :2], steps[:, 1:])
