"""CPU: the frequencies of a rotation, their fractions of a turn, and what is refused."""
import math
from fractions import Fraction

import pytest
import torch

from oracle import rotary as orot
from vdn_amd import _lib
from vdn_amd import rotary as vr

F32, BF16 = torch.float32, torch.bfloat16


def test_frequencies():
    f, a = vr.rotary_frequencies(64)
    assert a == 1.0 and len(f) == 32 and f[0] == 1.0
    assert f == pytest.approx([10000 ** (-2 * j / 64) for j in range(32)], rel=1e-15)
    g, a = vr.rotary_frequencies(64, scaling="linear", factor=4)
    assert a == 1.0 and g == pytest.approx([x / 4 for x in f], rel=1e-15)
    # the fastest pair stays, the slowest is slower by the factor
    g, a = vr.rotary_frequencies(64, scaling="base", factor=8)
    assert a == 1.0 and g[0] == 1.0 and g[-1] == pytest.approx(f[-1] / 8, rel=1e-13)
    g, a = vr.rotary_frequencies(128, 500000.0, scaling="parts", factor=8, original=8192, parts=(1, 4))
    assert a == pytest.approx(0.1 * math.log(8) + 1)
    assert g == pytest.approx(orot.bands(500000.0, 128, 8, 8192, 1, 4), rel=1e-14)
    assert vr.rotary_frequencies(2)[0] == [1.0]


def test_steps_are_turns():
    """position * step, modulo 2^64, is the fraction of a turn to within position / 2^65."""
    plan = vr.prepare_rotary_plan(128, rotary_dim=96, base=10000.0, device="cpu")
    assert plan.steps.shape == (48,) and plan.device == torch.device("cpu")
    frequencies, _ = vr.rotary_frequencies(96)
    turn = Fraction("6.28318530717958647692528676655900576839433879875")
    for f, step in zip(frequencies, plan.steps.tolist()):
        for p in (1, 2, 1000003, -77, 2 ** 31 - 1):
            exact = Fraction(f) * p / turn
            off = Fraction(p * (step % 2 ** 64) % 2 ** 64, 2 ** 64) - exact
            off -= round(off)
            assert abs(off) <= Fraction(abs(p), 2 ** 65) + Fraction(1, 2 ** 70)


@pytest.mark.parametrize("kwargs", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=64.0), dict(base=1.0), dict(base=math.inf),
    dict(scaling="other"), dict(factor=2.0), dict(scaling="linear", factor=0.5),
    dict(scaling="linear", factor=math.nan), dict(scaling="parts", factor=2.0), dict(original=100),
    dict(scaling="parts", factor=2.0, original=0), dict(scaling="base", factor=2.0, rotary_dim=2),
    dict(scaling="parts", factor=2.0, original=100, parts=(4.0, 4.0))])
def test_frequencies_refuse(kwargs):
    with pytest.raises(ValueError):
        vr.rotary_frequencies(**{"rotary_dim": 64, **kwargs})


@pytest.mark.parametrize("kwargs", [
    dict(head_dim=96), dict(rotary_dim=12), dict(rotary_dim=136), dict(rotary_dim=0), dict(rotary_dim=4),
    dict(layout="pairs"), dict(amplitude=math.inf)])
def test_plans_refuse(kwargs):
    with pytest.raises(ValueError):
        vr.prepare_rotary_plan(**{"head_dim": 128, "device": "cpu", **kwargs})


def test_calls_need_a_device_and_no_grad():
    plan = vr.prepare_rotary_plan(64, device="cpu")
    q, p = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="inference-only"):
        vr.rotate_qk(q, q, p, plan)
    with torch.no_grad():
        with pytest.raises(ValueError, match="CUDA"):
            vr.rotate_qk(q, q, p, plan)
        with pytest.raises(TypeError):
            vr.rotate_qk(q, q, p, None)


def test_entry_point_validates_before_launching():
    lib, p = _lib.load(), 1 << 20

    def call(q=p, st=128, w=None, w_f32=0, eps=1e-6, positions=p, wide=0, steps=p, rot=64, amplitude=1.0,
             tokens=4, heads=2, kv=2, dim=64, dtype=0, out=p):
        return lib.vdn_rotary(q, st, 64, p, 128, 64, w, None, w_f32, eps, positions, wide, steps, rot, 0,
                              amplitude, tokens, heads, kv, dim, dtype, out, 128, 64, p, 128, 64, None)

    for bad, said in ((dict(dim=96), b"head_dim"), (dict(rot=4), b"rotated"), (dict(rot=72), b"rotated"),
                      (dict(rot=12), b"rotated"), (dict(tokens=-1), b"tokens"), (dict(heads=0), b"heads"),
                      (dict(kv=0), b"heads"), (dict(heads=1 << 20), b"heads"), (dict(dtype=2), b"dtype"),
                      (dict(amplitude=math.nan), b"amplitude"), (dict(eps=-1.0), b"eps"),
                      (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(steps=None), b"null"),
                      (dict(positions=None), b"null"), (dict(st=126), b"alignment"),
                      (dict(q=p + 4), b"alignment"), (dict(positions=p + 4, wide=1), b"alignment"),
                      (dict(w=p + 1), b"alignment"), (dict(w=p + 2, w_f32=1), b"alignment"),
                      (dict(tokens=1 << 40), b"too many")):
        assert call(**bad) != 0, bad
        assert said in lib.vdn_last_error(), (bad, lib.vdn_last_error())
    assert call(tokens=0, q=None) == 0
