"""GPU: rotation of queries and keys by their positions against the definition in float64, within the
bound of oracle/rotary.py."""
import math

import pytest
import torch

from oracle import rotary as orot
from vdn_amd import rotary as vr

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def inputs(tokens, heads, kv_heads, dim, dtype, seed=0):
    """Column slices of one projection, on the device."""
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g).to(dtype).cuda()
    return qkv[:, :heads], qkv[:, heads:heads + kv_heads]


def check(out, x, positions, frequencies, plan, weight=None, eps=1e-6):
    value, size = orot.rotate(x.cpu(), positions.cpu(), frequencies, plan.layout, plan.amplitude,
                              None if weight is None else weight.cpu(), eps)
    off = (out.cpu().double() - value).abs()
    assert (off <= orot.tolerance(value, size, x.dtype)).all(), float(off.max())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,part", [(64, 64), (64, 8), (64, 24), (128, 128), (128, 96), (128, 16),
                                      (256, 256), (256, 64), (256, 136)])
@pytest.mark.parametrize("dtype,norm", [(BF16, None), (BF16, BF16), (FP16, FP16), (FP16, None),
                                        (BF16, torch.float32)])
@torch.no_grad()
def test_against_the_definition(device, layout, dim, part, dtype, norm):
    for tokens, heads, kv_heads in ((1, 1, 1), (37, 12, 2), (5, 16, 16), (300, 7, 1)):
        q, k = inputs(tokens, heads, kv_heads, dim, dtype, seed=tokens)
        g = torch.Generator().manual_seed(7)
        positions = torch.randint(-1000, 200000, (tokens,), generator=g).int().cuda()
        weights = [None if norm is None else (1 + 0.2 * torch.randn(dim, generator=g)).to(norm).cuda()
                   for _ in range(2)]
        scaling = dict(scaling="parts", factor=4.0, original=4096)
        plan = vr.prepare_rotary_plan(dim, rotary_dim=part, layout=layout, device="cuda", **scaling)
        frequencies, _ = vr.rotary_frequencies(part, **scaling)
        qo, ko = vr.rotate_qk(q, k, positions, plan, *weights)
        assert qo.is_contiguous() and ko.is_contiguous()
        check(qo, q, positions, frequencies, plan, weights[0])
        check(ko, k, positions, frequencies, plan, weights[1])


@torch.no_grad()
def test_many_tokens_and_one_norm_only(device):
    """Enough rows for workgroups of several tokens, with a ragged last one; only the keys are normed."""
    q, k = inputs(40003, 6, 2, 64, BF16)
    positions = torch.arange(40003).cuda()
    plan = vr.prepare_rotary_plan(64, layout="interleaved", device="cuda")
    w = torch.linspace(0.5, 1.5, 64).cuda()
    qo, ko = vr.rotate_qk(q, k, positions, plan, None, w, 1e-5)
    frequencies, _ = vr.rotary_frequencies(64)
    check(qo, q, positions, frequencies, plan)
    check(ko, k, positions, frequencies, plan, w, 1e-5)


@torch.no_grad()
def test_far_positions(device):
    """The angle of a position next to the ends of both integer types, from exact fractions of a turn."""
    from fractions import Fraction
    turn = Fraction("6.28318530717958647692528676655900576839433879875")
    at = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 53 + 1, 2 ** 62 - 1, -2 ** 63]
    plan = vr.prepare_rotary_plan(64, device="cuda")
    q, k = inputs(len(at), 2, 1, 64, FP16)
    steps = [s % 2 ** 64 for s in plan.steps.tolist()]
    qo, _ = vr.rotate_qk(q, k, torch.tensor(at).cuda(), plan)
    for t, p in enumerate(at):
        angles = [float(Fraction(p * s % 2 ** 64, 2 ** 64) * turn) for s in steps]
        value, size = orot.rotate(q[t:t + 1].cpu(), torch.ones(1), angles)
        off = (qo[t:t + 1].cpu().double() - value).abs()
        assert (off <= orot.tolerance(value, size, FP16)).all(), p
    narrow, _ = vr.rotate_qk(q[:5], k[:5], torch.tensor(at[:5], dtype=torch.int32).cuda(), plan)
    assert torch.equal(narrow, qo[:5])


@torch.no_grad()
def test_in_place_strides_and_nonfinite_rows(device):
    buffer = torch.randn(9, 4, 3, 128).to(BF16).cuda()
    q, k = buffer[:, :, 0].transpose(0, 1)[:, :5], buffer[:, :, 1].transpose(0, 1)[:, :2]   # heads outside
    q[1, 2, 5] = math.inf
    q[2, 0, 100] = math.nan
    plan = vr.prepare_rotary_plan(128, rotary_dim=64, device="cuda")
    positions = torch.tensor([3, 0, 7, 100000], dtype=torch.int32).cuda()
    qo, ko = vr.rotate_qk(q, k, positions, plan)
    frequencies, _ = vr.rotary_frequencies(64)
    clean = torch.ones(4, 5, dtype=torch.bool)
    clean[1, 2] = clean[2, 0] = False
    value, size = orot.rotate(q.cpu(), positions.cpu(), frequencies)
    off = (qo.cpu().double() - value).abs()
    assert (off <= orot.tolerance(value, size, BF16))[clean].all()
    # only the two channels of the infinity's pair are touched; a NaN that is not turned stays where it is
    bad = ~torch.isfinite(qo.cpu())
    assert bad[1, 2].nonzero().flatten().tolist() == [5, 37]
    assert bad[2, 0].nonzero().flatten().tolist() == [100] and int(bad.sum()) == 3
    beside = buffer[:, :, 2].clone()
    got = vr.rotate_qk(q, k, positions, plan, out=(q, k))
    assert got[0] is q and torch.equal(torch.nan_to_num(q), torch.nan_to_num(qo)) and torch.equal(k, ko)
    assert torch.equal(buffer[:, :, 2], beside)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@torch.no_grad()
def test_rows_at_odd_8_bytes(device, layout):
    """Rows that are 8-byte but not 16-byte aligned take the narrower pieces."""
    buffer = torch.randn(50, 9 * 128 + 4).to(FP16).cuda()
    plan = vr.prepare_rotary_plan(128, rotary_dim=96, layout=layout, device="cuda")
    positions = torch.arange(50).cuda()
    w = torch.rand(128).to(FP16).cuda()
    q, k = (buffer[:, 4 + a:4 + a + n * 128].unflatten(1, (n, 128)) for a, n in ((0, 7), (7 * 128, 2)))
    assert q.data_ptr() % 16 == 8
    want = vr.rotate_qk(q.contiguous(), k.contiguous(), positions, plan, w, w)
    got = vr.rotate_qk(q, k, positions, plan, w, w)
    for a, b in zip(got, want):      # the norm's sum is over 16 lanes instead of 8
        assert ((a.float() - b.float()).abs() <= torch.finfo(FP16).eps * b.float().abs() + 2.0 ** -24).all()
    frequencies, _ = vr.rotary_frequencies(96)
    check(got[0], q, positions, frequencies, plan, w)
    check(got[1], k, positions, frequencies, plan, w)


@torch.no_grad()
def test_rows_behind_2_31_elements(device):
    """Head rows of a strided buffer beyond 2^31 elements."""
    buffer = torch.empty(2 ** 31 + 2 ** 20, dtype=BF16, device="cuda")
    far = torch.as_strided(buffer, (3, 2, 64), (2 ** 30, 64, 1))
    far.copy_(torch.randn(3, 2, 64))
    near = far.contiguous()
    plan = vr.prepare_rotary_plan(64, device="cuda")
    positions = torch.arange(3, dtype=torch.int32).cuda()
    want = vr.rotate_qk(near, near, positions, plan)
    got = vr.rotate_qk(far, far, positions, plan)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@torch.no_grad()
def test_streams_graphs_and_no_tokens(device):
    q, k = inputs(64, 12, 2, 128, BF16)
    positions = torch.randint(0, 5000, (64,)).int().cuda()
    plan = vr.prepare_rotary_plan(128, device="cuda")
    want = vr.rotate_qk(q, k, positions, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = vr.rotate_qk(q, k, positions, plan)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = vr.rotate_qk(q, k, positions, plan)
    for seed in range(3):
        positions.copy_(torch.randint(0, 5000, (64,)).int())
        graph.replay()
        want = vr.rotate_qk(q, k, positions, plan)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    empty = vr.rotate_qk(q[:0], k[:0], positions[:0], plan)
    assert empty[0].shape == (0, 12, 128) and empty[1].shape == (0, 2, 128)


@torch.no_grad()
def test_refusals(device):
    q, k = inputs(4, 3, 1, 64, BF16)
    p = torch.zeros(4, dtype=torch.int32).cuda()
    plan = vr.prepare_rotary_plan(64, device="cuda")
    w = torch.ones(64, dtype=BF16).cuda()
    for call in (lambda: vr.rotate_qk(q[0], k, p, plan), lambda: vr.rotate_qk(q, k[:3], p, plan),
                 lambda: vr.rotate_qk(q, k.half(), p, plan), lambda: vr.rotate_qk(q.float(), k.float(), p, plan),
                 lambda: vr.rotate_qk(q, k, p[:3], plan), lambda: vr.rotate_qk(q, k, p.short(), plan),
                 lambda: vr.rotate_qk(q, k, p.cpu(), plan), lambda: vr.rotate_qk(q[:, :0], k, p, plan),
                 lambda: vr.rotate_qk(q[..., ::2], k[..., ::2], p, plan),
                 lambda: vr.rotate_qk(q, k, torch.zeros(8).int().cuda()[::2], plan),
                 lambda: vr.rotate_qk(q, k, p, vr.prepare_rotary_plan(128, device="cuda")),
                 lambda: vr.rotate_qk(q, k, p, vr.prepare_rotary_plan(64, device="cpu")),
                 lambda: vr.rotate_qk(q, k, p, plan, w.half()), lambda: vr.rotate_qk(q, k, p, plan, w[:32]),
                 lambda: vr.rotate_qk(q, k, p, plan, w, w.float()), lambda: vr.rotate_qk(q, k, p, plan, w.cpu()),
                 lambda: vr.rotate_qk(q, k, p, plan, eps=-1.0), lambda: vr.rotate_qk(q, k, p, plan, eps=math.nan),
                 lambda: vr.rotate_qk(q, k, p, plan, out=(k, q)),
                 lambda: vr.rotate_qk(q, k, p, plan, out=(q[:3], k)),
                 lambda: vr.rotate_qk(q, k, p, plan, out=(q.clone()[:, :1].expand(4, 3, 64), k))):
        with pytest.raises(ValueError):
            call()
    wide = torch.zeros(4, 8, 64, dtype=BF16).cuda()
    a, b, ahead = wide[:, :3], wide[:, 4:5], wide[:, 1:4]
    with pytest.raises(ValueError, match="overlap"):
        vr.rotate_qk(a, b, p, plan, out=(ahead, b))
    with pytest.raises(ValueError, match="overlap"):
        vr.rotate_qk(a, b, p, plan, out=(a, wide[:, 2:3]))
    with pytest.raises(ValueError, match="overlap"):
        vr.rotate_qk(a, b, p, plan, out=(wide[:, 4:7], b))
