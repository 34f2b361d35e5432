"""GPU: causal attention over packed prompts against the float64 oracle, within bounds derived
from the roundings (oracle/causal.py)."""
import math

import pytest
import torch

from oracle import causal as oc
from vdn_amd import causal as vc

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def make(lengths, heads, kv_heads, dim, dtype, seed=0, pad=0, amp=1.0):
    """Q, K, V as column slices of one wide buffer."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(lengths) + pad
    qkv = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g) * amp
    qkv = qkv.to(dtype).cuda()
    return qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]


def check(q, k, v, lengths, got, lse=None, scale=None):
    dim, dtype = q.shape[2], q.dtype
    scale = dim ** -0.5 if scale is None else scale
    n = sum(lengths)
    out, el, mass, size = oc.packed(q[:n].cpu(), k[:n].cpu(), v[:n].cpu(), lengths, scale)
    tol, ltol = oc.bounds(out, mass, size, v[:n].cpu(), dtype, dim, max(lengths))
    err = (got[:n].cpu().double() - out).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).max()}"
    if lse is not None:
        lerr = (lse[:n].cpu().double() - el).abs()
        assert bool((lerr <= ltol).all()), f"worst LSE {(lerr / ltol).max()}"


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16), (256, BF16),
                                       (256, FP16)])
@pytest.mark.parametrize("lengths", [[1], [2], [31], [129], [1, 0, 77, 3], [300, 1, 1, 64, 0, 257]])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 2), (14, 2), (9, 1), (16, 8)])
@torch.no_grad()
def test_against_oracle(device, dim, dtype, lengths, heads, kv_heads):
    q, k, v = make(lengths, heads, kv_heads, dim, dtype)
    plan = vc.prepare_causal_plan(lengths, heads, kv_heads, device=device)
    got, lse = vc.causal_attention(q, k, v, plan, return_lse=True)
    check(q, k, v, lengths, got, lse)


@pytest.mark.parametrize("dim,dtype,n,heads,kv_heads", [
    (64, BF16, 2049, 4, 4), (128, BF16, 1500, 7, 1), (128, FP16, 1023, 40, 1), (256, BF16, 1100, 3, 3),
    (128, BF16, 2305, 16, 16)])
@torch.no_grad()
def test_long(device, dim, dtype, n, heads, kv_heads):
    q, k, v = make([n], heads, kv_heads, dim, dtype, seed=3)
    plan = vc.prepare_causal_plan([n], heads, kv_heads, device=device)
    got, lse = vc.causal_attention(q, k, v, plan, return_lse=True)
    check(q, k, v, [n], got, lse)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([130, 1, 0, 700], 6, 2), ([513], 1, 1)])
@torch.no_grad()
def test_wide_blocks(device, dtype, lengths, heads, kv_heads):
    """The 256-row blocks, which the plan takes for long prompts, on small ones: within the bounds, and
    nonfinite values of later tokens stay away from a row there too."""
    q, k, v = make(lengths, heads, kv_heads, 128, dtype, seed=9)
    wide = vc._blocks(tuple(lengths), heads // kv_heads, 256).to(device)
    plan = vc.CausalPlan(tuple(lengths), heads, kv_heads, sum(lengths), wide, wide)
    got, lse = vc.causal_attention(q, k, v, plan, return_lse=True)
    check(q, k, v, lengths, got, lse)
    bad, last = v.clone(), sum(lengths) - 1
    bad[last] = math.inf
    same = vc.causal_attention(q, k, bad, plan)
    assert torch.equal(same[:last], got[:last]) and (same[last] == math.inf).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@torch.no_grad()
def test_long_prompt_takes_the_wide_blocks(device, dtype):
    """4200 tokens, 32 heads: the first and last rows, against the oracle of those rows."""
    n = 4200
    q, k, v = make([n], 32, 8, 128, dtype, seed=13)
    plan = vc.prepare_causal_plan([n], 32, 8, device=device)
    assert plan.wide_blocks is not None
    got, lse = vc.causal_attention(q, k, v, plan, return_lse=True)
    for a, b in ((0, 70), (2000, 2040), (n - 40, n)):
        out, el, mass, size = oc.attention(q[a:b].cpu(), k[:b].cpu(), v[:b].cpu(), a, 128 ** -0.5)
        tol, ltol = oc.bounds(out, mass, size, v[:b].cpu(), dtype, 128, b)
        assert bool(((got[a:b].cpu().double() - out).abs() <= tol).all())
        assert bool(((lse[a:b].cpu().double() - el).abs() <= ltol).all())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@torch.no_grad()
def test_scores_that_grow_and_another_scale(device, dtype):
    """Key magnitudes that ramp up: the running maximum is raised from tile to tile."""
    lengths = [900, 333]
    q, k, v = make(lengths, 6, 2, 128, dtype, seed=5, amp=3.0)
    k = (k.float() * torch.linspace(0.1, 4, k.shape[0], device=device)[:, None, None]).to(dtype)
    plan = vc.prepare_causal_plan(lengths, 6, 2, device=device)
    got, lse = vc.causal_attention(q, k, v, plan, 0.25, return_lse=True)
    check(q, k, v, lengths, got, lse, scale=0.25)


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@torch.no_grad()
def test_nonfinite_values_stay_with_the_rows_that_see_them(device, dim, dtype):
    """Nonfinite K and V of a token: rows before it and other sequences are as without it, bit for
    bit; rows from it on are nonfinite where a value is, with an infinity's sign."""
    lengths, at = [140, 90], 61
    q, k, v = make(lengths, 4, 2, dim, dtype, seed=7)
    plan = vc.prepare_causal_plan(lengths, 4, 2, device=device)
    clean = vc.causal_attention(q, k, v, plan)
    bad = v.clone()
    bad[at, 0, 3] = math.inf
    bad[at, 0, 9] = -math.inf
    bad[at, 0, 17] = math.nan
    bad[at + 2, 0, 3] = -math.inf
    got = vc.causal_attention(q, k, bad, plan)
    same = torch.ones(sum(lengths), dtype=torch.bool)
    same[at:140] = False
    assert torch.equal(got[same.cuda()], clean[same.cuda()])
    assert torch.equal(got[:, 2:], clean[:, 2:])          # heads of the other K/V head
    assert (got[at:at + 2, :2, 3] == math.inf).all() and got[at + 2:140, :2, 3].isnan().all()
    assert (got[at:140, :2, 9] == -math.inf).all() and got[at:140, :2, 17].isnan().all()
    other = [c for c in range(dim) if c not in (3, 9, 17)]
    assert torch.equal(got[at:140, :2][..., other], clean[at:140, :2][..., other])
    bad = k.clone()
    bad[at, 0] = math.nan
    got = vc.causal_attention(q, bad, v, plan)
    assert torch.equal(got[same.cuda()], clean[same.cuda()])
    assert got[at:140, :2].isnan().all()


@torch.no_grad()
def test_rows_behind_the_last_sequence(device):
    lengths = [65, 40]
    q, k, v = make(lengths, 4, 4, 64, BF16, pad=9)
    k[105:], v[105:] = math.nan, math.inf
    plan = vc.prepare_causal_plan(lengths, 4, 4, device=device)
    got, lse = vc.causal_attention(q, k, v, plan, return_lse=True)
    check(q, k, v, lengths, got, lse)
    assert got[105:].count_nonzero() == 0 and torch.isneginf(lse[105:]).all()
    wide = torch.full((114, 6, 72), 5.0, dtype=BF16, device=device)
    ret = vc.causal_attention(q, k, v, plan, out=wide[:, 1:5, 8:])
    assert ret.data_ptr() == wide[:, 1:5, 8:].data_ptr()
    assert torch.equal(ret[:105], got[:105])
    wide[:105, 1:5, 8:] = 5.0
    assert (wide == 5.0).all()


@torch.no_grad()
def test_strides_and_shared_keys(device):
    """Head-major storage, and K/V of one head broadcast over four."""
    lengths = [150]
    g = torch.Generator().manual_seed(1)
    q = torch.randn(4, 150, 128, generator=g).to(BF16).cuda().transpose(0, 1)
    k1, v1 = (torch.randn(150, 1, 128, generator=g).to(BF16).cuda() for _ in range(2))
    k, v = k1.expand(150, 4, 128), v1.expand(150, 4, 128)
    got = vc.causal_attention(q, k, v, vc.prepare_causal_plan(lengths, 4, 4, device=device))
    check(q, k, v, lengths, got)
    shared = vc.causal_attention(q, k1, v1, vc.prepare_causal_plan(lengths, 4, 1, device=device))
    check(q, k1, v1, lengths, shared)


@torch.no_grad()
def test_no_rows(device):
    for lengths in ([], [0, 0]):
        q, k, v = make(lengths, 4, 2, 128, BF16, pad=3)
        plan = vc.prepare_causal_plan(lengths, 4, 2, device=device)
        assert vc.causal_attention(q, k, v, plan).count_nonzero() == 0
        assert vc.causal_attention(q[:0], k[:0], v[:0], plan).shape == (0, 4, 128)


@torch.no_grad()
def test_side_stream_and_graph(device):
    """On a side stream; captured once and replayed with new inputs and eager work in between."""
    lengths = [200, 60]
    q, k, v = (t.contiguous() for t in make(lengths, 8, 2, 128, BF16, seed=11))
    plan = vc.prepare_causal_plan(lengths, 8, 2, device=device)
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = vc.causal_attention(q, k, v, plan)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        vc.causal_attention(q, k, v, plan, out=out)
    for i in range(4):
        if i:
            q.copy_(make(lengths, 8, 2, 128, BF16, seed=20 + i)[0])
        out.zero_()
        graph.replay()
        want = vc.causal_attention(q, k, v, plan)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        if i == 0:
            assert torch.equal(out, first)


@torch.no_grad()
def test_refusals(device):
    q, k, v = make([40], 4, 2, 128, BF16)
    plan = vc.prepare_causal_plan([40], 4, 2, device=device)
    with pytest.raises(ValueError, match="match the plan"):
        vc.causal_attention(q[:39], k[:39], v[:39], plan)
    with pytest.raises(ValueError, match="match the plan"):
        vc.causal_attention(q, k[:, :1], v[:, :1], plan)
    with pytest.raises(ValueError, match="match the plan"):
        vc.causal_attention(q[..., :96], k[..., :96], v[..., :96], plan)
    with pytest.raises(ValueError, match="share"):
        vc.causal_attention(q, k.half(), v, plan)
    with pytest.raises(ValueError, match="same CUDA device"):
        vc.causal_attention(q, k, v.cpu(), plan)
    with pytest.raises(ValueError, match="same CUDA device"):
        vc.causal_attention(q, k, v, vc.prepare_causal_plan([40], 4, 2))
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            vc.causal_attention(q, k, v, plan, scale)
    with pytest.raises(ValueError, match="out"):
        vc.causal_attention(q, k, v, plan, out=torch.empty_like(q, dtype=FP16))
    with pytest.raises(ValueError, match="out"):
        vc.causal_attention(q, k, v, plan, out=torch.empty(40, 1, 128, dtype=BF16, device=device).expand(40, 4, 128))
    with pytest.raises(RuntimeError, match="16-byte"):
        odd = torch.zeros(40, 4, 132, dtype=BF16, device=device)[..., 4:]
        vc.causal_attention(odd, k, v, plan)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="inference-only"):
        vc.causal_attention(q, k, v, plan)


@pytest.mark.parametrize("dim,dtype,block_rows", [(64, FP16, 128), (128, BF16, 128), (128, BF16, 256),
                                                  (256, BF16, 128)])
@torch.no_grad()
def test_keys_that_score_minus_infinity(device, dim, dtype, block_rows):
    """The first keys score -inf against every query, whole tiles of them: they get weight 0, and
    rows that see no others are NaN with LSE -inf."""
    n, shut = 451, 200
    q, k, v = (x.clone() for x in make([n], 4, 2, dim, dtype, seed=13))
    q[..., 5] = 1.0
    k[:shut, :, 5] = -math.inf
    plan = vc.prepare_causal_plan([n], 4, 2, device=device)
    if block_rows == 256:
        wide = vc._blocks((n,), 2, 256).cuda()
        plan = vc.CausalPlan(plan.lengths, 4, 2, n, plan.blocks, wide)
    got, lse = vc.causal_attention(q, k, v, plan, return_lse=True)
    assert got[:shut].isnan().all() and (lse[:shut] == -math.inf).all()
    check(q[shut:], k[shut:], v[shut:], [n - shut], got[shut:], lse[shut:])


@torch.no_grad()
def test_rows_behind_two_to_the_31_elements(device):
    """Rows of a wide buffer: the last sequence and the end of the first lie behind 2^31 elements."""
    lengths, wide = [33000, 70], 66000
    rows = sum(lengths)
    base = torch.empty(rows, wide, dtype=BF16, device=device)
    q, k, v = make(lengths, 2, 1, 64, BF16, seed=17)
    far = [base[:, 128 * i:128 * i + x.shape[1] * 64].unflatten(1, (-1, 64)) for i, x in enumerate((q, k, v, q))]
    for x, y in zip(far, (q, k, v)):
        x.copy_(y)
    plan = vc.prepare_causal_plan(lengths, 2, 1, device=device)
    got = vc.causal_attention(*far[:3], plan, out=far[3])
    assert got is far[3] and torch.equal(got, vc.causal_attention(q, k, v, plan))
    check(q[lengths[0]:], k[lengths[0]:], v[lengths[0]:], lengths[1:], got[lengths[0]:])
