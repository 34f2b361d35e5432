"""GPU: causal attention at the edges of its types, against the formula in 64 bits."""
import math

import pytest
import torch

from oracle import causal as oc
from vdn_amd import causal as vc

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def plan_of(lengths, heads, kv_heads, block_rows, device):
    """The plan of these sequences, with 256-row blocks also where it would not take them."""
    plan = vc.prepare_causal_plan(lengths, heads, kv_heads, device=device)
    if block_rows == 256:
        wide = vc._blocks(tuple(lengths), heads // kv_heads, 256).to(device)
        plan = vc.CausalPlan(plan.lengths, heads, kv_heads, plan.rows, plan.blocks, wide)
    return plan


VARIANTS = [(64, 128), (128, 128), (128, 256), (256, 128)]   # head_dim, block rows


@pytest.mark.parametrize("dim,block_rows", VARIANTS)
@torch.no_grad()
def test_fp16_means_of_the_largest_value(device, dim, block_rows):
    """Every value is 65504, so every output is. All weights but one lie a little over the middle of
    two fp16 numbers, 1/2 + 2^-12, and are rounded up by 2^-11 relative: 2^-12 of that takes the mean
    to where fp16 has an infinity."""
    n = 700
    q = torch.zeros(n, 1, dim, dtype=FP16, device=device)
    q[..., 0] = 1.0
    k = torch.zeros_like(q)
    k[1:, :, 0] = -1.0
    v = torch.full_like(q, 65504.0)
    v[..., 1] = -65504.0
    scale = -math.log(0.5 + 2.0 ** -12 + 2.0 ** -16)
    got = vc.causal_attention(q, k, v, plan_of([n], 1, 1, block_rows, device), scale)
    assert (got[..., 0] == 65504).all() and (got[..., 1] == -65504).all()
    assert torch.isfinite(got).all()
    v[n - 1, 0, 2], v[n - 1, 0, 3] = math.inf, -math.inf          # infinities stay
    got = vc.causal_attention(q, k, v, plan_of([n], 1, 1, block_rows, device), scale)
    assert got[n - 1, 0, 2] == math.inf and got[n - 1, 0, 3] == -math.inf
    assert torch.isfinite(got[:n - 1]).all()


@pytest.mark.parametrize("dim,block_rows", VARIANTS)
@pytest.mark.parametrize("heads,dtype", [(2, BF16), (2, FP16), (1, BF16), (1, FP16)])
@torch.no_grad()
def test_infinite_values_in_front_of_a_steep_rise(device, dim, block_rows, heads, dtype):
    """Scores rise by 288 binary orders from one tile of a block's diagonal to the next, so that fp32
    keeps nothing of what was summed before. An infinity of a token that a row sees, in the tile
    before the rise or in that of the rise, is in its output all the same; rows before it are as
    without it."""
    n, rise = 300, 70
    q = torch.zeros(n, heads, dim)
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, dim)
    k[rise:, :, 0] = 200.0
    v = torch.randn(n, 1, dim, generator=torch.Generator().manual_seed(2))
    q, k, v = (x.to(dtype).cuda() for x in (q, k, v))
    plan = plan_of([n], heads, 1, block_rows, device)
    clean = vc.causal_attention(q, k, v, plan, 1.0)
    notes = ((5, 3, math.inf), (5, 4, -math.inf), (rise, 9, math.inf), (rise + 1, 10, -math.inf))
    bad = v.clone()
    for token, channel, value in notes:
        bad[token, 0, channel] = value
    block = block_rows // heads                    # tokens of the first block
    for _ in range(3):
        got = vc.causal_attention(q, k, bad, plan, 1.0)
        for token, channel, value in notes:
            assert torch.equal(got[:token, :, channel], clean[:token, :, channel])
            assert (got[token:block, :, channel] == value).all()
            assert not torch.isfinite(got[max(block, token):, :, channel]).any()
        others = [c for c in range(dim) if c not in (3, 4, 9, 10)]
        assert torch.equal(got[..., others], clean[..., others])


@pytest.mark.parametrize("dim,block_rows", VARIANTS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@torch.no_grad()
def test_rows_without_weight_are_nan_also_over_infinite_values(device, dim, block_rows, dtype):
    """All scores of the first rows are -inf: no weights exist, so every channel is NaN, those with an
    infinity among the values too."""
    n, shut = 200, 90
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(n, 1, dim, generator=g) for _ in range(3))
    q[..., 5] = 1.0
    k[:shut, :, 5] = -math.inf
    v[3, 0, 7], v[40, 0, 8] = math.inf, -math.inf
    q, k, v = (x.to(dtype).cuda() for x in (q, k, v))
    got, lse = vc.causal_attention(q, k, v, plan_of([n], 1, 1, block_rows, device), return_lse=True)
    assert got[:shut].isnan().all() and torch.isneginf(lse[:shut]).all()
    others = [c for c in range(dim) if c not in (7, 8)]
    assert torch.isfinite(got[shut:][..., others]).all() and torch.isfinite(lse[shut:]).all()


@pytest.mark.parametrize("dim,block_rows", VARIANTS)
@pytest.mark.parametrize("heavy", [0, 20000])
@torch.no_grad()
def test_fp16_weights_that_are_small_but_many(device, dim, block_rows, heavy):
    """32767 tokens of weight 2^-25.3 relative to a heavy one, whose value is 0: their sum is the
    output. A weight is rounded to within 2^-36 of the largest or to half a step of fp16, the output
    to half a step or 2^-25 (the bound's own terms, 2^-25 for each weight and 2^-14, are larger)."""
    n = 32768
    q = torch.zeros(n, 1, dim)
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, dim)
    k[heavy, 0, 0] = 17.53
    v = torch.rand(n, 1, dim, generator=torch.Generator().manual_seed(3)) + 0.5
    v[heavy] = 0.0
    q, k, v = (x.to(FP16) for x in (q, k, v))
    got, lse = vc.causal_attention(q.cuda(), k.cuda(), v.cuda(), plan_of([n], 1, 1, block_rows, device), 1.0,
                                   return_lse=True)
    for a, b in ((32752, n), (25000, 25010), (heavy + 100, heavy + 105)):
        out, el, mass, size = oc.attention(q[a:b], k[:b], v[:b], a, 1.0)
        tol, ltol = oc.bounds(out, mass, size, v[:b], FP16, dim, b)
        top = float(v.abs().max())
        tol += b * (2.0 ** -36 - 2.0 ** -25) * top + 2.0 ** -25 - torch.finfo(FP16).tiny
        err = (got[a:b].cpu().double() - out).abs()
        assert bool((err <= tol).all()), f"rows {a}: worst {float((err / tol).max())}"
        assert bool(((lse[a:b].cpu().double() - el).abs() <= ltol).all())


@pytest.mark.parametrize("dim,block_rows", VARIANTS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@torch.no_grad()
def test_the_output_over_its_queries(device, dim, block_rows, dtype):
    """A workgroup has read its rows before it writes them: out = query gives what a fresh output
    does, also as a column slice beside key and value. What others still read is refused."""
    lengths, heads, kv_heads = [200, 1, 300], 6, 2
    g = torch.Generator().manual_seed(6)
    fused = torch.randn(510, heads + 2 * kv_heads, dim, generator=g).to(dtype).cuda()
    q, k, v = fused.split((heads, kv_heads, kv_heads), 1)
    plan = plan_of(lengths, heads, kv_heads, block_rows, device)
    want = vc.causal_attention(q, k, v, plan)
    rest = q[501:].clone()
    for out in (fused[:, 1:7], fused[:, 3:9], fused[:, 4:10]):
        with pytest.raises(ValueError, match="overlap"):
            vc.causal_attention(q, k, v, plan, out=out)
    with pytest.raises(ValueError, match="itself"):
        vc.causal_attention(q, k, v, plan, out=torch.zeros(510 * heads * dim, dtype=dtype, device=device)
                            .as_strided((510, heads, dim), (dim * (heads - 1), dim, 1)))
    assert torch.equal(vc.causal_attention(q, k, v, plan), want)      # nothing was written
    got = vc.causal_attention(q, k, v, plan, out=q)
    assert got is q and torch.equal(q[:501], want[:501]) and torch.equal(q[501:], rest)
