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
