"""GPU: attention whose scores are as large as fp32 holds them well: far beyond the range in which their steps are
under one, so that a row's weights are one and zeros. What the exponents are taken relative to has to be kept within
the weights' range of the largest score there, too."""
import pytest
import torch

from oracle import causal as oc
from test_prefix_gpu import Batch, ints, queries, values_of
from vdn_amd import causal as vc
from vdn_amd import kvcache as kv
from vdn_amd import sparse as sp
from vdn_amd import window as vw

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
# scores around 2^6 (ordinary) to 2^60 (about the largest whose errors stay within fp32 by far)
FAR = [0.7312 * 2.0 ** e for e in (3, 12, 19, 21, 22, 23, 24, 25, 27, 30, 33, 40, 57)]


def check_decided(q, k, v, first, scale, out, lse):
    """Rows of q over k, v; returns how many of them have one weight."""
    want, near, top, l_near, sure = oc.decided(q, k, v, first, scale)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert (out.abs() <= 1.02 * v.double().abs().max()).all()
    assert ((out - want).abs() <= near)[sure].all(), float(((out - want).abs() - near)[sure].max())
    assert ((lse - top).abs() <= l_near)[sure].all()
    return int(sure.sum())


# ------------------------------------------------------------ cache, selection, tails ----

@pytest.mark.parametrize("dim,dtype,page", [(64, BF16, 16), (64, FP16, 64), (128, BF16, 64), (128, FP16, 16), (256, BF16, 32),
                                            (256, FP16, 128)])
@pytest.mark.parametrize("heads", [6, 40])                            # row blocks of 16 and of 32
@pytest.mark.parametrize("wide", [False, True])                       # whole units, and units that are split
@torch.no_grad()
def test_cache_attention(device, dim, dtype, page, heads, wide):
    case = Batch([], [], [300, 2, 500, 257] + ([900, 1500] if wide else []), 2, dim, page)
    q = queries(len(case.tails), 2, heads, dim, dtype)
    k_all, v_all = values_of(case.cache)
    for scale in FAR:
        scale *= 2.0 ** 5 / dim
        out, lse = kv.cache_attention(q, case.cache, case.table.cuda(), ints(*case.tails), scale, return_lse=True)
        sure = 0
        for b, m in enumerate(case.tails):
            k, v = (case.keys(case.table[b], m, s) for s in (k_all, v_all))
            for i in range(2):
                sure += check_decided(q[b, i:i + 1].cpu(), k[:m - 1 + i], v[:m - 1 + i], m - 1 + i, scale,
                                      out[b, i:i + 1], lse[b, i:i + 1])
        assert scale < 2 ** 10 or sure > 0.7 * lse.numel(), (scale, sure)
    case.cache.check()


@pytest.mark.parametrize("dim,dtype,page", [(64, FP16, 64), (128, BF16, 64), (128, FP16, 16), (256, FP16, 128)])
@torch.no_grad()
def test_few_rows_and_tails(device, dim, dtype, page):
    """Few rows of a prefix and tails, which take the cache's own code, and the selection's."""
    case = Batch([300, 1000], [1, 2], [500, 400, 270], 2, dim, page)
    q = queries(3, 1, 6, dim, dtype)
    plan = case.plan(6)
    k_all, v_all = values_of(case.cache)
    page_ids = case.table[:, None, None].expand(-1, 1, 2, -1).contiguous().cuda()
    for scale in FAR:
        scale *= 2.0 ** 5 / dim
        out, lse = case.run(q, plan, scale=scale, return_lse=True)
        tail, tail_lse = sp.selected_attention(q, case.cache, page_ids, ints(*case.tails).view(3, 1), scale, return_lse=True)
        sure = 0
        for b, p in enumerate(case.owner):
            n, m = case.prefixes[p], case.tails[b]
            own = [case.keys(case.table[b], m, s) for s in (k_all, v_all)]
            both = [torch.cat((case.keys(case.shared[p], n, s), x)) for s, x in zip((k_all, v_all), own)]
            sure += check_decided(q[b].cpu(), *both, n + m, scale, out[b], lse[b])
            sure += check_decided(q[b].cpu(), *own, m, scale, tail[b], tail_lse[b])
        assert scale < 2 ** 10 or sure > 25, (scale, sure)            # of 36
    case.cache.check()


# ---------------------------------------------------------------------- prefixes ----

@pytest.mark.parametrize("dim,dtype,page", [(64, BF16, 16), (64, FP16, 64), (128, BF16, 64), (128, FP16, 32), (256, BF16, 32),
                                            (256, FP16, 128)])
@torch.no_grad()
def test_prefix_blocks(device, dim, dtype, page):
    """Blocks of rows: 34 of each K/V head behind the first prefix, 68 behind the second."""
    case = Batch([300, 65], [1, 2], [5, 0, 70], 2, dim, page)
    q = queries(3, 2, 34, dim, dtype)
    plan = case.plan(34, 2)
    k_all, v_all = values_of(case.cache)
    for scale in FAR:
        scale *= 2.0 ** 5 / dim
        out, lse = case.run(q, plan, scale=scale, return_lse=True)
        sure = 0
        for b, p in enumerate(case.owner):
            n, m = case.prefixes[p], case.tails[b]
            k, v = (torch.cat((case.keys(case.shared[p], n, s), case.keys(case.table[b], m, s))) for s in (k_all, v_all))
            for i in range(2):
                sees = n + max(0, m - 1 + i)
                sure += check_decided(q[b, i:i + 1].cpu(), k[:sees], v[:sees], sees, scale, out[b, i:i + 1], lse[b, i:i + 1])
        assert scale < 2 ** 10 or sure > 150, (scale, sure)        # of 204
    case.cache.check()


@pytest.mark.parametrize("page", [16, 64])
@torch.no_grad()
def test_prefix_keys_behind_the_last_where_scales_vanish(device, page):
    """A page's scale times a small softmax scale may be zero in fp32: a key that is not there stays hidden."""
    case = Batch([70], [20], [0] * 20, 1, 64, page)
    c = case.cache
    c.k_codes.zero_()
    c.k_scales.fill_(27)                                              # 2^-100, the scale of a page of zeros
    q = queries(20, 1, 1, 64, BF16)
    out, lse = case.run(q, case.plan(1), scale=2.0 ** -60, return_lse=True)
    case.check(q, out, lse, 2.0 ** -60)


# ------------------------------------------------------------------------- prompts ----

@pytest.mark.parametrize("dim,dtype,wide", [(64, BF16, False), (64, FP16, False), (128, BF16, False), (128, FP16, False),
                                            (128, BF16, True), (128, FP16, True), (256, BF16, False), (256, FP16, False)])
@torch.no_grad()
def test_causal_attention(device, dim, dtype, wide):
    """Blocks of 128 rows, and of 256."""
    lengths, heads, kv_heads = [130, 1, 0, 400], 6, 2
    g = torch.Generator().manual_seed(dim)
    qkv = torch.randn(sum(lengths), heads + 2 * kv_heads, dim, generator=g).to(dtype)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    plan = vc.prepare_causal_plan(lengths, heads, kv_heads, device=device)
    if wide:
        blocks = vc._blocks(tuple(lengths), heads // kv_heads, 256).to(device)
        plan = vc.CausalPlan(tuple(lengths), heads, kv_heads, sum(lengths), blocks, blocks)
    rows = qkv.cuda()
    for scale in FAR:
        scale *= 2.0 ** 6 / dim
        out, lse = vc.causal_attention(*rows.split([heads, kv_heads, kv_heads], 1), plan, scale, return_lse=True)
        sure, at = 0, 0
        for n in lengths:
            here = slice(at, at + n)
            at += n
            if n:
                sure += check_decided(q[here], k[here], v[here], 0, scale, out[here], lse[here])
        assert scale < 2 ** 10 or sure > 0.7 * lse.numel(), (scale, sure)


# ------------------------------------------------------------------------- windows ----

@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16), (256, BF16), (256, FP16)])
@torch.no_grad()
def test_window_attention(device, dim, dtype):
    """One frame and text in front of it: every row sees all."""
    layout = vw.SequenceLayout(203, 3, 1, 200)
    plan = vw.prepare_paper_window_plan(layout, vw.window_bounds(1, 0), device=device)
    g = torch.Generator().manual_seed(dim)
    q, k, v = torch.randn(3, 203, 4, dim, generator=g).to(dtype)
    for scale in FAR:
        scale *= 2.0 ** 6 / dim
        out, lse = vw.paper_window_attention(q.cuda(), k.cuda(), v.cuda(), plan, scale, enabled=True, return_lse=True)
        sure = check_decided(q, k, v, 203, scale, out, lse)
        assert scale < 2 ** 10 or sure > 0.7 * lse.numel(), (scale, sure)
