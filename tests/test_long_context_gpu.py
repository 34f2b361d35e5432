"""GPU: rotation, cache, shared prefix and selected pages together, as a decoder with grouped heads uses
them: a prompt is rotated, attended and cached once, sequences continue behind it in steps. Every
step's output is checked against float64 over what the cache holds."""
import math

import pytest
import torch

from oracle import causal as oc
from oracle import rotary as orot
from oracle import sparse as osp
from vdn_amd import kvcache as kv
from vdn_amd import prefix as vp
from vdn_amd import rotary as vr
from vdn_amd import sparse as sp
from vdn_amd.causal import causal_attention, prepare_causal_plan

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS = 8, 2


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cached(cache):
    k = cache.k_codes.cpu().view(torch.float8_e4m3fn).double()
    v = cache.v_codes.cpu().view(torch.float8_e4m3fn).double()
    return k * torch.exp2(cache.k_scales.cpu().double() - 127)[..., None, None], \
        (v * torch.exp2(cache.v_scales.cpu().double() - 127)[..., None, None]).transpose(2, 3)


def near(out, q, k, v, scale):
    """out, q [H, D] over k, v [n, kv_heads, D], all of them seen."""
    n = k.shape[0]
    o, _, mass, size = oc.attention(q[None].cpu(), k, v, n, scale)
    bound, _ = oc.bounds(o, mass, size, v, q.dtype, q.shape[-1], n)
    assert ((out.cpu().double() - o[0]).abs() <= bound[0]).all()


@pytest.mark.parametrize("dim,dtype,page,layout", [(64, torch.float16, 16, "interleaved"),
                                                   (128, torch.bfloat16, 64, "half")])
@torch.no_grad()
def test_prompt_then_steps_behind_it(device, dim, dtype, page, layout):
    g = torch.Generator().manual_seed(page)
    prompt, batch, steps = 3 * page + 5, 3, 2 * page + 3
    width = -(-steps // page)
    cache = kv.empty_cache(4 + batch * width + 3, KV_HEADS, dim, page, device="cuda")
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.fill_(0x7f)                       # NaN codes of earlier owners
    order = torch.randperm(cache.pages, generator=g).int()
    shared, table = order[:4].view(1, 4).cuda(), order[4:4 + batch * width].view(batch, width).cuda()
    rotary = vr.prepare_rotary_plan(dim, rotary_dim=dim // 2, layout=layout, scaling="parts", factor=4.0,
                                    original=64, device="cuda")
    frequencies, amplitude = vr.rotary_frequencies(dim // 2, scaling="parts", factor=4.0, original=64)
    weights = [(1 + 0.1 * torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2)]
    qkv = torch.randn(prompt, HEADS + 2 * KV_HEADS, dim, generator=g).to(dtype).cuda()
    q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]

    # ---- the prompt: in place, as slices of the projection ----
    raw = k.cpu().clone()
    positions = torch.arange(prompt, dtype=torch.int32).cuda()
    vr.rotate_qk(q, k, positions, rotary, *weights, out=(q, k))
    value, size = orot.rotate(raw, positions.cpu(), frequencies, layout, amplitude, weights[1].cpu())
    assert ((k.cpu().double() - value).abs() <= orot.tolerance(value, size, dtype)).all()
    out = causal_attention(q, k, v, prepare_causal_plan([prompt], HEADS, KV_HEADS, device="cuda"))
    near(out[-1], q[-1], k.cpu().double(), v.cpu().double(), dim ** -0.5)
    kv.write_cache(cache, k, v, shared, ints(0), ints(0, prompt))

    # ---- steps behind it, eagerly and then captured ----
    plan = vp.prepare_prefix_plan([prompt], [batch], HEADS, KV_HEADS, dim, device="cuda")
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    step_qkv = torch.empty(batch, HEADS + 2 * KV_HEADS, dim, dtype=dtype, device="cuda")
    sq, sk, sv = (step_qkv[:, :HEADS], step_qkv[:, HEADS:HEADS + KV_HEADS], step_qkv[:, HEADS + KV_HEADS:])

    def step():
        a, b = vr.rotate_qk(sq, sk, lengths + prompt, rotary, *weights)
        kv.write_cache(cache, b, sv, table, lengths)
        lengths.add_(1)
        return a, vp.prefix_attention(a, cache, shared, plan, table, lengths)

    graph = None
    for n in range(1, steps + 1):
        step_qkv.copy_(torch.randn(step_qkv.shape, generator=g))
        if n == 3:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                a, got = step()
        if graph is None:
            a, got = step()
        else:
            graph.replay()
        if n not in (1, 2, 3, page, page + 1, steps):
            continue
        torch.cuda.synchronize()
        assert lengths.tolist() == [n] * batch
        keys, values = cached(cache)
        for b in range(batch):
            rows = [torch.cat([side[int(p)].transpose(0, 1) for p in t])[:m]
                    for side in (keys, values) for t, m in ((shared[0], prompt), (table[b], n))]
            near(got[b], a[b], torch.cat(rows[:2])[:, :], torch.cat(rows[2:]), dim ** -0.5)
    cache.check()

    # ---- the same sequences over whole tables: the prefix's full pages are shared, its last one copied ----
    full, rest = prompt // page, prompt % page
    own_last = order[4 + batch * width:4 + batch * width + batch]
    assert len(own_last) == batch
    src = int(shared[0, full])
    for p in own_last.tolist():
        for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
            t[p] = t[src]
    whole = torch.cat((shared[:, :full].expand(batch, full), own_last.view(batch, 1).cuda()), 1).contiguous()
    held = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
    means = sp.empty_means(cache)
    sp.write_means(cache, means, whole, torch.zeros_like(held), held)
    pages, tokens = sp.select_pages(a, cache, means, whole, held, 3)
    picked = sp.selected_attention(a, cache, pages, tokens)
    keys, values = cached(cache)
    for b in range(batch):
        (want, seen), = osp.select(a[b:b + 1].cpu(), means.cpu(), whole[b].tolist(), prompt, page, 3, 1, 1)
        assert pages[b].tolist() == want and int(tokens[b]) == seen == 2 * page + rest
        for u in range(KV_HEADS):
            hs = slice(u * HEADS // KV_HEADS, (u + 1) * HEADS // KV_HEADS)
            rows = [torch.cat([side[p, u] for p in want[u]])[:seen, None] for side in (keys, values)]
            near(picked[b, hs], a[b, hs], *rows, dim ** -0.5)
    cache.check()
    assert math.isfinite(float(picked.float().sum()))
