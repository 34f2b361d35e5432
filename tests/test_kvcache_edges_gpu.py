"""GPU: the 8-bit cache at the edges of its types, against the formula in 64 bits."""
import math

import pytest
import torch

from oracle import causal as oc
from oracle import kvcache as ok
from vdn_amd import kvcache as kv

from test_kvcache_gpu import check, filled, tables

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def in_order(n, page):
    """The table of one sequence of n tokens whose pages lie in order."""
    return torch.arange(-(-n // page), dtype=torch.int32)[None]


@pytest.mark.parametrize("n", [1, 300, 3000])          # one token, a whole unit, a split one
@pytest.mark.parametrize("dim", [64, 128, 256])
@torch.no_grad()
def test_fp16_outputs_next_to_the_largest_value(device, n, dim):
    """65504 and 63488 are stored as 65536: an output of theirs is 65504. (The rounded weights sum
    to within 2^-11 of 1, and from 65536 (1 - 2^-11) on fp16 gives 65504.)"""
    cache = kv.empty_cache(-(-n // 16), 2, dim, 16, device=device)
    table = in_order(n, 16).cuda()
    v = torch.full((n, 2, dim), 65504.0)
    v[..., 1::4], v[..., 2::4], v[..., 3::4] = -65504.0, 63488.0, -1.0
    k = torch.randn(n, 2, dim, generator=torch.Generator().manual_seed(n))
    kv.write_cache(cache, k.to(FP16).cuda(), v.to(FP16).cuda(), table, ints(0), ints(0, n))
    q = torch.randn(1, 6, dim, generator=torch.Generator().manual_seed(1)).to(FP16).cuda()
    out, lse = kv.cache_attention(q, cache, table, ints(n), return_lse=True)
    assert (out[..., 0::4] == 65504).all() and (out[..., 1::4] == -65504).all()
    assert (out[..., 2::4] == 65504).all() and torch.isfinite(lse).all()
    assert torch.isfinite(out).all()
    cache.check()


def faulty(cache, key, table, starts, offsets):
    """Whether a write of these rows, and a read, raise the fault word; their results may be anything."""
    said = []
    for call in (lambda: kv.write_cache(cache, key, key, table, starts, offsets),
                 lambda: kv.read_cache(cache, table, starts, offsets, key.shape[0])):
        call()
        said.append(bool(cache.faults.item()))
        cache.faults.zero_()
    assert said[0] == said[1]
    return said[0]


@pytest.mark.parametrize("offsets", [(0, 40, 8, 60), (0, 60, 0, 60), (0, 17, 16, 60), (0, 59, 60, 59),
                                     (0, 30, 61, 61), (0, -1, 20, 60), (1, 20, 40, 60)])
@torch.no_grad()
def test_offsets_that_fall_or_leave_the_rows(device, offsets):
    """The sequence between 40 and 8 owns no page step, so the search for a page passes it over. No
    page of these sequences changes."""
    cache = kv.empty_cache(13, 1, 64, 16, device=device)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.fill_(0x38)
    table = torch.arange(12, dtype=torch.int32, device=device).view(3, 4)
    x = torch.randn(60, 1, 64, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    assert not faulty(cache, x, table, ints(0, 0, 0), ints(0, 20, 20, 60))
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.fill_(0x38)
    assert faulty(cache, x, table, ints(0, 0, 0), ints(*offsets))
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        assert (t == 0x38).all()


@pytest.mark.parametrize("batch", [64, 65, 200, 5000])
@pytest.mark.parametrize("page", [16, 256])
@torch.no_grad()
def test_one_fall_among_many_offsets(device, batch, page):
    """Wherever the pair lies that falls, and however far, the word is raised."""
    rows, places = 3 * batch, {0, 1, 62, 63, 64, 127, 128, batch // 2, batch - 2, batch - 1}
    cache = kv.empty_cache(batch, 1, 64, page, device=device)
    table = torch.arange(batch, dtype=torch.int32, device=device)[:, None]
    x = torch.zeros(rows, 1, 64, dtype=BF16, device=device)
    starts = torch.zeros(batch, dtype=torch.int32, device=device)
    good = 3 * torch.arange(batch + 1, dtype=torch.int32)
    assert not faulty(cache, x, table, starts, good.cuda())
    for i in sorted(p for p in places if p < batch):
        for value in {int(good[i + 1]) + 4, 0, rows, rows + 1, -1}:
            bad = good.clone()
            bad[i] = value
            ok_pairs = bool((bad.diff() >= 0).all()) and bad[0] == 0 and int(bad.max()) <= rows
            assert faulty(cache, x, table, starts, bad.cuda()) == (not ok_pairs), (i, value)


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@pytest.mark.parametrize("n", [3, 100, 500, 3000])     # fewer than the queries, whole units, a split one
@torch.no_grad()
def test_rows_whose_scores_are_all_minus_infinity(device, dim, dtype, n):
    """A query whose every score is -inf has no softmax: NaN, its LSE -inf. A query that sees no key
    is zero; the others are as without it."""
    tokens = 5
    cache = kv.empty_cache(-(-n // 16), 1, dim, 16, device=device)
    table = in_order(n, 16).cuda()
    if n > 500:
        table = torch.cat((table, torch.zeros_like(table)), 1)
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(n, 1, dim, generator=g) for _ in range(2))
    k[..., 0] = 1.0 + k[..., 0].abs()
    kv.write_cache(cache, k.to(dtype).cuda(), v.to(dtype).cuda(), table, ints(0), ints(0, n))
    q = torch.randn(1, tokens, 3, dim, generator=g).to(dtype).cuda()
    want, wlse = kv.cache_attention(q, cache, table, ints(n), return_lse=True)
    shut = q.clone()
    shut[0, 0, 1, 0] = shut[0, tokens - 1, 2, 0] = -math.inf
    got, lse = kv.cache_attention(shut, cache, table, ints(n), return_lse=True)
    first = (0, 0, 1)
    if n < tokens:                                     # the first query sees none
        assert got[first].count_nonzero() == 0 and not got[first].isnan().any()
    else:
        assert got[first].isnan().all()
    assert torch.isneginf(lse[first]) and got[0, -1, 2].isnan().all() and torch.isneginf(lse[0, -1, 2])
    got[first], lse[first] = want[first], wlse[first]
    got[0, -1, 2], lse[0, -1, 2] = want[0, -1, 2], wlse[0, -1, 2]
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    cache.check()


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@pytest.mark.parametrize("at", [0, 70, 250, 600, 2900])
@pytest.mark.parametrize("n", [300, 3000])             # a whole unit, a split one
@torch.no_grad()
def test_a_nan_value_outweighed(device, dim, dtype, n, at):
    """The NaN code of a seen token reaches its channel wherever the heavy token lies, also where the
    token's weight underflows in fp32: in the same wave, another one of the workgroup, another slot."""
    if at >= n:
        return
    cache = kv.empty_cache(-(-n // 16), 1, dim, 16, device=device)
    table = in_order(n, 16).cuda()
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(n, 1, dim, generator=g) for _ in range(2))
    k[..., 0] = 0.0
    v[at, 0, 5] = math.nan
    q = torch.randn(1, 2, dim, generator=g)
    q[..., 0] = 16.0
    others = [c for c in range(dim) if c != 5]
    for heavy in (10, 90, 130, 260, 700, 1500, 2990):
        if heavy >= n or heavy // 16 == at // 16:      # (a page with one loud channel keeps its own scale)
            continue
        loud = k.clone()
        loud[heavy, 0, 0] = 400.0
        kv.write_cache(cache, loud.to(dtype).cuda(), v.to(dtype).cuda(), table, ints(0), ints(0, n))
        out, lse = kv.cache_attention(q.to(dtype).cuda(), cache, table, ints(n), 1.0, return_lse=True)
        assert out[..., 5].isnan().all(), heavy
        assert torch.isfinite(out[..., others]).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heavy", [0, 20000])
@pytest.mark.parametrize("n,heads", [(500, 1), (32768, 1), (32768, 24)])
@torch.no_grad()
def test_fp16_weights_that_are_small_but_many(device, dim, heavy, n, heads):
    """Tokens of weight 2^-25.3 relative to a heavy one, whose value is 0: their sum is the output. A
    weight is rounded to within 2^-39 of the largest or to half a step of fp16, the output to half a
    step or 2^-25 (the bound's own terms, 2^-25 for each weight and 2^-14, are larger than that)."""
    heavy = min(heavy, n - 1)
    cache = kv.empty_cache(-(-n // 64), 1, dim, 64, device=device)
    oracle = ok.Cache(-(-n // 64), 1, 64, dim)
    table = in_order(n, 64)
    k = torch.zeros(n, 1, dim)
    k[heavy, 0, 0] = 16.0
    v = torch.rand(n, 1, dim, generator=torch.Generator().manual_seed(3)) + 0.5
    v[heavy] = 0.0
    k, v = k.to(FP16), v.to(FP16)
    kv.write_cache(cache, k.cuda(), v.cuda(), table.cuda(), ints(0), ints(0, n))
    oracle.write(k, v, table, [0], [n])
    kk, vv = (oracle.tokens(side, table[0], 0, n) for side in range(2))
    assert kk[heavy, 0, 0] == 16
    q = torch.zeros(1, heads, dim)
    q[..., 0] = 1.0957
    q = q.to(FP16)
    got, lse = kv.cache_attention(q.cuda(), cache, table.cuda(), ints(n), 1.0, return_lse=True)
    out, el, mass, size = oc.attention(q, kk, vv, n - 1, 1.0)
    tol, ltol = oc.bounds(out, mass, size, vv, FP16, dim, n)
    tol += n * (2.0 ** -39 - 2.0 ** -25) * float(vv.abs().max()) + 2.0 ** -25 - torch.finfo(FP16).tiny
    err = (got.cpu().double() - out).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max())}"
    assert bool(((lse.cpu().double() - el).abs() <= ltol).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,tokens", [(16, 1), (32, 3)])
@pytest.mark.parametrize("drop", [-112.0, -20.0, 0.0])   # score of the loud page's tokens
@pytest.mark.parametrize("apart", [4, 12, 15, 16, 20, 26, 33])
@torch.no_grad()
def test_fp16_pages_of_different_scales_in_one_tile(device, dim, page, tokens, drop, apart):
    """A page of values up to fp16's largest beside pages 2^-apart of it: what those are worth in fp16
    reaches the output. A weight w is rounded to half a step of fp16, or to within 2^-39 of the
    largest (at most w); where it also takes a page's scale, to within 2^-25 of a value of at most 448
    2^-15 units of 2^8, less the weights' 2^14: 2^-37. The output to half a step, 2^-25 if subnormal."""
    n, loud = 150, 80                              # the loud page lies inside the second tile
    pages = -(-n // page)
    g = torch.Generator().manual_seed(apart)
    cache = kv.empty_cache(pages, 1, dim, page, device=device)
    kc = (torch.randn(pages, 1, page, dim, generator=g) * 100).clamp(-400, 400)
    kc[..., 0] = 0.0
    kc[loud // page, :, :, 0] = drop
    vc = (torch.randn(pages, 1, dim, page, generator=g) * 100).clamp(-224, 224)
    kc, vc = kc.to(torch.float8_e4m3fn), vc.to(torch.float8_e4m3fn)
    ke = torch.zeros(pages, 1, dtype=torch.int64)
    ve = torch.full((pages, 1), 8 - apart, dtype=torch.int64)
    ve[loud // page] = 8
    for to, x in ((cache.k_codes, kc), (cache.v_codes, vc)):
        to.copy_(x.view(torch.uint8))
    for to, e in ((cache.k_scales, ke), (cache.v_scales, ve)):
        to.copy_((e + 127).to(torch.uint8))
    k = (kc.double() * torch.exp2(ke.double())[..., None, None]).transpose(0, 1).flatten(1, 2)[0, :n, None]
    v = (vc.double() * torch.exp2(ve.double())[..., None, None]).permute(1, 0, 3, 2).flatten(1, 2)[0, :n, None]
    q = torch.randn(1, tokens, 2, dim, generator=g) * 0.004
    q[..., 0] = 1.0
    q = q.to(FP16)
    got = kv.cache_attention(q.cuda(), cache, in_order(n, page).cuda(), ints(n), 1.0)
    out, lse, mass, size = oc.attention(q[0], k, v, n - tokens, 1.0)
    tol, _ = oc.bounds(out, mass, size, v, FP16, dim, n)
    tol -= torch.finfo(FP16).tiny + n * 2.0 ** -25 * float(v.abs().max())
    s = torch.einsum("ihd,jd->ihj", q[0].double(), k[:, 0])
    s = s.masked_fill(torch.arange(n) > torch.arange(tokens)[:, None, None] + n - tokens, -math.inf)
    w = torch.exp(s - lse[..., None])
    tol += w.clamp_max(2.0 ** -39) @ v[:, 0].abs() + n * 2.0 ** -37 + 2.0 ** -25
    err = (got[0].cpu().double() - out).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max())}"
    assert float(out.abs().max()) > 8 * 2.0 ** (8 - apart)       # the output is worth looking at
    cache.check()


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@pytest.mark.parametrize("n", [400, 6000])             # whole units, split ones
@torch.no_grad()
def test_the_output_over_its_queries(device, dim, dtype, n):
    """out = query gives what a fresh output does; another overlap is refused."""
    cache = kv.empty_cache(-(-n // 16), 2, dim, 16, device=device)
    table = in_order(n, 16).cuda().repeat(3, 1)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, 2, dim, generator=g).to(dtype).cuda()
    kv.write_cache(cache, x, -x, table[:1], ints(0), ints(0, n))
    q = torch.randn(3, 5, 20, dim, generator=g).to(dtype).cuda()
    lengths = ints(n, n - 7, 3)
    want = kv.cache_attention(q, cache, table, lengths)
    part, pwant = q.clone()[:, :, 4:10], kv.cache_attention(q[:, :, 4:10], cache, table, lengths)
    with pytest.raises(ValueError, match="overlap"):
        kv.cache_attention(q[:, :4], cache, table, lengths, out=q[:, 1:])
    with pytest.raises(ValueError, match="itself"):
        kv.cache_attention(q, cache, table, lengths, out=q.as_strided(q.shape, (4 * 20 * dim, 20 * dim, dim, 1)))
    assert torch.equal(kv.cache_attention(q, cache, table, lengths), want)
    for queries, result in ((q, want), (part, pwant)):
        got = kv.cache_attention(queries, cache, table, lengths, out=queries)
        assert got is queries and torch.equal(queries, result)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16), (256, BF16)])
@torch.no_grad()
def test_codes_behind_the_end_stay(device, page, dim, dtype):
    """What a write leaves of a page that it fills in part, for ends at, before and behind multiples of 16
    and 4: every code behind the end, but that a run of 16 V codes which holds earlier tokens is
    rounded again with them when the scale grows."""
    g = torch.Generator().manual_seed(page + dim)
    for held, new in ((0, 1), (0, 16), (0, page - 16), (3, 1), (5, 4), (16, 16), (page // 2, 2), (7, 9),
                      (page // 2 + 1, page // 4), (page - 3, 2)):
        n = held + new
        if not 0 < new or n > page:
            continue
        for growth in (0.01, 100.0):
            cache = kv.empty_cache(3, 2, dim, page, device=device)
            for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
                t.copy_(torch.randint(0, 120, t.shape, generator=g))
            table = ints(1)[None]
            x = torch.randn(max(held, 1), 4, dim, generator=g).to(dtype).cuda()
            if held:
                kv.write_cache(cache, x[:, :2], x[:, 2:], table, ints(0), ints(0, held))
            k0, v0, ks0, vs0 = (t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales))
            y = (torch.randn(new, 4, dim, generator=g) * growth).to(dtype).cuda()
            kv.write_cache(cache, y[:, :2], y[:, 2:], table, ints(held), ints(0, new))
            assert torch.equal(cache.k_codes[1, :, n:], k0[1, :, n:])
            # the runs that begin in front of the first new token are rounded again where V's scale grew
            again = -(-held // 16) * 16 if held else 0
            assert torch.equal(cache.v_codes[1, :, :, max(n, again):], v0[1, :, :, max(n, again):]), (held, new)
            for u in range(2):
                grew = held and int(cache.v_scales[1, u]) != int(vs0[1, u])
                assert not held or bool(grew) == (growth > 1)
                if not grew:
                    assert torch.equal(cache.v_codes[1, u, :, n:], v0[1, u, :, n:]), (held, new)
                    assert torch.equal(cache.v_codes[1, u, :, :held], v0[1, u, :, :held])
            for p in (0, 2):
                assert torch.equal(cache.k_codes[p], k0[p]) and torch.equal(cache.v_codes[p], v0[p])
                assert torch.equal(cache.k_scales[p], ks0[p]) and torch.equal(cache.v_scales[p], vs0[p])
    cache.check()


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(33, 4, 2), (130, 5, 1), (256, 4, 4), (700, 2, 1)])
@torch.no_grad()
def test_many_queries(device, dim, dtype, tokens, heads, kv_heads):
    """A piece of a prompt behind cached tokens: more queries than a row block, lengths around them (some
    queries then see nothing), whole and split units."""
    lengths = [tokens, tokens + 1, 700 + tokens, 0, tokens // 2, 3000]
    table, pages = tables([-(-n // 64) for n in lengths], seed=dim)
    cache, kval, vval = filled(pages, kv_heads, dim, 64, seed=heads)
    q = torch.randn(len(lengths), tokens, heads, dim, generator=torch.Generator().manual_seed(tokens))
    q = q.to(dtype).cuda()
    out, lse = kv.cache_attention(q, cache, table.cuda(), ints(*lengths), return_lse=True)
    check(q, cache, kval, vval, table, lengths, out, lse)
    assert out[3].count_nonzero() == 0
    short = kv.cache_attention(q[:1], cache, table[:1, :-(-tokens // 64)].cuda(), ints(tokens))
    check(q[:1], cache, kval, vval, table[:1], lengths[:1], short)
    cache.check()
