"""GPU: the 8-bit key/value cache. What a write stores is bit for bit the oracle's (oracle/kvcache.py);
attention over the codes is within the bounds derived from its roundings (oracle/causal.py)."""
import math

import pytest
import torch

from oracle import causal as oc
from oracle import kvcache as ok
from vdn_amd import causal as vc
from vdn_amd import kvcache as kv

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tables(counts, seed=0, spare=2):
    """A table with the pages of every sequence in random order (-1 behind them), and the pool."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(counts) + spare, generator=g).tolist()
    table = torch.full((len(counts), max(max(counts), 1)), -1, dtype=torch.int32)
    for i, n in enumerate(counts):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table, sum(counts) + spare


def filled(pages, kv_heads, dim, page, seed=0):
    """A cache of random finite codes and scales, and the float64 values of its K and V."""
    g = torch.Generator().manual_seed(seed)
    cache = kv.empty_cache(pages, kv_heads, dim, page, device="cuda")
    values = []
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        x = (torch.randn(codes.shape, generator=g) * 100).clamp(-448, 448)
        c = x.to(torch.float8_e4m3fn)
        e = torch.randint(-9, -4, scales.shape, generator=g)
        codes.copy_(c.view(torch.uint8))
        scales.copy_((e + 127).to(torch.uint8))
        values.append(c.double() * torch.exp2(e.double())[..., None, None])
    return cache, values[0], values[1].transpose(2, 3)


def rows_of(values, pages, n, page):
    """[n, heads, dim] of a sequence."""
    if n == 0:
        return values[0].transpose(0, 1)[:0]
    return torch.cat([values[int(p)].transpose(0, 1) for p in pages[:-(-n // page)]])[:n]


# --------------------------------------------------------------------- write, read ----

@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16), (128, BF16), (256, BF16), (256, FP16)])
@torch.no_grad()
def test_write_and_read_bit_for_bit(device, page, dim, dtype):
    """Prompts, then pieces and single tokens whose magnitude grows and falls, in pages out of order:
    the values read back are the oracle's; what no row touched keeps its codes."""
    heads, steps = 3, ([page + 3, 0, 2 * page, 1], [5, 1, 0, page - 1], [1, 1, 1, 1], [2, page, 3, 0],
                       [1, 0, 1, 1])
    totals = [sum(s[i] for s in steps) for i in range(4)]
    table, pages = tables([-(-t // page) for t in totals], seed=page)
    cache = kv.empty_cache(pages, heads, dim, page, device=device)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.copy_(torch.randint(0, 127, t.shape, generator=torch.Generator().manual_seed(1)))
    spare = [p for p in range(pages) if p not in table]
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)]
    oracle = ok.Cache(pages, heads, page, dim)
    g = torch.Generator().manual_seed(7)
    held = [0] * 4
    for amp, sizes in zip((1.0, 0.3, 40.0, 700.0, 0.01), steps):
        n = sum(sizes)
        kvs = (torch.randn(n + 2, 2 * heads, dim, generator=g) * amp).to(dtype)   # two rows too many
        if amp == 1.0:
            kvs[0, 0, :5] = torch.tensor([math.nan, math.inf, -math.inf, 1e-7, 0.0])
            kvs[page + 3:page + 3 + page, heads + 1] = 0                      # an all-zero V page
        key, value = kvs[:, :heads], kvs[:, heads:]
        offsets = [sum(sizes[:i]) for i in range(5)]
        on_gpu = kvs.cuda()
        kv.write_cache(cache, on_gpu[:, :heads], on_gpu[:, heads:], table.cuda(), ints(*held),
                       ints(*offsets))
        oracle.write(key[:n], value[:n], table, held, sizes)
        held = [h + s for h, s in zip(held, sizes)]
        offs = [sum(held[:i]) for i in range(5)]
        got = kv.read_cache(cache, table.cuda(), ints(0, 0, 0, 0), ints(*offs), offs[-1] + 1, dtype=dtype)
        for side in range(2):
            want = torch.cat([oracle.tokens(side, table[i], 0, held[i]) for i in range(4)])
            top = torch.finfo(dtype).max
            want = want.clamp(-top, top).to(dtype) if dtype == FP16 else want.to(dtype)
            assert torch.equal(got[side][:-1].cpu().nan_to_num(nan=-77), want.nan_to_num(nan=-77))
            assert got[side][-1].count_nonzero() == 0
    for t, old in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales), before):
        assert torch.equal(t[spare], old[spare])
    # positions behind a sequence's end
    for i, n in enumerate(totals):
        if n % page:
            p = int(table[i, n // page])
            assert torch.equal(cache.v_codes[p, :, :, n % page:], before[1][p, :, :, n % page:]) or \
                n % 16       # (a run of 16 that holds earlier tokens may be rounded again with them)
            assert torch.equal(cache.k_codes[p, :, n % page:], before[0][p, :, n % page:])
    cache.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@torch.no_grad()
def test_extreme_magnitudes(device, dtype):
    """The largest and smallest numbers of the type, a page each: finite values stay finite."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    cache = kv.empty_cache(3, 1, 64, 16, device=device)
    oracle = ok.Cache(3, 1, 16, 64)
    x = torch.zeros(48, 1, 64)
    x[:16] = torch.linspace(-1, 1, 64) * top
    x[16:32] = torch.linspace(-3, 3, 64) * tiny
    x = x.to(dtype)
    x[0, 0, 0], x[0, 0, 63] = -top, top
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    kv.write_cache(cache, x.cuda(), x.cuda(), table.cuda(), ints(0), ints(0, 48))
    oracle.write(x, x, table, [0], [48])
    want = oracle.tokens(0, table[0], 0, 48)
    got = kv.read_cache(cache, table.cuda(), ints(0), ints(0, 48), 48, dtype=BF16)
    for side in range(2):
        assert torch.isfinite(got[side]).all() and torch.equal(got[side].cpu().double(), want)
    got = kv.read_cache(cache, table.cuda(), ints(0), ints(0, 48), 48, dtype=FP16)
    for side in range(2):
        assert torch.isfinite(got[side]).all()
        assert torch.equal(got[side].cpu(), want.clamp(-65504, 65504).to(FP16))


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 300, 4200])
@torch.no_grad()
def test_many_sequences(device, batch):
    """The search for a sequence over one, two and three rounds of 64; sequences without rows."""
    sizes = [(7 * i) % 4 for i in range(batch)]
    table, pages = tables([1] * batch, seed=batch)
    cache = kv.empty_cache(pages, 1, 64, 16, device=device)
    offsets = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()
    starts = torch.tensor([i % 13 for i in range(batch)], dtype=torch.int32, device=device)
    zero = torch.zeros_like(starts)
    g = torch.Generator().manual_seed(batch)
    first = torch.randn(13 * batch, 1, 64, generator=g).to(BF16).cuda()
    kv.write_cache(cache, first, first, table.cuda(), zero,
                   (torch.arange(batch + 1) * 13).to(torch.int32).cuda())
    x = torch.randn(sum(sizes), 1, 64, generator=g).to(BF16).cuda()
    kv.write_cache(cache, x, -x, table.cuda(), starts, offsets)
    k, v = kv.read_cache(cache, table.cuda(), starts, offsets, sum(sizes))
    if sum(sizes):
        assert torch.equal(k, -v)
        # a page's values are within 2^8 of its largest: E4M3 rounds by 2^-4, or 2^-10 of the scale
        limit = x.abs().double() / 16 + 2.0 ** -10 * max(first.abs().max(), x.abs().max()).double() / 224
        assert bool(((k.double() - x.double()).abs() <= limit).all())
    one = torch.randn(batch, 1, 64, generator=g).to(BF16).cuda()
    kv.write_cache(cache, one, one, table.cuda(), zero + 15)            # no offsets: one row each
    k, v = kv.read_cache(cache, table.cuda(), zero + 15, None, batch)
    assert torch.equal(k, v)
    assert bool(((k - one).abs().double() <= one.abs().double() / 16
                 + 2.0 ** -10 * max(first.abs().max(), one.abs().max()).double() / 224).all())
    cache.check()


@torch.no_grad()
def test_faults_are_reported_and_not_followed(device):
    page, heads, dim = 16, 2, 64
    table, pages = tables([2, 2, 2], spare=0)
    cache, kval, _ = filled(pages, heads, dim, page)
    x = torch.randn(9, heads, dim, dtype=BF16, device=device)
    q = torch.randn(3, heads, dim, dtype=BF16, device=device)
    good = kv.cache_attention(q, cache, table.cuda(), ints(20, 20, 20))
    cache.check()
    codes = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)]
    for bad_id in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        bad = table.clone()
        bad[1, 1] = bad_id
        kv.write_cache(cache, x[3:6], x[3:6], bad.cuda(), ints(16, 16, 16), ints(0, 0, 3, 3))
        with pytest.raises(RuntimeError, match="does not have"):
            cache.check()
        cache.check()
        k, _ = kv.read_cache(cache, bad.cuda(), ints(14, 14, 14), ints(0, 4, 8, 12), 12)
        assert k[6:8].isnan().all() and not k[:6].isnan().any() and not k[8:].isnan().any()
        with pytest.raises(RuntimeError):
            cache.check()
        out, lse = kv.cache_attention(q, cache, bad.cuda(), ints(20, 20, 20), return_lse=True)
        assert out[1].isnan().all() and lse[1].isnan().all()
        assert torch.equal(out[[0, 2]], good[[0, 2]])
        with pytest.raises(RuntimeError):
            cache.check()
        # the bad page lies behind the sequence's end: not looked at
        assert torch.equal(kv.cache_attention(q, cache, bad.cuda(), ints(20, 16, 20))[[0, 2]], good[[0, 2]])
        cache.check()
    for n in (33, -1, 2 ** 31 - 1, -2 ** 31):
        out = kv.cache_attention(q, cache, table.cuda(), ints(20, n, 20))
        assert out[1].isnan().all() and torch.equal(out[[0, 2]], good[[0, 2]])
        with pytest.raises(RuntimeError):
            cache.check()
    for starts, offsets in (((32, 0, 0), (0, 3, 3, 3)), ((-1, 0, 0), (0, 3, 3, 3)),
                            ((31, 0, 0), (0, 3, 3, 3)), ((2 ** 31 - 1, 0, 0), (0, 3, 3, 3))):
        kv.write_cache(cache, x, x, table.cuda(), ints(*starts), ints(*offsets))
        with pytest.raises(RuntimeError):
            cache.check()
    p = int(table[0, 1])   # starts = 31 wrote its one good token
    keep = torch.ones(pages, dtype=torch.bool)
    keep[p] = False
    for t, old in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales), codes):
        assert torch.equal(t[keep.cuda()], old[keep.cuda()])
    for offsets in ((0, 12, 12, 12), (-4, 2, 2, 2), (0, 5, 3, 3), (2, 3, 5, 9), (40, 50, 60, 70)):
        kv.read_cache(cache, table.cuda(), ints(0, 0, 0), ints(*offsets), 9)
        with pytest.raises(RuntimeError):
            cache.check()


# ----------------------------------------------------------------------- attention ----

def check(q, cache, kval, vval, table, lengths, out, lse=None, scale=None):
    """q [batch, Q, H, D]."""
    dim, dtype = q.shape[3], q.dtype
    scale = dim ** -0.5 if scale is None else scale
    for i, n in enumerate(lengths):
        k = rows_of(kval, table[i], n, cache.page)
        v = rows_of(vval, table[i], n, cache.page)
        o, l, mass, size = oc.attention(q[i].cpu(), k, v, n - q.shape[1], scale)
        tol, ltol = oc.bounds(o, mass, size, v, dtype, dim, max(n, 1))
        err = (out[i].cpu().double() - o).abs()
        assert bool((err <= tol).all()), f"sequence {i} of {n}: worst {(err / tol).max()}"
        if lse is not None:
            got = lse[i].cpu().double()
            none = torch.isneginf(l)
            assert torch.equal(torch.isneginf(got), none)
            assert bool(((got - l).abs() <= ltol)[~none].all())


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16), (256, BF16),
                                       (256, FP16)])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (4, 2), (24, 1), (6, 3)])
@pytest.mark.parametrize("tokens", [1, 3, 9])
@torch.no_grad()
def test_attention(device, dim, dtype, heads, kv_heads, tokens):
    """Lengths around the tile (64) and quad (256) borders, empty, shorter than the queries."""
    lengths = [1, 0, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 600]
    page = 16 if heads % 2 else 64
    table, pages = tables([-(-n // page) for n in lengths], seed=dim)
    cache, kval, vval = filled(pages, kv_heads, dim, page, seed=heads)
    g = torch.Generator().manual_seed(tokens)
    q = torch.randn(len(lengths), tokens, heads, dim, generator=g).to(dtype).cuda()
    out, lse = kv.cache_attention(q, cache, table.cuda(), ints(*lengths), return_lse=True)
    check(q, cache, kval, vval, table, lengths, out, lse)
    assert out[1].count_nonzero() == 0
    cache.check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@torch.no_grad()
def test_pages(device, page, dim, dtype):
    lengths = [1000, 1, page - 1, page, page + 1, 3 * page + 7]
    table, pages = tables([-(-n // page) for n in lengths], seed=page)
    cache, kval, vval = filled(pages, 2, dim, page, seed=dim)
    q = torch.randn(len(lengths), 10, dim, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    out, lse = kv.cache_attention(q, cache, table.cuda(), ints(*lengths), 0.3, return_lse=True)
    check(q[:, None], cache, kval, vval, table, lengths, out[:, None], lse[:, None], scale=0.3)


@pytest.mark.parametrize("batch,longest,heads,kv_heads,dim,dtype", [
    (1, 40000, 8, 1, 128, BF16), (3, 9000, 5, 5, 64, FP16), (300, 700, 2, 1, 64, BF16),
    (2, 5000, 36, 2, 128, BF16), (1, 20000, 2, 2, 256, BF16), (700, 30, 3, 3, 64, BF16),
    (300, 512, 8, 2, 128, BF16), (900, 500, 3, 1, 64, FP16), (1, 512, 2, 2, 256, BF16),
    (1, 1500, 1, 1, 64, BF16), (5, 1100, 4, 2, 128, FP16), (70, 3000, 8, 4, 128, BF16)])
@torch.no_grad()
def test_split_work(device, batch, longest, heads, kv_heads, dim, dtype):
    """Sequences that many workgroups share, workgroups that go through many sequences; the same
    call gives the same bits; every row of the output is written."""
    g = torch.Generator().manual_seed(batch)
    lengths = [longest] + torch.randint(0, longest, (batch - 1,), generator=g).tolist()
    table, pages = tables([-(-n // 64) for n in lengths], seed=1)
    cache, kval, vval = filled(pages, kv_heads, dim, 64, seed=3)
    q = torch.randn(batch, 1, heads, dim, generator=g).to(dtype).cuda()
    out = torch.full_like(q, math.nan)
    _, lse = kv.cache_attention(q, cache, table.cuda(), ints(*lengths), return_lse=True, out=out)
    pick = range(batch) if batch < 10 else [0, 1, 2, batch // 2, batch - 1]
    check(q[list(pick)], cache, kval, vval, table[list(pick)], [lengths[i] for i in pick],
          out[list(pick)], lse[list(pick)])
    assert torch.isfinite(out).all()
    again = kv.cache_attention(q, cache, table.cuda(), ints(*lengths))
    assert torch.equal(out, again)


@torch.no_grad()
def test_scores_that_grow_and_scales_that_differ(device):
    """K scales that rise 2^12 over the pages: the maximum moves from tile to tile; V scales over a wide
    range, all-zero V pages among them."""
    for dtype in (BF16, FP16):
        table, pages = tables([16], seed=4)
        cache, kval, vval = filled(pages, 2, 128, 64, seed=5)
        for j in range(16):
            p = int(table[0, j])
            for vals, scales, e in ((kval, cache.k_scales, j - 15), (vval, cache.v_scales, (j * 7) % 13 - 15)):
                old = scales[p].cpu().double() - 127
                vals[p] *= torch.exp2(e - old)[:, None, None]
                scales[p] = 127 + e
            if j in (3, 9):
                cache.v_codes[p] = 0
                cache.v_scales[p] = 27
                vval[p] = 0
        q = torch.randn(1, 2, 4, 128, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        out, lse = kv.cache_attention(q, cache, table.cuda(), ints(1000), return_lse=True)
        check(q, cache, kval, vval, table, [1000], out, lse)


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@torch.no_grad()
def test_nan_codes(device, dim, dtype):
    """NaN codes behind the end (a page's stale rest) reach nothing; those of a drafted token reach
    the queries that see it, and no earlier one."""
    lengths, page = [70, 131], 64
    table, pages = tables([2, 3])
    cache, kval, vval = filled(pages, 2, dim, page, seed=8)
    q = torch.randn(2, 4, 4, dim, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    clean = kv.cache_attention(q, cache, table.cuda(), ints(*lengths))
    for i, n in enumerate(lengths):
        p = int(table[i, n // page])
        cache.k_codes[p, :, n % page:] = 0x7f
        cache.v_codes[p, :, :, n % page:] = 0xff
    assert torch.equal(kv.cache_attention(q, cache, table.cuda(), ints(*lengths)), clean)
    p, at = int(table[0, 1]), (70 - 2) % page      # the third of the four newest tokens
    cache.v_codes[p, 0, 5, at] = 0x7f
    got = kv.cache_attention(q, cache, table.cuda(), ints(*lengths))
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :2], clean[0, :2])
    assert torch.equal(got[0, :, 2:], clean[0, :, 2:]) and got[0, 2:, :2, 5].isnan().all()
    others = [c for c in range(dim) if c != 5]
    assert torch.equal(got[0, 2:, :2][..., others], clean[0, 2:, :2][..., others])
    cache.v_codes[p, 0, 5, at] = 0x30
    cache.k_codes[p, 0, at, 3] = 0xff
    got = kv.cache_attention(q, cache, table.cuda(), ints(*lengths))
    assert torch.equal(got[0, :2], clean[0, :2]) and got[0, 2:, :2].isnan().all()


@torch.no_grad()
def test_strides_and_out(device):
    table, pages = tables([3, 2])
    cache, kval, vval = filled(pages, 2, 64, 64, seed=8)
    wide = torch.randn(2, 9, 3, 80, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    q = wide[:, 1:7, :, 8:72].transpose(1, 2)                    # [batch, Q = 3, H = 6, 64]
    backing = torch.full((4, 2, 6, 72), 7.0, dtype=BF16, device=device)
    out = backing[:3].transpose(0, 1)[..., 8:]
    ret = kv.cache_attention(q, cache, table.cuda(), ints(150, 100), out=out)
    assert ret.data_ptr() == out.data_ptr()
    check(q, cache, kval, vval, table, [150, 100], out)
    out.fill_(7.0)
    assert (backing == 7.0).all()
    padded = torch.full((2, 9), -5, dtype=torch.int32)
    padded[:, 2:2 + table.shape[1]] = table
    same = kv.cache_attention(q, cache, padded.cuda()[:, 2:2 + table.shape[1]], ints(150, 100))
    check(q, cache, kval, vval, table, [150, 100], same)


@torch.no_grad()
def test_far_pages(device):
    """A pool over 4 GiB: byte offsets of pages pass 32 bits."""
    pages = 2 ** 32 // (16 * 256 * 64) + 40
    cache = kv.empty_cache(pages, 16, 64, 256, device=device)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    x = torch.randn(600, 32, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    on_gpu = x.cuda()
    kv.write_cache(cache, on_gpu[:, :16], on_gpu[:, 16:], table.cuda(), ints(0), ints(0, 600))
    k, v = kv.read_cache(cache, table.cuda(), ints(0), ints(0, 600), 600)
    want = ok.Cache(3, 16, 256, 64)
    want.write(x[:, :16], x[:, 16:], torch.tensor([[0, 1, 2]]), [0], [600])
    kd, vd = (want.tokens(s, [0, 1, 2], 0, 600) for s in range(2))
    assert torch.equal(k.cpu().double(), kd) and torch.equal(v.cpu().double(), vd)
    q = torch.randn(1, 16, 64, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    out = kv.cache_attention(q, cache, table.cuda(), ints(600))
    o, _, mass, size = oc.attention(q.cpu(), kd, vd, 599, 64 ** -0.5)
    assert bool(((out.cpu().double() - o).abs() <= oc.bounds(o, mass, size, vd, BF16, 64, 600)[0]).all())


# -------------------------------------------------------------------- used together ----

@pytest.mark.parametrize("dtype", [BF16, FP16])
@torch.no_grad()
def test_prompt_then_steps(device, dtype):
    """Two prompts go through causal attention and into the cache, then steps of one token append and
    attend, captured once and replayed: each step's output is that of the codes it was to read."""
    heads, kv_heads, dim, page, lengths = 12, 2, 64, 32, [45, 130]
    g = torch.Generator().manual_seed(3)
    table, pages = tables([3, 5])
    cache = kv.empty_cache(pages, kv_heads, dim, page, device=device)
    oracle = ok.Cache(pages, kv_heads, page, dim)

    def draw(rows):
        x = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g).to(dtype).cuda()
        return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]

    q, k, v = draw(sum(lengths))
    plan = vc.prepare_causal_plan(lengths, heads, kv_heads, device=device)
    out = vc.causal_attention(q, k, v, plan)
    o, _, mass, size = oc.packed(q.cpu(), k.cpu(), v.cpu(), lengths, dim ** -0.5)
    assert bool(((out.cpu().double() - o).abs()
                 <= oc.bounds(o, mass, size, v.cpu(), dtype, dim, 130)[0]).all())
    kv.write_cache(cache, k, v, table.cuda(), ints(0, 0), ints(0, 45, 175))
    oracle.write(k.cpu(), v.cpu(), table, [0, 0], lengths)

    held, on_gpu = ints(*lengths), table.cuda()
    sq, sk, sv = (torch.empty_like(t) for t in draw(2))
    sout = torch.empty(2, heads, dim, dtype=dtype, device=device)

    def step():
        kv.write_cache(cache, sk, sv, on_gpu, held)
        held.add_(1)
        kv.cache_attention(sq, cache, on_gpu, held, out=sout)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        for t, x in zip((sq, sk, sv), draw(2)):
            t.copy_(x * (1 + i))
        graph.replay() if i % 3 != 2 else step()       # eager steps in between
        torch.cuda.synchronize()
        oracle.write(sk.cpu(), sv.cpu(), table, lengths, [1, 1])
        lengths = [n + 1 for n in lengths]
        for b in range(2):
            kk, vv = (oracle.tokens(s, table[b], 0, lengths[b]) for s in range(2))
            o, _, mass, size = oc.attention(sq[b:b + 1].cpu(), kk, vv, lengths[b] - 1, dim ** -0.5)
            tol = oc.bounds(o, mass, size, vv, dtype, dim, lengths[b])[0]
            assert bool(((sout[b:b + 1].cpu().double() - o).abs() <= tol).all()), (i, b)
    assert held.tolist() == lengths
    cache.check()


@torch.no_grad()
def test_two_streams_and_two_graphs(device):
    """Calls on two streams at once, and two captured graphs replayed at once: own workspaces."""
    table, pages = tables([160, 120])
    cache, _, _ = filled(pages, 2, 128, 64, seed=8)
    qs = [torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in (0, 1)]
    on_gpu, lengths = table.cuda(), ints(10000, 7000)
    want = [kv.cache_attention(q, cache, on_gpu, lengths) for q in qs]
    streams, outs, graphs = [torch.cuda.Stream() for _ in qs], [torch.empty_like(q) for q in qs], []
    for q, out in zip(qs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kv.cache_attention(q, cache, on_gpu, lengths, out=out)
    for replay in (False, True, True):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for q, out, st, graph in zip(qs, outs, streams, graphs):
                with torch.cuda.stream(st):
                    graph.replay() if replay else kv.cache_attention(q, cache, on_gpu, lengths, out=out)
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)


@torch.no_grad()
def test_refusals(device):
    cache = kv.empty_cache(4, 2, 64, 16, device=device)
    table, one = torch.zeros(2, 2, dtype=torch.int32, device=device), ints(1, 1)
    q = torch.zeros(2, 4, 64, dtype=BF16, device=device)
    x = torch.zeros(2, 2, 64, dtype=BF16, device=device)
    for bad in (dict(query=q.float()), dict(query=q[:, :3]), dict(query=q[..., :32]), dict(query=q.cpu()),
                dict(query=q[0]), dict(query=q[:, :, None].expand(2, 4, 3, 64)[:, :0]),
                dict(table=table.long()), dict(table=table[0]), dict(table=table[:, :0]),
                dict(table=table.t().contiguous().t()), dict(table=table.cpu()), dict(lengths=one.long()),
                dict(lengths=one[:1]), dict(lengths=one.cpu()), dict(scale=-1.0), dict(scale=math.inf),
                dict(out=q.float()), dict(out=q[:1]),
                dict(out=q[:, :1].expand(2, 4, 64))):
        args = dict(query=q, cache=cache, table=table, lengths=one) | bad
        with pytest.raises(ValueError):
            kv.cache_attention(**args)
    for bad in (dict(key=x.float()), dict(key=x[:, :1]), dict(key=x[..., :32]), dict(value=x.half()),
                dict(value=x.cpu()), dict(value=x[:1]), dict(starts=one.long()), dict(starts=one[:1]),
                dict(offsets=one), dict(table=table.long()), dict(key=x[:1], value=x[:1])):
        args = dict(cache=cache, key=x, value=x, table=table, starts=one) | bad
        with pytest.raises(ValueError):
            kv.write_cache(**args)
    for bad in (dict(rows=-1), dict(rows=2.0), dict(dtype=torch.float32), dict(offsets=one), dict(rows=3)):
        args = dict(cache=cache, table=table, starts=one, offsets=None, rows=2) | bad
        with pytest.raises(ValueError):
            kv.read_cache(**args)
    for call in (lambda: kv.cache_attention(q, None, table, one), lambda: kv.write_cache(None, x, x, table, one),
                 lambda: kv.read_cache(None, table, one, None, 2)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError, match="16-byte"):
        kv.write_cache(cache, torch.zeros(2, 2, 68, dtype=BF16, device=device)[..., 4:], x, table, one)
    with torch.enable_grad():
        for call in (lambda: kv.cache_attention(q, cache, table, one),
                     lambda: kv.write_cache(cache, x, x, table, one),
                     lambda: kv.read_cache(cache, table, one, None, 2)):
            with pytest.raises(RuntimeError, match="inference-only"):
                call()


@torch.no_grad()
def test_nothing_to_do(device):
    cache = kv.empty_cache(4, 2, 64, 16, device=device)
    none = torch.zeros(0, 2, dtype=torch.int32, device=device)
    x = torch.zeros(0, 2, 64, dtype=BF16, device=device)
    empty = torch.zeros(0, dtype=torch.int32, device=device)
    kv.write_cache(cache, x, x, none, empty)
    kv.write_cache(cache, x, x, none, empty, ints(0))
    k, v = kv.read_cache(cache, none, empty, ints(0), 5)
    assert k.shape == (5, 2, 64) and not k.any() and not v.any()
    out, lse = kv.cache_attention(torch.zeros(0, 4, 64, dtype=BF16, device=device), cache, none, empty,
                                  return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    cache.check()


@torch.no_grad()
def test_rows_behind_two_to_the_31_elements(device):
    """Written rows of a wide buffer, the last ones behind 2^31 elements."""
    rows, wide, page = 33070, 66000, 256
    base = torch.empty(rows, wide, dtype=BF16, device=device)
    near = torch.randn(2, rows, 1, 64, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    far = [base[:, 64 * i:64 * i + 64].unflatten(1, (1, 64)) for i in range(2)]
    for x, y in zip(far, near):
        x.copy_(y)
    pages = -(-rows // page)
    table = torch.arange(pages, dtype=torch.int32, device=device)[None]
    starts = torch.zeros(1, dtype=torch.int32, device=device)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=device)
    got = []
    for key, value in (far, near):
        cache = kv.empty_cache(pages, 1, 64, page, device=device)
        kv.write_cache(cache, key, value, table, starts, offsets)
        cache.check()
        got.append(kv.read_cache(cache, table, starts, offsets, rows))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert (got[0][0].float() - near[0].float()).abs().max() <= 2.0 ** -4 * near[0].abs().max()
