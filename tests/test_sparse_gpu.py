"""GPU: mean keys (bit for bit), the selection by them (equal) and attention over it (within the bounds of
oracle/causal.py) against float64."""
import math

import pytest
import torch

from oracle import causal as oc
from oracle import sparse as osp
from vdn_amd import kvcache as kv
from vdn_amd import sparse as sp

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
        c = (torch.randn(codes.shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        e = torch.randint(-9, -4, scales.shape, generator=g)
        codes.copy_(c.view(torch.uint8))
        scales.copy_((e + 127).to(torch.uint8))
        values.append(c.double() * torch.exp2(e.double())[..., None, None])
    return cache, values[0], values[1].transpose(2, 3)


# --------------------------------------------------------------------------- means ----

@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
@torch.no_grad()
def test_means_bit_for_bit(device, page, dim):
    lengths = [1, 5 * page, 3 * page + 7, page - 1, 0, 2 * page]
    starts = [0, 0, page + 3, page - 2, 0, 2 * page]        # the last two touch nothing
    table, pages = tables([-(-n // page) for n in lengths])
    cache, keys, _ = filled(pages, 3, dim, page)
    means = sp.empty_means(cache)
    means.fill_(-7.0)
    want = torch.full(means.shape, -7.0, dtype=torch.float64)
    for b, (lo, n) in enumerate(zip(starts, lengths)):
        for at in range(lo // page, -(-n // page) if lo < n else 0):
            p = int(table[b, at])
            want[p] = osp.mean(keys[p], min(page, n - at * page))
    sp.write_means(cache, means, table.cuda(), ints(*starts), ints(*lengths))
    assert torch.equal(means.cpu().double(), want)
    cache.check()


@pytest.mark.parametrize("batch", [1, 63, 65, 300])
@torch.no_grad()
def test_means_of_many_sequences(device, batch):
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 200, (batch,), generator=g).tolist()
    starts = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in lengths]
    table, pages = tables([-(-n // 16) for n in lengths])
    cache, keys, _ = filled(pages, 2, 64, 16)
    means = sp.empty_means(cache).zero_()
    want = torch.zeros(means.shape, dtype=torch.float64)
    for b, (lo, n) in enumerate(zip(starts, lengths)):
        for at in range(lo // 16, -(-n // 16) if lo < n else 0):
            want[int(table[b, at])] = osp.mean(keys[int(table[b, at])], min(16, n - at * 16))
    sp.write_means(cache, means, table.cuda(), ints(*starts), ints(*lengths))
    assert torch.equal(means.cpu().double(), want)


@torch.no_grad()
def test_means_of_extreme_codes(device):
    """The largest sums that a page can have, the smallest beside them, scales at both ends, and NaN."""
    cache = kv.empty_cache(4, 1, 64, 256, device="cuda")
    codes = torch.full((4, 1, 256, 64), 0x7e, dtype=torch.uint8)              # 448
    codes[0, 0, 200] = 0x01                                                   # 2^-9
    codes[1, 0, :, ::2] = 0xfe                                                # -448
    codes[2, 0, 0, :] = 0x81
    codes[2, 0, 1:] = 0
    codes[3, 0, 17, 5] = 0x7f
    codes[3, 0, 250, 6] = 0xff                                                # behind the length
    cache.k_codes.copy_(codes)
    cache.k_scales.copy_(torch.tensor([[127 + 90], [27], [127], [120]]))
    values = codes.view(torch.float8_e4m3fn).double() * \
        torch.exp2(cache.k_scales.cpu().double() - 127)[..., None, None]
    means = sp.empty_means(cache)
    lengths = [256, 256, 255, 250]
    sp.write_means(cache, means, ints(0, 1, 2, 3).view(4, 1), ints(0, 0, 0, 0), ints(*lengths))
    want = torch.stack([osp.mean(values[p], n) for p, n in enumerate(lengths)])
    assert want.isnan().nonzero().tolist() == [[3, 0, 5]]
    assert torch.equal(torch.nan_to_num(means.cpu().double(), 1.5), torch.nan_to_num(want, 1.5))


@torch.no_grad()
def test_means_faults(device):
    cache, keys, _ = filled(4, 1, 64, 16)
    means = sp.empty_means(cache).zero_()
    table = ints(0, 1, 2, 9, -1, 3).view(3, 2)
    for starts, lengths, written in (((0, 0, 0), (32, 32, 32), [0, 1, 2, 3]), ((-1, 0, 0), (20, 10, 33), [2]),
                                     ((0, 0, 0), (-5, 16, 0), [2])):
        means.zero_()
        sp.write_means(cache, means, table, ints(*starts), ints(*lengths))
        with pytest.raises(RuntimeError):
            cache.check()
        assert (means != 0).any(2).any(1).nonzero().flatten().tolist() == written
    sp.write_means(cache, means, table, ints(0, 0, 0), ints(32, 16, 0))
    cache.check()


# ----------------------------------------------------------------------- selection ----

def check_selection(q, cache, means, table, lengths, count, first, last, got):
    pages, tokens = (t.cpu() for t in got)
    page, kv_heads = cache.page, cache.kv_heads
    for b, n in enumerate(lengths):
        want = osp.select(q[b].cpu(), means.cpu(), table[b], n, page, count, first, last)
        for i, (picked, seen) in enumerate(want):
            assert int(tokens[b, i]) == seen
            for u in range(kv_heads):
                row = picked[u] if picked else []
                assert pages[b, i, u].tolist() == row + [-1] * (count - len(row)), (b, i, u)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16), (256, BF16),
                                       (256, FP16)])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (10, 2), (24, 1), (6, 3)])
@pytest.mark.parametrize("tokens", [1, 3])
@torch.no_grad()
def test_selection(device, dim, dtype, heads, kv_heads, tokens):
    g = torch.Generator().manual_seed(dim + heads)
    lengths = [1, 16, 17, 700, 333, 2, 95]
    table, pages = tables([-(-n // 16) for n in lengths])
    cache = kv.empty_cache(pages, kv_heads, dim, 16, device="cuda")
    means = torch.randn(pages, kv_heads, dim, generator=g).to(BF16).cuda()
    wide = torch.randn(7, tokens, heads + 3, dim, generator=g).to(dtype).cuda()
    q = wide[:, :, 1:heads + 1]
    for count, first, last in ((1, 0, 1), (5, 1, 1), (12, 2, 3), (44, 0, 1), (60, 4, 4)):
        got = sp.select_pages(q, cache, means, table.cuda(), ints(*lengths), count, first=first, last=last)
        check_selection(q, cache, means, table, lengths, count, first, last, got)
        if tokens == 1:
            flat = sp.select_pages(q[:, 0], cache, means, table.cuda(), ints(*lengths), count, first=first,
                                   last=last)
            assert torch.equal(flat[0], got[0][:, 0]) and torch.equal(flat[1], got[1][:, 0])
    cache.check()


@pytest.mark.parametrize("length,count", [(16 * 257, 3), (16 * 1500 - 3, 64), (16 * 5000, 700), (16 * 9000, 8999), (16 * 20000, 37)])
@torch.no_grad()
def test_selection_of_long_sequences(device, length, count):
    """Keys in a workspace, and scores that share their upper bits."""
    g = torch.Generator().manual_seed(length)
    table, pages = tables([-(-length // 16), 3])
    cache = kv.empty_cache(pages, 2, 64, 16, device="cuda")
    means = (1 + 2.0 ** -7 * torch.randint(0, 3, (pages, 2, 64), generator=g)).to(BF16).cuda()
    q = torch.ones(2, 1, 4, 64, dtype=BF16).cuda()
    q[:, :, 1] = -1
    got = sp.select_pages(q, cache, means, table.cuda(), ints(length, 40), count)
    check_selection(q, cache, means, table, [length, 40], count, 1, 1, got)


@pytest.mark.parametrize("pages_of_one", [100, 300, 1100])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (128, FP16), (256, BF16), (256, FP16)])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1), (5, 1), (8, 1), (9, 1), (36, 2)])
@torch.no_grad()
def test_selection_of_every_group(device, pages_of_one, dim, dtype, heads, kv_heads):
    """Groups that end in the first and second four rows, scored by the workgroup that takes or by a
    grid over all pages."""
    g = torch.Generator().manual_seed(heads)
    table, pages = tables([pages_of_one, pages_of_one - 7])
    cache = kv.empty_cache(pages, kv_heads, dim, 16, device="cuda")
    means = torch.randn(pages, kv_heads, dim, generator=g).to(BF16).cuda()
    q = torch.randn(2, 1, heads, dim, generator=g).to(dtype).cuda()
    lengths = [16 * pages_of_one - 3, 16 * (pages_of_one - 7)]
    got = sp.select_pages(q, cache, means, table.cuda(), ints(*lengths), 20)
    check_selection(q, cache, means, table, lengths, 20, 1, 1, got)


@pytest.mark.parametrize("spread", ["even", "alike", "two", "infinite"])
@torch.no_grad()
def test_selection_where_scores_crowd(device, spread):
    """Many pages: scores spread evenly, all within a millionth but for two far off, of two values only,
    and with infinities of both signs among them."""
    n, dim = 6001, 64
    g = torch.Generator().manual_seed(1)
    table, pages = tables([n, 700])
    cache = kv.empty_cache(pages, 1, dim, 16, device="cuda")
    means = torch.zeros(pages, 1, dim)
    if spread == "even":
        means[:, 0, :4] = torch.randn(pages, 4, generator=g)
    elif spread == "alike":
        means[:, 0, 0] = 1000
        means[:, 0, 1] = 2.0 ** -8 * torch.rand(pages, generator=g)
        means[table[0, 17], 0, 0], means[table[0, 400], 0, 0] = 3e38, -3e38
    elif spread == "two":
        means[:, 0, 0] = torch.randint(0, 2, (pages,), generator=g).float()
    else:
        means[:, 0, 0] = torch.randn(pages, generator=g)
        means[table[0, 5::100].long(), 0, 0] = math.inf
        means[table[0, 7::50].long(), 0, 0] = -math.inf
    means = means.to(BF16).cuda()
    q = torch.zeros(2, 1, 2, dim, dtype=BF16, device="cuda")
    q[..., :4] = 1
    lengths = [16 * n - 5, 16 * 700]
    for count in (2, 50, 300, 5000):
        got = sp.select_pages(q, cache, means, table.cuda(), ints(*lengths), count)
        check_selection(q, cache, means, table, lengths, count, 1, 1, got)


@pytest.mark.parametrize("width", [256, 257, 511, 512, 513, 4096])
@pytest.mark.parametrize("dim,dtype,tokens,crowded", [(64, BF16, 1, False), (128, FP16, 1, True), (256, BF16, 2, False)])
@torch.no_grad()
def test_selection_of_many_units(device, width, dim, dtype, tokens, crowded):
    """Four units a CU and more: one workgroup scores and takes a unit's pages, up to 4096. A few sequences against the
    oracle, all against themselves in small batches, which go through a workspace."""
    g = torch.Generator().manual_seed(width)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    kv_heads, heads, page = 8, 16, 16
    batch = 4 * cus // (kv_heads * tokens) + 2
    pool = 5000
    cache = kv.empty_cache(pool, kv_heads, dim, page, device="cuda")
    if crowded:                                              # few values, ties everywhere
        means = torch.randint(-1, 2, (pool, kv_heads, dim), generator=g).to(BF16)
        q = torch.zeros(batch, tokens, heads, dim)
        q[..., :2] = 1
        q = q.to(dtype).cuda()
    else:
        means = torch.randn(pool, kv_heads, dim, generator=g).to(BF16)
        q = torch.randn(batch, tokens, heads, dim, generator=g).to(dtype).cuda()
    table = torch.stack([torch.randperm(pool, generator=g)[:width] for _ in range(batch)]).int()
    lengths = torch.randint(1, width * page + 1, (batch,), generator=g).tolist()
    lengths[:6] = [width * page, width * page - 15, 1, 20 * page, 21 * page + 1, 0]
    count, ids = 20, ints(*lengths)
    got = sp.select_pages(q, cache, means.cuda(), table.cuda(), ids, count, first=2, last=2)
    for b in (0, 1, 2, 3, 4, 5, batch - 1):
        check_selection(q[b:b + 1], cache, means, table[b:b + 1], lengths[b:b + 1], count, 2, 2, [t[b:b + 1] for t in got])
    for b in range(0, batch, 10):
        part = slice(b, b + 10)
        alone = sp.select_pages(q[part], cache, means.cuda(), table[part].cuda(), ids[part], count, first=2, last=2)
        assert torch.equal(alone[0], got[0][part]) and torch.equal(alone[1], got[1][part])
    cache.check()


@torch.no_grad()
def test_selection_from_the_widest_tables(device):
    """512 sequences with tables of 65536 pages: 2 GiB of keys. The long ones, at both ends, against themselves
    alone; and one sequence too many is refused."""
    pool, heads, dim, batch, width, count = 3000, 8, 64, 512, 65536, 40
    g = torch.Generator().manual_seed(2)
    cache = kv.empty_cache(pool, heads, dim, 16, device="cuda")
    means = torch.randn(pool, heads, dim, generator=g).to(BF16).cuda()
    q = torch.randn(batch, heads, dim, generator=g).to(BF16).cuda()
    table = torch.randint(0, pool, (batch, width), generator=g, dtype=torch.int32).cuda()
    lengths = torch.randint(1, 2000, (batch,), generator=g, dtype=torch.int32)
    long = [0, 1, batch - 2, batch - 1]
    lengths[long] = torch.tensor([16 * width, 16 * 9000, 16 * 5000 - 3, 16 * width - 20], dtype=torch.int32)
    lengths = lengths.cuda()
    got = sp.select_pages(q, cache, means, table, lengths, count)
    for b in [*long, 7, 300]:
        rows = slice(b, b + 1)
        alone = sp.select_pages(q[rows], cache, means, table[rows], lengths[rows], count)
        assert torch.equal(got[0][rows], alone[0]) and torch.equal(got[1][rows], alone[1])
    cache.check()
    many = 2 ** 14 // heads
    with pytest.raises(ValueError, match="too many"):
        sp.select_pages(q[:1].expand(many, -1, -1), cache, means, table[:1].expand(many, -1), lengths[:1].repeat(many), count)


@pytest.mark.parametrize("length", [16 * 40, 16 * 600])
@torch.no_grad()
def test_equal_scores_go_to_the_front_and_nan_first(device, length):
    n = length // 16
    table, pages = tables([n])
    cache = kv.empty_cache(pages, 1, 64, 16, device="cuda")
    means = torch.zeros(pages, 1, 64, dtype=BF16)
    q = torch.ones(1, 1, 1, 64, dtype=FP16).cuda()
    for special in ((), (7,), (7, 30)):
        means.zero_()
        for at in special:
            means[int(table[0, at]), 0, 3] = math.nan
        means[int(table[0, 20])] = -0.0                       # equals 0
        means[int(table[0, 21])] = -math.inf
        got = sp.select_pages(q, cache, means.cuda(), table.cuda(), ints(length), 9)
        check_selection(q, cache, means, table, [length], 9, 1, 1, got)
    all_nan = sp.select_pages(q * math.nan, cache, means.cuda(), table.cuda(), ints(length), 9)
    assert all_nan[0][0, 0, 0].tolist() == table[0, :8].tolist() + [int(table[0, n - 1])]


@torch.no_grad()
def test_selection_faults_reach_the_attention(device):
    for width in (40, 400):
        cache, _, _ = filled(6 * width, 2, 64, 16)
        means = torch.randn(6 * width, 2, 64).to(BF16).cuda()
        table = torch.arange(3 * width, dtype=torch.int32).view(3, width)
        table[1, width // 2] = 6 * width                      # not in the pool
        q = torch.randn(3, 1, 4, 64).to(BF16).cuda()
        lengths = ints(width * 16, width * 16, width * 16 + 1)
        got = sp.select_pages(q, cache, means, table.cuda(), lengths, 4)
        with pytest.raises(RuntimeError):
            cache.check()
        check_selection(q[:1], cache, means, table, [width * 16], 4, 1, 1, got)
        assert (got[0][1] == 6 * width).any(-1).all() and int(got[1][2]) == -1 and (got[0][2] == -1).all()
        out = sp.selected_attention(q, cache, *got)
        with pytest.raises(RuntimeError):
            cache.check()
        assert torch.isfinite(out[0]).all() and out[1:].isnan().all()


# ----------------------------------------------------------------------- attention ----

def check_attention(q, values, page, pages, tokens, out, lse, scale):
    keys, vals = values
    kv_heads = keys.shape[1]
    group = q.shape[2] // kv_heads
    for b in range(q.shape[0]):
        for i in range(q.shape[1]):
            n = int(tokens[b, i])
            for u in range(kv_heads):
                p = pages[b, i, u, :-(-n // page)].long().cpu()
                k = keys[p, u].flatten(0, 1)[:n, None]
                v = vals[p, u].flatten(0, 1)[:n, None]
                hs = slice(u * group, (u + 1) * group)
                o, l, mass, size = oc.attention(q[b, i, None, hs].cpu(), k, v, n, scale)
                near, l_near = oc.bounds(o, mass, size, v, q.dtype, q.shape[-1], max(n, 1))
                assert ((out[b, i, hs].cpu().double() - o[0]).abs() <= near[0]).all(), (b, i, u)
                if lse is not None and n:
                    assert ((lse[b, i, hs].cpu().double() - l[0]).abs() <= l_near[0]).all(), (b, i, u)
                if n == 0:
                    assert (out[b, i] == 0).all() and (lse is None or (lse[b, i] == -math.inf).all())


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16), (256, BF16)])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(3, 3, 1), (10, 2, 2), (20, 1, 1)])
@torch.no_grad()
def test_attention_over_selected_pages(device, page, dim, dtype, heads, kv_heads, tokens):
    g = torch.Generator().manual_seed(page)
    lengths = [1, 9 * page + 5, 4 * page, 700 + page]
    table, pages = tables([-(-n // page) for n in lengths])
    cache, *values = filled(pages, kv_heads, dim, page)
    means = sp.empty_means(cache)
    sp.write_means(cache, means, table.cuda(), ints(0, 0, 0, 0), ints(*lengths))
    wide = torch.randn(4, tokens, heads + 2, dim, generator=g).to(dtype).cuda()
    q = wide[:, :, :heads]
    got = sp.select_pages(q, cache, means, table.cuda(), ints(*lengths), 5, first=1, last=2)
    out, lse = sp.selected_attention(q, cache, *got, return_lse=True)
    check_attention(q, values, page, *got, out, lse, dim ** -0.5)
    again = sp.selected_attention(q, cache, *got, scale=0.02, out=q)
    assert again is q
    cache.check()


@pytest.mark.parametrize("batch,kv_heads,dim,count", [(70, 8, 128, 9), (130, 3, 64, 40), (40, 8, 256, 3)])
@torch.no_grad()
def test_many_queries_a_workgroup_each(device, batch, kv_heads, dim, count):
    """As many units as the card has places, short and empty ones among them."""
    g = torch.Generator().manual_seed(batch)
    page = 16
    lengths = torch.randint(0, 50 * page, (batch,), generator=g).tolist()
    lengths[3], lengths[5] = 0, 1
    table, pages = tables([-(-n // page) for n in lengths])
    cache, *values = filled(pages, kv_heads, dim, page)
    q = torch.randn(batch, 1, 2 * kv_heads, dim, generator=g).to(BF16).cuda()
    means = sp.empty_means(cache)
    sp.write_means(cache, means, table.cuda(), torch.zeros(batch, dtype=torch.int32).cuda(), ints(*lengths))
    got = sp.select_pages(q, cache, means, table.cuda(), ints(*lengths), count)
    out, lse = sp.selected_attention(q, cache, *got, return_lse=True)
    some = [0, 3, 5, batch // 2, batch - 1]
    check_attention(q[some], values, page, got[0][some], got[1][some], out[some], lse[some], dim ** -0.5)
    again = sp.selected_attention(q[7:8], cache, got[0][7:8].contiguous(), got[1][7:8].contiguous())
    assert (again - out[7:8]).abs().max() <= 2.0 ** -6 * out[7:8].abs().max()       # alone it may be split
    cache.check()


@torch.no_grad()
def test_all_pages_are_the_dense_attention(device):
    """A selection that leaves nothing out gives cache_attention's bits, steps of a prompt and behind it."""
    lengths = [300, 64, 1, 4097]
    table, pages = tables([-(-n // 64) for n in lengths])
    cache, _, _ = filled(pages, 4, 128, 64)
    means = sp.empty_means(cache).zero_()
    q = torch.randn(4, 8, 128).to(BF16).cuda()
    got = sp.select_pages(q, cache, means, table.cuda(), ints(*lengths), 65)
    dense = kv.cache_attention(q, cache, table.cuda(), ints(*lengths), return_lse=True)
    some = sp.selected_attention(q, cache, *got, return_lse=True)
    assert torch.equal(dense[0], some[0]) and torch.equal(dense[1], some[1])


@torch.no_grad()
def test_write_means_select_attend(device):
    """A prompt and steps behind it as they are used: every mean is that of the codes, the selection the
    oracle's, the attention within its bounds; eagerly and captured, on another stream."""
    dim, page, kv_heads, heads, batch, count = 64, 16, 2, 6, 3, 6
    g = torch.Generator().manual_seed(5)
    prompts = [100, 37, 250]
    table = torch.randperm(64, generator=g)[:60].int().view(3, 20)
    cache = kv.empty_cache(64, kv_heads, dim, page, device="cuda")
    for s in (cache.k_scales, cache.v_scales):
        s.fill_(127)
    for c in (cache.k_codes, cache.v_codes):
        c.zero_()
    means = sp.empty_means(cache).zero_()
    dev_table, lengths = table.cuda(), ints(*prompts)
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    rows = torch.randn(2, sum(prompts), kv_heads, dim, generator=g).to(BF16).cuda()
    kv.write_cache(cache, rows[0], rows[1], dev_table, zero, ints(0, 100, 137, 387))
    sp.write_means(cache, means, dev_table, zero, lengths)
    q = torch.zeros(batch, heads, dim, dtype=BF16, device="cuda")
    k, v = (torch.zeros(batch, kv_heads, dim, dtype=BF16, device="cuda") for _ in range(2))

    def step():
        kv.write_cache(cache, k, v, dev_table, lengths)
        after = lengths + 1
        sp.write_means(cache, means, dev_table, lengths, after)
        lengths.copy_(after)
        got = sp.select_pages(q, cache, means, dev_table, lengths, count)
        return got, sp.selected_attention(q, cache, *got, return_lse=True)

    side = torch.cuda.Stream()
    graph = None
    for n in range(1, 8):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        if n == 4:
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got, (out, lse) = step()
        if graph is None:
            got, (out, lse) = step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        now = [p + n for p in prompts]
        assert lengths.tolist() == now
        codes = cache.k_codes.cpu().view(torch.float8_e4m3fn).double()
        keys = codes * torch.exp2(cache.k_scales.cpu().double() - 127)[..., None, None]
        codes = cache.v_codes.cpu().view(torch.float8_e4m3fn).double()
        vals = (codes * torch.exp2(cache.v_scales.cpu().double() - 127)[..., None, None]).transpose(2, 3)
        for b, m in enumerate(now):
            for at in range(-(-m // page)):
                p = int(table[b, at])
                assert torch.equal(means[p].cpu().double(), osp.mean(keys[p], min(page, m - at * page)))
        check_selection(q[:, None], cache, means, table, now, count, 1, 1, [t[:, None] for t in got])
        check_attention(q[:, None], (keys, vals), page, *(t[:, None] for t in got), out[:, None], lse[:, None],
                        dim ** -0.5)
    cache.check()


@torch.no_grad()
def test_two_graphs_of_a_long_selection(device):
    """Captured selections with workspaces of their own, replayed in turn."""
    table, pages = tables([600, 500])
    cache, _, _ = filled(pages, 2, 64, 16)
    means = torch.randn(pages, 2, 64).to(BF16).cuda()
    lengths = ints(9600, 8000)
    q = [torch.randn(2, 1, 4, 64).to(BF16).cuda() for _ in range(2)]
    graphs, outs = [], []
    for x in q:
        sp.select_pages(x, cache, means, table.cuda(), lengths, 30)
        t = table.cuda()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = sp.select_pages(x, cache, means, t, lengths, 30)
            outs.append((*got, sp.selected_attention(x, cache, *got)))
        graphs.append((graph, t))
    for _ in range(3):
        for x, (graph, t), out in zip(q, graphs, outs):
            x.normal_()
            graph.replay()
            got = sp.select_pages(x, cache, means, t, lengths, 30)
            want = (*got, sp.selected_attention(x, cache, *got))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@torch.no_grad()
def test_refusals_and_nothing_to_do(device):
    cache, _, _ = filled(4, 2, 64, 16)
    means = sp.empty_means(cache).zero_()
    t, n, q = ints(0, 1).view(1, 2), ints(20), torch.zeros(1, 1, 4, 64, dtype=BF16).cuda()
    pages, tokens = sp.select_pages(q, cache, means, t, n, 2)
    for call in (lambda: sp.write_means(cache, means[:2], t, n, n), lambda: sp.write_means(cache, means.half(), t, n, n),
                 lambda: sp.write_means(cache, means, t.long(), n, n), lambda: sp.write_means(cache, means, t, n, n.cpu()),
                 lambda: sp.write_means(cache, means, t, ints(1, 2), n), lambda: sp.write_means(cache, means, t[:, :0], n, n),
                 lambda: sp.write_means(cache, means.cpu(), t, n, n),
                 lambda: sp.select_pages(q[0, 0], cache, means, t, n, 2), lambda: sp.select_pages(q[:, :, :3], cache, means, t, n, 2),
                 lambda: sp.select_pages(q.float(), cache, means, t, n, 2), lambda: sp.select_pages(q, cache, means.float(), t, n, 2),
                 lambda: sp.select_pages(q, cache, means, t, n, 1), lambda: sp.select_pages(q, cache, means, t, n, 2.0),
                 lambda: sp.select_pages(q, cache, means, t, n, 3, last=0), lambda: sp.select_pages(q, cache, means, t, n, 3, first=-1),
                 lambda: sp.select_pages(q, cache, means, ints(0, 1).view(2, 1), n, 2),
                 lambda: sp.selected_attention(q, cache, pages[0], tokens), lambda: sp.selected_attention(q, cache, pages.long(), tokens),
                 lambda: sp.selected_attention(q, cache, pages[..., :0], tokens), lambda: sp.selected_attention(q, cache, pages[:, :, :1], tokens),
                 lambda: sp.selected_attention(q, cache, pages, tokens[0]), lambda: sp.selected_attention(q, cache, pages, tokens.long()),
                 lambda: sp.selected_attention(q, cache, pages.cpu(), tokens), lambda: sp.selected_attention(q, cache, pages, tokens, 0.0),
                 lambda: sp.selected_attention(q, cache, pages, tokens, out=q[:, :, :2]),
                 lambda: sp.selected_attention(q, cache, pages, tokens, out=q[..., :1].expand(1, 1, 4, 64))):
        with pytest.raises(ValueError):
            call()
    wide = torch.zeros(3, 2, 2, 4, 64, dtype=BF16).cuda()
    with pytest.raises(ValueError, match="stride"):
        sp.selected_attention(wide[:, 0], cache, torch.zeros(3, 2, 2, 1).int().cuda(), torch.zeros(3, 2).int().cuda())
    assert sp.selected_attention(q[:0], cache, pages[:0], tokens[:0]).shape == (0, 1, 4, 64)
    none = sp.select_pages(q[:0], cache, means, t[:0], n[:0], 2)
    assert none[0].shape == (0, 1, 2, 2) and none[1].shape == (0, 1)
    sp.write_means(cache, means, t[:0], n[:0], n[:0])
    cache.check()
