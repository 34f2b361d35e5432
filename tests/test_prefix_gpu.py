"""GPU: attention over shared prefixes and own tails against float64, within the bounds of oracle/causal.py."""
import math

import pytest
import torch

from oracle import causal as oc
from vdn_amd import kvcache as kv
from vdn_amd import prefix as vp

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def filled(pages, kv_heads, dim, page, seed=0, low=-9):
    """A cache of random finite codes and scales, and the float64 values of its K and V."""
    g = torch.Generator().manual_seed(seed)
    cache = kv.empty_cache(pages, kv_heads, dim, page, device="cuda")
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        c = (torch.randn(codes.shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        codes.copy_(c.view(torch.uint8))
        scales.copy_((torch.randint(low, -4, scales.shape, generator=g) + 127).to(torch.uint8))
    return cache


def values_of(cache):
    k = cache.k_codes.cpu().view(torch.float8_e4m3fn).double()
    v = cache.v_codes.cpu().view(torch.float8_e4m3fn).double()
    return k * torch.exp2(cache.k_scales.cpu().double() - 127)[..., None, None], \
        (v * torch.exp2(cache.v_scales.cpu().double() - 127)[..., None, None]).transpose(2, 3)


class Batch:
    """Prefixes and tails with pages of their own in random order, -1 behind them."""

    def __init__(self, prefixes, counts, tails, kv_heads, dim, page, seed=0, **kwargs):
        g = torch.Generator().manual_seed(seed)
        self.prefixes, self.counts, self.tails, self.page = prefixes, counts, tails, page
        need = [-(-n // page) for n in prefixes + tails]
        order = torch.randperm(sum(need) + 2, generator=g).tolist()
        rows = [[order.pop() for _ in range(n)] for n in need]

        def table(rows):
            width = max([len(r) for r in rows] + [1])
            return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32).view(-1, width)

        self.shared, self.table = table(rows[:len(prefixes)]), table(rows[len(prefixes):])
        self.cache = filled(sum(need) + 2, kv_heads, dim, page, seed, **kwargs)
        self.owner = [p for p, n in enumerate(counts) for _ in range(n)]

    def plan(self, heads, tokens=1):
        return vp.prepare_prefix_plan(self.prefixes, self.counts, heads, self.cache.kv_heads, self.cache.head_dim,
                                      tokens=tokens, device="cuda")

    def run(self, q, plan, **kwargs):
        return vp.prefix_attention(q, self.cache, self.shared.cuda(), plan, self.table.cuda(), ints(*self.tails),
                                   **kwargs)

    def keys(self, row, n, side):
        if n == 0:
            return side[:1].flatten(0, 1)[:0].transpose(0, 1).reshape(0, side.shape[1], side.shape[3])
        return torch.cat([side[int(p)].transpose(0, 1) for p in row[:-(-n // self.page)]])[:n]

    def check(self, q, out, lse=None, scale=None, rows=None):
        k_all, v_all = values_of(self.cache)
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        q, out = q.cpu(), out.cpu().double()
        tokens = q.shape[1]
        for b, p in enumerate(self.owner):
            if rows is not None and b not in rows:
                continue
            n, m = self.prefixes[p], self.tails[b]
            k, v = (torch.cat((self.keys(self.shared[p], n, s), self.keys(self.table[b], m, s)))
                    for s in (k_all, v_all))
            for i in range(tokens):
                sees = n + max(0, m - tokens + 1 + i)
                o, l, mass, size = oc.attention(q[b, i:i + 1], k[:sees], v[:sees], sees, scale)
                near, l_near = oc.bounds(o, mass, size, v[:sees], q.dtype, q.shape[-1], max(sees, 1))
                assert ((out[b, i] - o[0]).abs() <= near[0]).all(), (b, i, float((out[b, i] - o[0]).abs().max()))
                if sees == 0:
                    assert (out[b, i] == 0).all() and (lse is None or (lse[b, i] == -math.inf).all())
                elif lse is not None:
                    assert ((lse[b, i].cpu().double() - l[0]).abs() <= l_near[0]).all(), (b, i)


def queries(batch, tokens, heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(batch, tokens, heads + 2, dim, generator=g).to(dtype).cuda()[:, :, 1:heads + 1]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16), (256, BF16), (256, FP16)])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(1, 1, 1), (10, 2, 1), (6, 3, 3), (24, 1, 2)])
@torch.no_grad()
def test_against_the_definition(device, page, dim, dtype, heads, kv_heads, tokens):
    case = Batch([65, 0, 300, 1, 64, 17], [2, 2, 3, 1, 0, 1], [5, 1, 3, 0, 70, 33, 2, 1, 16], kv_heads, dim, page)
    q = queries(9, tokens, heads, dim, dtype)
    out, lse = case.run(q, case.plan(heads, tokens), return_lse=True)
    assert out.is_contiguous() and lse.shape == out.shape[:-1]
    case.check(q, out, lse)
    case.cache.check()
    if tokens == 1:
        flat = case.run(q[:, 0], case.plan(heads))
        assert flat.shape == (9, heads, dim) and torch.equal(flat, out[:, 0])


@pytest.mark.parametrize("prefix,count,heads,kv_heads,dim,dtype,page", [
    (5000, 40, 32, 4, 128, BF16, 64),      # three blocks of rows, many pieces, a ragged tile
    (4099, 9, 16, 8, 64, FP16, 16),        # eight K/V heads, small pages
    (3001, 33, 8, 2, 256, BF16, 128),
    (20000, 3, 4, 1, 128, FP16, 256),      # few rows and many pieces
])
@torch.no_grad()
def test_blocks_and_pieces(device, prefix, count, heads, kv_heads, dim, dtype, page):
    tails = [(37 * i) % 700 for i in range(count)]           # wide tables: tails may be split, too
    case = Batch([prefix], [count], tails, kv_heads, dim, page)
    q = queries(count, 1, heads, dim, dtype)
    plan = case.plan(heads)
    assert plan.items.shape[0] > 3
    out, lse = case.run(q, plan, return_lse=True)
    case.check(q, out, lse, rows={0, 1, count // 2, count - 1})
    again = case.run(q, plan, return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("longest", [40, 500])              # a wave's tile, and tables of two steps
@pytest.mark.parametrize("dim,dtype,page", [(64, FP16, 16), (128, BF16, 64), (128, FP16, 128), (256, BF16, 32)])
@torch.no_grad()
def test_many_short_tails(device, longest, dim, dtype, page):
    """More tails than the card takes at once, empty ones between them, more query rows than a row block."""
    count, heads, kv_heads, tokens = 75, 48, 16, 6
    tails = [(53 * i) % (longest + 1) if i % 7 else 0 for i in range(count - 1)] + [longest]
    case = Batch([70, 0], [count - 1, 1], tails, kv_heads, dim, page)
    q = queries(count, tokens, heads, dim, dtype)
    plan = case.plan(heads, tokens)
    out, lse = case.run(q, plan, return_lse=True)
    case.check(q, out, lse, rows={0, 1, 2, 7, 30, 51, count - 2, count - 1})
    again = case.run(q, plan, return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    case.cache.check()
    case.table[5, 0] = case.cache.pages                      # a page outside the pool
    bad = case.run(q, plan)
    assert bad[5].isnan().all() and torch.equal(bad[[4, 6, count - 1]], out[[4, 6, count - 1]])
    with pytest.raises(RuntimeError):
        case.cache.check()


@torch.no_grad()
def test_as_cache_attention_over_both_parts(device):
    """The same pages through tables that repeat the prefix: both within the bound of the definition."""
    page, heads, kv_heads, dim = 16, 12, 4, 64
    case = Batch([160, 48], [3, 2], [20, 1, 33, 7, 16], kv_heads, dim, page)
    q = queries(5, 1, heads, dim, BF16)
    out, lse = case.run(q, case.plan(heads), return_lse=True, scale=0.3)
    rows = [case.shared[p, :case.prefixes[p] // page].tolist() + [t for t in case.table[b].tolist() if t >= 0]
            for b, p in enumerate(case.owner)]
    width = max(len(r) for r in rows)
    both = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32).cuda()
    lengths = ints(*(case.prefixes[p] + t for p, t in zip(case.owner, case.tails)))
    dense = kv.cache_attention(q, case.cache, both, lengths, 0.3, return_lse=True)
    case.check(q, out, lse, 0.3)
    case.check(q, *dense, 0.3)


@pytest.mark.parametrize("dim,dtype,page", [(64, FP16, 16), (128, BF16, 64), (128, FP16, 256), (256, BF16, 32)])
@torch.no_grad()
def test_nan_codes(device, dim, dtype, page):
    """NaN codes behind a prefix's last token reach nobody; a NaN value inside reaches its channel in
    all its sequences and no other's; a NaN key makes its prefix's rows NaN."""
    case = Batch([page + 5, 3 * page - 7, 40], [2, 1, 2], [3, 2, 20, 1, 5], 2, dim, page)
    c = case.cache
    for p, n in enumerate(case.prefixes):
        last = int(case.shared[p, (n - 1) // page])
        c.k_codes[last, :, (n - 1) % page + 1:] = 0x7f
        c.v_codes[last, :, :, (n - 1) % page + 1:] = 0xff
    q = queries(5, 1, 4, dim, dtype)
    plan = case.plan(4)
    clean = case.run(q, plan)
    assert torch.isfinite(clean).all()
    c.v_codes[int(case.shared[1, 1]), 1, 9, 3] = 0x7f
    out = case.run(q, plan)
    bad = out.isnan().nonzero().tolist()
    assert bad == [[2, 0, 2, 9], [2, 0, 3, 9]]
    assert torch.equal(torch.nan_to_num(out)[[0, 1, 3, 4]], clean[[0, 1, 3, 4]])
    c.k_codes[int(case.shared[0, 0]), 0, 2, 7] = 0xff
    out = case.run(q, plan)
    assert out[:2, :, :2].isnan().all() and torch.isfinite(out[:2, :, 2:]).all()
    assert torch.equal(out[3:], clean[3:])
    c.check()


@torch.no_grad()
def test_fp16_scales_far_apart(device):
    """fp16: pages whose values are 2^-20 of their neighbours', the heavy token in a small page."""
    page, dim = 16, 64
    case = Batch([128], [2], [4, 20], 1, dim, page)
    c = case.cache
    low = case.shared[0, ::2].long().cuda()
    c.v_scales[low] = 127 - 24
    c.v_scales[case.shared[0, 1::2].long().cuda()] = 127 - 2
    c.v_scales[case.table[1, :2].long().cuda()] = 127 - 30
    q = queries(2, 1, 2, dim, FP16)
    out, lse = case.run(q, case.plan(2), return_lse=True)
    case.check(q, out, lse)
    # one token takes all the weight: its small value comes through
    c.k_codes.zero_()
    c.k_codes[int(low[1]), 0, 5] = 0x7e
    c.k_scales.fill_(127)
    q = torch.ones(2, 1, 2, dim, dtype=FP16, device="cuda")
    out = case.run(q, case.plan(2), scale=1.0)
    _, v = values_of(c)
    want = v[int(low[1]), 0, 5]
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -24).all()


@torch.no_grad()
def test_rows_that_see_nothing_and_scores_that_are_infinite(device):
    case = Batch([0, 40], [2, 2], [0, 2, 0, 1], 1, 64, 16)
    q = queries(4, 3, 2, 64, BF16)
    out, lse = case.run(q, case.plan(2, 3), return_lse=True)
    case.check(q, out, lse)
    assert (out[0] == 0).all() and (out[1, 0] == 0).all() and (out[1, 1] != 0).any()
    case.cache.k_codes.fill_(0xb8)                              # -1
    q[2:] = math.inf                                            # scores -inf: no softmax
    out, lse = case.run(q, case.plan(2, 3), return_lse=True)
    assert out[2:].isnan().all() and (lse[2:] == -math.inf).all() and torch.isfinite(out[:2]).all()


@torch.no_grad()
def test_faults(device):
    for page in (16, 64):
        case = Batch([4 * page + 3, page], [2, 1], [3, 2, 5], 2, 64, page)
        q = queries(3, 1, 4, 64, BF16)
        plan = case.plan(4)
        clean = case.run(q, plan)
        good = int(case.shared[0, 2])
        for bad in (-1, case.cache.pages, 2 ** 31 - 1):
            case.shared[0, 2] = bad
            out = case.run(q, plan)
            with pytest.raises(RuntimeError):
                case.cache.check()
            assert out[:2].isnan().all() and torch.equal(out[2], clean[2])
        case.shared[0, 2] = good
        for bad in (-1, case.table.shape[1] * page + 1):
            case.tails[1] = bad
            out = case.run(q, plan)
            with pytest.raises(RuntimeError):
                case.cache.check()
            assert out[1].isnan().all() and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
        case.tails[1] = 2


@torch.no_grad()
def test_strides_out_and_tables(device):
    case = Batch([100, 30], [3, 2], [9, 1, 4, 20, 2], 2, 128, 32)
    q = queries(5, 2, 6, 128, BF16)
    plan = case.plan(6, 2)
    want, want_lse = case.run(q, plan, return_lse=True)
    wide = torch.zeros(5, 2, 9, 3, 128, dtype=BF16, device="cuda")
    out = wide[:, :, 1:7, 1]
    got, lse = case.run(q, plan, return_lse=True, out=out)
    assert got is out and torch.equal(out, want) and torch.equal(lse, want_lse)
    out.zero_()
    assert (wide == 0).all()
    tables = [torch.cat((t, t.flip(0)), 1).cuda() for t in (case.shared, case.table)]      # wider rows
    got = vp.prefix_attention(q, case.cache, tables[0][:, :case.shared.shape[1]], plan,
                              tables[1][:, :case.table.shape[1]], ints(*case.tails))
    assert torch.equal(got, want)
    assert case.run(q, plan, out=q) is q and torch.equal(q, want)


@torch.no_grad()
def test_growing_tails_streams_and_two_graphs(device):
    """Steps behind a prefix: tails grow in place, eagerly on a side stream and in two captured graphs
    that are replayed in turn, each with a workspace of its own."""
    page, heads, kv_heads, dim = 16, 8, 2, 64
    case = Batch([200, 33], [4, 2], [600] * 6, kv_heads, dim, page)
    shared, table, lengths = case.shared.cuda(), case.table.cuda(), ints(*[1] * 6)
    plan = case.plan(heads)
    q = [torch.randn(6, heads, dim).to(BF16).cuda() for _ in range(2)]
    graphs, outs = [], []
    vp.prefix_attention(q[0], case.cache, shared, plan, table, lengths)
    for x in q:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(vp.prefix_attention(x, case.cache, shared, plan, table, lengths, return_lse=True))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for step in (1, 2, 63, 64, 600):
        lengths.copy_(torch.tensor([max(1, step - 7 * i) for i in range(6)], dtype=torch.int32))
        for x, graph, out in zip(q, graphs, outs):
            x.normal_()
            graph.replay()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                want = vp.prefix_attention(x, case.cache, shared, plan, table, lengths, return_lse=True)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            case.tails = lengths.tolist()
            case.check(x[:, None], out[0][:, None], out[1][:, None])


@torch.no_grad()
def test_pages_behind_two_to_the_31_bytes(device):
    """A prefix and tails in the last pages of a pool of more than 2^31 bytes a side."""
    page, dim = 256, 256
    pages = 2 ** 31 // (page * dim) + 40
    cache = kv.empty_cache(pages, 1, dim, page, device="cuda")
    small = Batch([700], [2], [300, 5], 1, dim, page)
    n = small.cache.pages
    for a, b in ((cache.k_codes, small.cache.k_codes), (cache.v_codes, small.cache.v_codes),
                 (cache.k_scales, small.cache.k_scales), (cache.v_scales, small.cache.v_scales)):
        a[-n:] = b
    q = queries(2, 1, 4, dim, BF16)
    plan = small.plan(4)
    want = small.run(q, plan)

    def moved(t):
        return torch.where(t >= 0, t + pages - n, t).int().cuda()

    got = vp.prefix_attention(q, cache, moved(small.shared), plan, moved(small.table), ints(*small.tails))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dim,dtype,page", [(64, FP16, 16), (64, BF16, 128), (128, BF16, 64), (128, FP16, 32),
                                            (256, BF16, 16), (256, FP16, 64)])
@pytest.mark.parametrize("count,group,tokens", [(4, 4, 1), (1, 17, 1), (5, 13, 2), (3, 7, 6)])
@torch.no_grad()
def test_few_rows(device, dim, dtype, page, count, group, tokens):
    """16 rows, 17, 130 (a block and two) and 126: few rows are taken by tiles, more by rows."""
    tails = [(41 * i + 7) % 90 for i in range(count + 1)]
    case = Batch([1100, 64 * 4 + 1], [count, 1], tails, 2, dim, page)
    q = queries(count + 1, tokens, 2 * group, dim, dtype)
    plan = case.plan(2 * group, tokens)
    out, lse = case.run(q, plan, return_lse=True)
    case.check(q, out, lse)
    again = case.run(q, plan, return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    case.cache.check()


@pytest.mark.parametrize("dim,dtype,page", [(64, FP16, 16), (128, BF16, 64), (128, FP16, 256), (256, BF16, 32)])
@pytest.mark.parametrize("heads", [4, 68])                      # few rows of a prefix, and a block of them
@torch.no_grad()
def test_odd_values_in_prefixes(device, dim, dtype, page, heads):
    """NaN codes behind the last token and inside, bad pages, infinite scores."""
    case = Batch([page + 5, 3 * page - 7, 40], [2, 1, 2], [3, 2, 20, 1, 5], 2, dim, page)
    c = case.cache
    for p, n in enumerate(case.prefixes):
        last = int(case.shared[p, (n - 1) // page])
        c.k_codes[last, :, (n - 1) % page + 1:] = 0x7f
        c.v_codes[last, :, :, (n - 1) % page + 1:] = 0xff
    q = queries(5, 1, heads, dim, dtype)
    plan, half = case.plan(heads), heads // 2
    clean = case.run(q, plan)
    assert torch.isfinite(clean).all()
    good = int(case.shared[1, 1])
    for bad in (-1, c.pages, 2 ** 31 - 1):
        case.shared[1, 1] = bad
        out = case.run(q, plan)
        with pytest.raises(RuntimeError):
            c.check()
        assert out[2].isnan().all() and torch.equal(out[[0, 1, 3, 4]], clean[[0, 1, 3, 4]])
    case.shared[1, 1] = good
    c.v_codes[good, 1, 9, 3] = 0x7f
    out = case.run(q, plan)
    assert out.isnan().nonzero().tolist() == [[2, 0, h, 9] for h in range(half, heads)]
    assert torch.equal(torch.nan_to_num(out)[[0, 1, 3, 4]], clean[[0, 1, 3, 4]])
    c.k_codes[int(case.shared[0, 0]), 0, 2, 7] = 0xff
    out = case.run(q, plan)
    assert out[:2, :, :half].isnan().all() and torch.isfinite(out[:2, :, half:]).all()
    assert torch.equal(out[3:], clean[3:])
    c.check()
    c.k_codes.fill_(0xb8)                                       # -1
    q[3:] = math.inf                                            # scores -inf: no softmax
    out, lse = case.run(q, plan, return_lse=True)
    assert out[3:].isnan().all() and (lse[3:] == -math.inf).all()


@torch.no_grad()
def test_fp16_scales_far_apart_in_a_block(device):
    page, dim, heads = 16, 64, 40
    case = Batch([128], [2], [4, 20], 1, dim, page)
    c = case.cache
    low = case.shared[0, ::2].long().cuda()
    c.v_scales[low] = 127 - 24
    c.v_scales[case.shared[0, 1::2].long().cuda()] = 127 - 2
    c.v_scales[case.table[1, :2].long().cuda()] = 127 - 30
    q = queries(2, 1, heads, dim, FP16)
    out, lse = case.run(q, case.plan(heads), return_lse=True)
    case.check(q, out, lse)
    c.k_codes.zero_()
    c.k_codes[int(low[1]), 0, 5] = 0x7e
    c.k_scales.fill_(127)
    q = torch.ones(2, 1, heads, dim, dtype=FP16, device="cuda")
    out = case.run(q, case.plan(heads), scale=1.0)
    _, v = values_of(c)
    want = v[int(low[1]), 0, 5]
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -24).all()


@torch.no_grad()
def test_a_block_behind_two_to_the_31_bytes(device):
    page, dim = 256, 256
    pages = 2 ** 31 // (page * dim) + 40
    cache = kv.empty_cache(pages, 1, dim, page, device="cuda")
    small = Batch([700], [2], [300, 5], 1, dim, page)
    n = small.cache.pages
    for a, b in ((cache.k_codes, small.cache.k_codes), (cache.v_codes, small.cache.v_codes),
                 (cache.k_scales, small.cache.k_scales), (cache.v_scales, small.cache.v_scales)):
        a[-n:] = b
    q = queries(2, 1, 40, dim, BF16)
    plan = small.plan(40)
    want = small.run(q, plan)

    def moved(t):
        return torch.where(t >= 0, t + pages - n, t).int().cuda()

    got = vp.prefix_attention(q, cache, moved(small.shared), plan, moved(small.table), ints(*small.tails))
    assert torch.equal(got, want)


@torch.no_grad()
def test_refusals_and_nothing_to_do(device):
    case = Batch([40, 20], [2, 1], [3, 2, 5], 2, 64, 16)
    c, s, t, n = case.cache, case.shared.cuda(), case.table.cuda(), ints(3, 2, 5)
    q, plan = queries(3, 1, 4, 64, BF16), case.plan(4)
    for call in (lambda: vp.prefix_attention(q[:2], c, s, plan, t[:2], n[:2]),
                 lambda: vp.prefix_attention(q, c, s, case.plan(4, 2), t, n),
                 lambda: vp.prefix_attention(q, c, s, case.plan(8), t, n),
                 lambda: vp.prefix_attention(q, c, s[:1], plan, t, n),
                 lambda: vp.prefix_attention(q, c, s[:, :2], plan, t, n),
                 lambda: vp.prefix_attention(q, c, s.long(), plan, t, n),
                 lambda: vp.prefix_attention(q, c, s, plan, t[:2], n),
                 lambda: vp.prefix_attention(q, c, s, plan, t[:, :0], n),
                 lambda: vp.prefix_attention(q, c, s, plan, t, n[:2]),
                 lambda: vp.prefix_attention(q, c, s, plan, t, n.cpu()),
                 lambda: vp.prefix_attention(q.float(), c, s, plan, t, n),
                 lambda: vp.prefix_attention(q, c, s, plan, t, n, 0.0),
                 lambda: vp.prefix_attention(q, c, s, plan, t, n, out=q[:, :, :2]),
                 lambda: vp.prefix_attention(q, c, s, plan, t, n, out=q[:1].expand(3, 1, 4, 64)),
                 lambda: vp.prefix_attention(q, c, s, vp.prepare_prefix_plan([40, 20], [2, 1], 4, 2, 64, device="cpu"),
                                             t, n)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        vp.prefix_attention(q, c, s, None, t, n)
    none = vp.prepare_prefix_plan([40], [0], 4, 2, 64, device="cuda")
    assert vp.prefix_attention(q[:0], c, s[:1], none, t[:0], n[:0]).shape == (0, 1, 4, 64)
    c.check()


@pytest.mark.parametrize("dim,dtype,page", [(64, FP16, 16), (128, BF16, 64), (256, BF16, 32)])
@torch.no_grad()
def test_many_small_prefixes(device, dim, dtype, page):
    """Prefixes of one to forty rows a K/V head in one call, whose partial results lie behind each other: the
    workspace is what their rows need."""
    n, heads, kv_heads = 300, 8, 4
    counts = [1 + (7 * i) % 20 if i % 3 == 0 else 1 for i in range(n)]
    case = Batch([1 + (37 * i) % 150 for i in range(n)], counts, [(11 * i) % 40 for i in range(sum(counts))], kv_heads, dim, page)
    q = queries(sum(counts), 1, heads, dim, dtype)
    plan = case.plan(heads)
    case.run(q, plan, return_lse=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = case.run(q, plan, return_lse=True)
    rows = 4 * (dim + 4) * (plan.slot_rows * kv_heads + sum(counts) * heads)
    assert torch.cuda.max_memory_allocated() - before < rows + 2 ** 23       # output, LSE, tables; blocks of the allocator
    case.check(q, out, lse, rows={0, 1, 5, 13, 14, 20, 100, 333, sum(counts) - 1})
    case.cache.check()
