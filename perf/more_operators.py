"""Workloads of long contexts and shared prefixes over the 8-bit key/value cache.

A case is a plain dict; its "kind" names the operator that a pass goes through:

  rotary   rotate_qk: queries and keys turned by their positions, with or without the norm of each head
  means    write_means: the mean key of every page that a prompt or a step touched
  select   select_pages: for each query and K/V head the pages whose mean keys score highest
  attend   selected_attention: each query over the pages that were selected for it
  prefix   prefix_attention: sequences that share long prefixes, each with a tail of its own

`own` selects how run() computes them: the framework's entry points, or plain torch in 32 bits (angles
and the selecting scores in 64).

The cache: pages of `page` tokens; K codes [pages, kv_heads, page, dim], V codes [pages, kv_heads,
dim, page], both E4M3 in uint8; one E8M0 byte (exponent + 127) for each page and head of K and of
V. A sequence's tokens lie in the pages that its row of the table names, in order.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FIRST, LAST = 1, 2       # pages that a selection always holds: the first ones and the newest
PARTS = (1.0, 32.0)      # turns within the original context below which a frequency is stretched
                         # wholly, and above which it is kept
EPS = 1e-6
MOST_ROTATED = 32768 * 48 * 128     # values of the largest listed rotation
MOST_CACHED = 1048576               # cached tokens x kv heads / 8 of the largest cache
MOST_PREFIX = 1.8e11                # operations of the largest listed prefix


def _rotary(name, sizes, far, heads, kv_heads, dim=128, part=None, layout="half", dtype="bf16",
            norm=False, scaling="none", factor=1.0):
    """`far`: the highest position that a sequence's first token has; `part`: rotated channels."""
    return dict(name=name, kind="rotary", batch=sizes[0], shortest=sizes[1], longest=sizes[2], far=far,
                heads=heads, kv_heads=kv_heads, dim=dim, part=part or dim, layout=layout, dtype=dtype,
                norm=norm, scaling=scaling, factor=factor)


def _means(name, sizes, new, kv_heads, dim=128, page=64):
    """`sizes`: tokens that the sequences hold; `new`: the most of them that are new."""
    return dict(name=name, kind="means", batch=sizes[0], shortest=sizes[1], longest=sizes[2], new=new,
                kv_heads=kv_heads, dim=dim, page=page)


def _cached(kind, name, sizes, count, heads, kv_heads, tokens=1, dim=128, dtype="bf16", page=64,
            lse=False):
    return dict(name=name, kind=kind, batch=sizes[0], shortest=sizes[1], longest=sizes[2], count=count,
                heads=heads, kv_heads=kv_heads, tokens=tokens, dim=dim, dtype=dtype, page=page,
                lse=lse)


def _prefix(name, prefixes, each, tails, heads, kv_heads, tokens=1, dim=128, dtype="bf16", page=64,
            lse=False):
    """`prefixes`: how many, the shortest and the longest; `each`: the most sequences of one."""
    return dict(name=name, kind="prefix", prefixes=prefixes[0], shortest=prefixes[1],
                longest=prefixes[2], each=each, short_tail=tails[0], long_tail=tails[1], heads=heads,
                kv_heads=kv_heads, tokens=tokens, dim=dim, dtype=dtype, page=page, lse=lse)


def listed():
    return [
        # a long document's projections, each head normalised and turned
        _rotary("rotary_prompt", (1, 32768, 32768), 0, 40, 8, norm=True),
        # a decode step far behind the trained context: one token each, neighbouring channels in pairs
        _rotary("rotary_step", (64, 1, 1), 131072, 32, 8, layout="interleaved", scaling="parts",
                factor=8.0),
        # ragged prompts, a quarter of wide heads turned, half precision
        _rotary("rotary_part", (24, 77, 400), 4097, 16, 2, dim=256, part=64, dtype="fp16", norm=True,
                scaling="linear", factor=4.0),
        # whole prompts went into the cache
        _means("means_prompts", (8, 2048, 8192), 8192, 8),
        # a decode step: one new token in each of 64 sequences
        _means("means_step", (64, 512, 8192), 1, 8),
        # a decode step over ragged sequences: 16 pages of up to 128
        _cached("select", "select_step", (64, 512, 8192), 16, 40, 8),
        # one sequence with a long past in small pages
        _cached("select", "select_long", (1, 131072, 131072), 128, 56, 8, page=16),
        # the step behind that selection: 2048 tokens of each long sequence
        _cached("attend", "attend_step", (64, 512, 16384), 32, 40, 8),
        # four drafted tokens, each with pages of its own, as many key heads as query heads
        _cached("attend", "attend_draft", (16, 100, 4097), 24, 12, 12, tokens=4, dim=64, dtype="fp16",
                page=16, lse=True),
        # a long document that 128 sequences ask about
        _prefix("prefix_document", (1, 65536, 65536), 128, (16, 1000), 40, 8),
        # a few samples of each of several prompts, an odd length, small pages, half precision
        _prefix("prefix_samples", (12, 77, 4097), 8, (1, 300), 32, 8, dim=64, dtype="fp16", page=16,
                lse=True),
        # the smallest: four sequences behind one short instruction
        _prefix("prefix_instruction", (1, 500, 500), 4, (4, 60), 12, 2, dim=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Query and key heads: one to one, grouped (odd groups too), one for all."""
    return rng.choice(((16, 16), (12, 12), (12, 2), (32, 8), (40, 8), (56, 8), (40, 40), (16, 1), (10, 2)))


def _spread(rng, most, longest):
    """How many, the shortest and the longest."""
    n, hi = _log(rng, 1, most), _log(rng, 1, longest)
    return n, hi if n == 1 else max(1, int(hi * rng.uniform(0.02, 1.0))), hi


def draw(rng):
    kind = rng.choice(("rotary", "means", "select", "attend", "prefix", "prefix"))
    dim, dtype = rng.choice((64, 128, 128, 256)), rng.choice(("bf16", "bf16", "fp16"))
    heads, kv_heads = _heads(rng)
    page = rng.choice((16, 32, 64, 64, 128, 256))
    lse = rng.random() < 0.3
    while True:
        if kind == "rotary":
            part = dim if rng.random() < 0.5 else 16 * rng.randint(1, dim // 16)
            scaling = rng.choice(("none", "linear", "base", "parts"))
            case = _rotary("", _spread(rng, 128, 32768), rng.choice((0, _log(rng, 1, 1000000))), heads,
                           kv_heads, dim, part, rng.choice(("half", "interleaved")), dtype,
                           rng.random() < 0.5, scaling,
                           1.0 if scaling == "none" else rng.choice((2.0, 4.0, 7.5, 32.0)))
            fits = sum(_sizes(case)) * (heads + kv_heads) * dim <= MOST_ROTATED
        elif kind == "means":
            sizes = _spread(rng, 128, 65536)
            new = 1 if rng.random() < 0.5 else _log(rng, 1, sizes[2])
            case = _means("", sizes, new, kv_heads, dim, page)
            fits = work(case)["bytes"] <= 70e6
        elif kind == "prefix":
            tail = _log(rng, 8, 2000)
            case = _prefix("", _spread(rng, 16, 65536), _log(rng, 1, 128),
                           (rng.randint(8, tail), tail), heads, kv_heads,
                           rng.choice((1, 1, 1, 2, 3, 5)), dim, dtype, page, lse)
            fits = work(case)["flops"] <= MOST_PREFIX
        else:
            case = _cached(kind, "", _spread(rng, 128, 131072), _log(rng, FIRST + LAST, 200), heads,
                           kv_heads, rng.choice((1, 1, 1, 2, 4)), dim, dtype, page,
                           lse and kind == "attend")
            fits = work(case)["bytes"] <= 600e6
        if kind != "rotary" and fits:
            fits = sum(_tokens_held(case)) * kv_heads * dim <= MOST_CACHED * 1024
        if fits:
            case.pop("name")
            return case


# ------------------------------------------------------------------------- inputs ----

def _sizes(case):
    """The sequences' lengths: spread between the shortest and the longest, both present."""
    n = case["batch"] if "batch" in case else case["prefixes"]
    r = random.Random(n * 1000003 + case["longest"])
    lo, hi = case["shortest"], case["longest"]
    return [hi] + [lo] * (n > 1) + [_log(r, lo, hi) for _ in range(n - 2)]


def _counts(case):
    """Sequences that share each prefix."""
    r = random.Random(case["prefixes"] * 17 + case["each"])
    return [case["each"]] + [r.randint(1, case["each"]) for _ in range(case["prefixes"] - 1)]


def _tails(case):
    r = random.Random(case["each"] * 1000003 + case["long_tail"])
    return [max(case["tokens"], r.randint(case["short_tail"], case["long_tail"]))
            for _ in range(sum(_counts(case)))]


def _tokens_held(case):
    return _sizes(case) + (_tails(case) if case["kind"] == "prefix" else [])


def _starts(case):
    """The first new token of each sequence."""
    r = random.Random(case["batch"] + case["new"])
    return [max(0, n - (case["new"] if i == 0 else max(1, int(case["new"] * r.uniform(0.3, 1.0)))))
            for i, n in enumerate(_sizes(case))]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _exponent(amax):
    """The least e with amax <= 448 2^e."""
    mantissa, exponent = torch.frexp(amax)                  # amax = mantissa 2^exponent, in [1/2, 1)
    return (exponent - 9 + (mantissa > 0.875).to(exponent.dtype)).clamp_min(-100)


def _quantize(x):
    """E4M3 codes and E8M0 bytes of x [pages, heads, ...], one scale for each page and head."""
    e = _exponent(x.abs().amax((2, 3)))
    return torch.ldexp(x, -e[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8), \
        (e + 127).to(torch.uint8)


def _cache(g, pages, kv_heads, dim, page):
    """A filled cache; a page's keys have something in common, and a few channels are loud."""
    parts = ([], [], [], [])
    for lo in range(0, pages, 512):
        n = min(512, pages - lo)
        k = torch.randn(n, kv_heads, page, dim, generator=g, device=DEVICE)
        k += 0.7 * torch.randn(n, kv_heads, 1, dim, generator=g, device=DEVICE)
        k[..., :dim // 32] *= 4
        v = torch.randn(n, kv_heads, dim, page, generator=g, device=DEVICE)
        v *= torch.exp(0.5 * torch.randn(n, kv_heads, 1, 1, generator=g, device=DEVICE))
        for part, t in zip(parts, (*_quantize(k), *_quantize(v))):
            part.append(t)
    return [torch.cat(p) for p in parts]


def _tables(g, counts, spare=3):
    """int32 [batch, most pages] with the pages of every sequence in any order, and the pages
    that the pool has."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros(len(counts), max(counts), dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _handle(cache):
    from vdn_amd.kvcache import KVCache
    return KVCache(*cache, torch.zeros(1, dtype=torch.int32, device=DEVICE))


def _query(g, case, batch):
    return torch.randn(batch, case["tokens"], case["heads"], case["dim"], generator=g,
                       device=DEVICE).to(DTYPES[case["dtype"]])


def _prepare_rotary(case, g):
    dtype, heads, kv_heads, dim = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    sizes = _sizes(case)
    first = torch.randint(0, case["far"] + 1, (len(sizes),), generator=g, device=DEVICE).tolist()
    positions = torch.cat([torch.arange(f, f + n, dtype=torch.int32, device=DEVICE)
                           for f, n in zip(first, sizes)])
    # column slices of one fused projection's output
    qkv = torch.randn(sum(sizes), heads + 2 * kv_heads, dim, generator=g, device=DEVICE).to(dtype)
    state = dict(kind="rotary", case=case, q=qkv[:, :heads], k=qkv[:, heads:heads + kv_heads],
                 positions=positions, weights=(None, None))
    if case["norm"]:
        state["weights"] = tuple((1 + 0.1 * torch.randn(dim, generator=g, device=DEVICE)).to(dtype)
                                 for _ in range(2))
    if own:
        from vdn_amd.rotary import prepare_rotary_plan
        scaling = None if case["scaling"] == "none" else case["scaling"]
        state["plan"] = prepare_rotary_plan(
            dim, rotary_dim=case["part"], base=10000.0, layout=case["layout"], scaling=scaling,
            factor=case["factor"], original=8192 if scaling == "parts" else None, device=DEVICE)
    return state


def _prepare_prefix(case, g):
    page, prefixes, tails, counts = case["page"], _sizes(case), _tails(case), _counts(case)
    table, pages = _tables(g, [-(-n // page) for n in prefixes + tails])
    state = dict(kind="prefix", q=_query(g, case, len(tails)), prefixes=prefixes, tails=tails,
                 counts=counts, shared=table[:len(prefixes)].contiguous(),
                 table=table[len(prefixes):, :-(-max(tails) // page)].contiguous(),
                 cache=_cache(g, pages, case["kv_heads"], case["dim"], page), lse=case["lse"])
    if own:
        from vdn_amd.prefix import prepare_prefix_plan
        state.update(cache=_handle(state["cache"]), lengths=_ints(tails),
                     plan=prepare_prefix_plan(prefixes, counts, case["heads"], case["kv_heads"],
                                              case["dim"], tokens=case["tokens"], device=DEVICE))
    return state


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = case["kind"]
    if kind == "rotary":
        return _prepare_rotary(case, g)
    if kind == "prefix":
        return _prepare_prefix(case, g)
    page, kv_heads, dim, sizes = case["page"], case["kv_heads"], case["dim"], _sizes(case)
    table, pages = _tables(g, [-(-n // page) for n in sizes])
    cache = _cache(g, pages, kv_heads, dim, page)
    state = dict(kind=kind, cache=cache, table=table, sizes=sizes)
    if kind == "means":
        starts = _starts(case)
        state.update(starts=starts, means=torch.randn(pages, kv_heads, dim, generator=g,
                                                      device=DEVICE).to(torch.bfloat16))
        if own:
            state["starts"] = _ints(starts)
    else:
        state.update(q=_query(g, case, len(sizes)), count=case["count"], lse=case["lse"])
        if kind == "select":
            state["means"] = torch.cat([_mean(*(t[lo:lo + 256] for t in cache[:2]), page)
                                        for lo in range(0, pages, 256)])
        else:
            state.update(_random_selection(g, table, sizes, case))
    if own:
        state.update(cache=_handle(cache), lengths=_ints(sizes))
    return state


def _random_selection(g, table, sizes, case):
    """Pages of each query and K/V head: the first ones, the newest, and any between; in order."""
    tokens, kv_heads, page, count = case["tokens"], case["kv_heads"], case["page"], case["count"]
    pages = torch.full((len(sizes), tokens, kv_heads, count), -1, dtype=torch.int32, device=DEVICE)
    seen = []
    for b, n in enumerate(sizes):
        for i in range(tokens):
            sees = max(0, n - tokens + 1 + i)
            have = -(-sees // page)
            key = torch.rand(kv_heads, have, generator=g, device=DEVICE)
            key[:, :FIRST] = 2
            key[:, max(0, have - LAST):] = 2
            take = key.argsort(-1, descending=True)[:, :count].sort(-1)[0]
            pages[b, i, :, :take.shape[1]] = table[b][take]
            seen.append((min(have, count) - 1) * page + (sees - 1) % page + 1 if sees else 0)
    return dict(pages=pages, seen=seen, tokens=_ints(seen).view(len(sizes), tokens))


# --------------------------------------------------------------------- plain form ----

def _frequencies(case):
    """Angle of a step of one position for each pair of channels (float64), and the amplitude."""
    part, factor, base = case["part"], case["factor"], 10000.0
    if case["scaling"] == "base" and part > 2:
        base *= factor ** (part / (part - 2))
    f = base ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEVICE) / part)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] != "parts":
        return f, 1.0
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - PARTS[0]) / (PARTS[1] - PARTS[0])).clamp(0, 1)
    return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0


def _plain_rotary(state):
    case = state["case"]
    f, amplitude = _frequencies(case)
    angle = state["positions"].double()[:, None, None] * f
    cos, sin = (torch.cos(angle) * amplitude).float(), (torch.sin(angle) * amplitude).float()
    half = case["part"] // 2
    outs = []
    for x, w in zip((state["q"], state["k"]), state["weights"]):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        turned = y[..., :2 * half]
        if case["layout"] == "half":
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        outs.append(torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype))
    return tuple(outs)


def _values(codes, scales):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(),
                       scales.int()[:, :, None, None] - 127)


def _mean(codes, scales, n):
    """The mean of the first n keys of pages, [pages, kv_heads, dim]: the sum in 64 bits."""
    return (_values(codes, scales)[:, :, :n].double().sum(2) / n).to(torch.bfloat16)


def _plain_means(state):
    codes, scales = state["cache"][:2]
    means, page = state["means"], codes.shape[2]
    for i, (lo, n) in enumerate(zip(state["starts"], state["sizes"])):
        pages = state["table"][i, lo // page:-(-n // page)].long()
        full = pages if n % page == 0 else pages[:-1]
        for p in full.split(256):
            means[p] = _mean(codes[p], scales[p], page)
        if n % page:
            means[pages[-1:]] = _mean(codes[pages[-1:]], scales[pages[-1:]], n % page)
    return means


def _plain_select(state):
    q, means, count, page = state["q"], state["means"], state["count"], state["cache"][0].shape[2]
    batch, tokens, heads, dim = q.shape
    kv_heads = means.shape[1]
    pages = torch.full((batch, tokens, kv_heads, count), -1, dtype=torch.int32, device=q.device)
    seen = torch.zeros(batch, tokens, dtype=torch.int32, device=q.device)
    for b, n in enumerate(state["sizes"]):
        row = state["table"][b, :-(-n // page)]
        qq = q[b].double().view(tokens, kv_heads, heads // kv_heads, dim).transpose(0, 1)
        m = means[row.long()].double().permute(1, 2, 0)                         # [kv_heads, dim, pages]
        score = (qq.flatten(1, 2) @ m).view(kv_heads, tokens, -1, m.shape[2]).amax(2)
        for i in range(tokens):
            sees = n - tokens + 1 + i
            if sees <= 0:
                continue
            have = -(-sees // page)
            s = score[:, i, :have].clone()
            s[:, :FIRST] = math.inf
            s[:, max(0, have - LAST):] = math.inf
            best = s.sort(dim=-1, descending=True, stable=True)[1][:, :count].sort(-1)[0]
            pages[b, i, :, :best.shape[1]] = row[best]
            seen[b, i] = (best.shape[1] - 1) * page + (sees - 1) % page + 1
    return pages, seen


def _page_tokens(cache, pages, n):
    """The first n tokens of `pages` [kv_heads, pages] as K, V [kv_heads, n, dim] in 32 bits."""
    u = torch.arange(pages.shape[0], device=pages.device)[:, None]
    k = torch.ldexp(cache[0][pages, u].view(torch.float8_e4m3fn).float(),
                    cache[1][pages, u].int()[..., None, None] - 127)
    v = torch.ldexp(cache[2][pages, u].view(torch.float8_e4m3fn).float(),
                    cache[3][pages, u].int()[..., None, None] - 127)
    return k.flatten(1, 2)[:, :n], v.transpose(2, 3).flatten(1, 2)[:, :n]


def _softmax(s, v):
    """Weights of scores [heads, m, n], their product with v [heads, n, d], and the log-sum-exp."""
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    return p @ v / total.clamp_min(torch.finfo(s.dtype).tiny), (m + torch.log(total))[..., 0]


def _plain_attend(state):
    q, cache = state["q"], state["cache"]
    batch, tokens, heads, dim = q.shape
    kv_heads, page = cache[0].shape[1:3]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    for b in range(batch):
        for i in range(tokens):
            n = state["seen"][b * tokens + i]
            k, v = _page_tokens(cache, state["pages"][b, i, :, :-(-n // page)].long(), n)
            s = q[b, i].float().view(kv_heads, -1, dim) @ k.transpose(1, 2) * dim ** -0.5
            if n == 0:
                out[b, i], lse[b, i] = 0, -math.inf
                continue
            o, l = _softmax(s, v)
            out[b, i] = o.flatten(0, 1).to(q.dtype)
            lse[b, i] = l.flatten()
    return (out, lse) if state["lse"] else out


def _plain_prefix(state):
    q, cache, counts = state["q"], state["cache"], state["counts"]
    batch, tokens, heads, dim = q.shape
    kv_heads, page = cache[0].shape[1:3]
    group = heads // kv_heads
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    first = 0
    for p, (n, count) in enumerate(zip(state["prefixes"], counts)):
        k, v = _page_tokens(cache, state["shared"][p, :-(-n // page)].long().expand(kv_heads, -1), n)
        for b in range(first, first + count):
            m = state["tails"][b]
            pages = state["table"][b, :-(-m // page)].long().expand(kv_heads, -1)
            kt, vt = _page_tokens(cache, pages, m)
            qq = q[b].float().view(tokens, kv_heads, group, dim).transpose(0, 1).flatten(1, 2) * dim ** -0.5
            tail = (qq @ kt.transpose(1, 2)).view(kv_heads, tokens, group, m)
            sees = torch.arange(m - tokens + 1, m + 1, device=q.device)[:, None, None]
            tail = tail.masked_fill(torch.arange(m, device=q.device) >= sees, -math.inf)
            o, l = _softmax(torch.cat((qq @ k.transpose(1, 2), tail.flatten(1, 2)), 2),
                            torch.cat((v, vt), 1))
            out[b] = o.view(kv_heads, tokens, group, dim).transpose(0, 1).flatten(1, 2).to(q.dtype)
            lse[b] = l.view(kv_heads, tokens, group).transpose(0, 1).flatten(1, 2)
        first += count
    return (out, lse) if state["lse"] else out


# ------------------------------------------------------------------------ one pass ----

@torch.no_grad()
def run(state):
    kind = state["kind"]
    if not own:
        return {"rotary": _plain_rotary, "means": _plain_means, "select": _plain_select,
                "attend": _plain_attend, "prefix": _plain_prefix}[kind](state)
    if kind == "rotary":
        from vdn_amd.rotary import rotate_qk
        return rotate_qk(state["q"], state["k"], state["positions"], state["plan"], *state["weights"],
                         eps=EPS)
    if kind == "prefix":
        from vdn_amd.prefix import prefix_attention
        return prefix_attention(state["q"], state["cache"], state["shared"], state["plan"],
                                state["table"], state["lengths"], return_lse=state["lse"])
    from vdn_amd.sparse import select_pages, selected_attention, write_means
    if kind == "means":
        write_means(state["cache"], state["means"], state["table"], state["starts"], state["lengths"])
        return state["means"]
    if kind == "select":
        return select_pages(state["q"], state["cache"], state["means"], state["table"],
                            state["lengths"], state["count"], first=FIRST, last=LAST)
    return selected_attention(state["q"], state["cache"], state["pages"], state["tokens"],
                              return_lse=state["lse"])


def work(case):
    """What a pass has to read and write (each input and output once) and to compute."""
    kind, dim, kv_heads = case["kind"], case["dim"], case["kv_heads"]
    if kind == "rotary":
        tokens = sum(_sizes(case))
        rows = tokens * (case["heads"] + kv_heads)
        return {"bytes": rows * dim * 4 + tokens * 4,
                "flops": rows * (3.0 * case["part"] + 4.0 * dim * case["norm"])}
    page, sizes = case["page"], _sizes(case)
    if kind == "means":
        spans = [(n - lo // page * page, -(-n // page) - lo // page) for lo, n in zip(_starts(case), sizes)]
        keys, pages = sum(s[0] for s in spans), sum(s[1] for s in spans)
        return {"bytes": kv_heads * (keys * dim + pages * (2 * dim + 1)), "flops": 1.0 * kv_heads * keys * dim}
    tokens, heads = case["tokens"], case["heads"]
    if kind == "prefix":
        pairs = sum(n * c for n, c in zip(sizes, _counts(case))) + sum(_tails(case))
        rows = sum(_counts(case)) * tokens * heads
        return {"bytes": 2 * kv_heads * dim * (sum(sizes) + sum(_tails(case)))
                + rows * (4 * dim + 4 * case["lse"]),
                "flops": 4.0 * dim * heads * tokens * pairs}
    rows = len(sizes) * tokens * heads
    if kind == "select":
        pages = sum(-(-n // page) for n in sizes)
        return {"bytes": pages * (kv_heads * dim * 2 + 4) + rows * dim * 2
                + len(sizes) * tokens * (kv_heads * case["count"] + 1) * 4,
                "flops": 2.0 * dim * heads * tokens * pages}
    seen = sum(min(n, case["count"] * page) for n in sizes) * tokens
    return {"bytes": 2 * kv_heads * dim * seen + rows * (4 * dim + 4 * case["lse"]),
            "flops": 4.0 * dim * heads * seen}


# ---------------------------------------------------------------------- definition ----

def _double(codes, scales):
    """Codes of [..., a, b] pages as float64: sign, four exponent bits, three mantissa bits."""
    c = codes.long()
    exponent, mantissa = (c >> 3) & 15, (c & 7).double()
    value = torch.where(exponent > 0, (8 + mantissa) * torch.exp2(exponent.double() - 10),
                        mantissa * 2.0 ** -9)
    return torch.where(c > 127, -value, value) * torch.exp2(scales.double() - 127)[..., None, None]


def _exact_rotary(case, state):
    part, dim = case["part"], case["dim"]
    base = 10000.0
    if case["scaling"] == "base" and part > 2:
        base = base * case["factor"] ** (part / (part - 2))
    steps, amplitude = [], 1.0
    for j in range(part // 2):
        f = math.pow(base, -2 * j / part)
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "parts":
            keep = min(1.0, max(0.0, (8192 * f / math.tau - PARTS[0]) / (PARTS[1] - PARTS[0])))
            f = f * keep + f / case["factor"] * (1 - keep)
            amplitude = 1.0 + 0.1 * math.log(case["factor"])
        steps.append(f)
    f = torch.tensor(steps, dtype=torch.float64, device=DEVICE)
    turn = torch.polar(torch.full_like(f, amplitude).expand(len(state["positions"]), -1).contiguous(),
                       state["positions"].double()[:, None] * f)[:, None]
    j = torch.arange(part // 2, device=DEVICE)
    re, im = (j, j + part // 2) if case["layout"] == "half" else (2 * j, 2 * j + 1)
    outs = []
    for x, w in ((state["q"], state["weights"][0]), (state["k"], state["weights"][1])):
        y = x.double().clone()
        if w is not None:
            y *= w.double() / (y.square().sum(-1, keepdim=True) / dim + EPS).sqrt()
        z = torch.complex(y[..., re], y[..., im]) * turn
        y[..., re], y[..., im] = z.real, z.imag
        outs.append(y)
    return tuple(outs)


def _exact_means(case, state):
    means, page = state["means"].double(), case["page"]
    k, ks = state["cache"][:2]
    for i, (lo, n) in enumerate(zip(state["starts"], state["sizes"])):
        for at in range(lo // page, -(-n // page)):
            p = int(state["table"][i, at])
            means[p] = _double(k[p], ks[p])[:, :min(page, n - at * page)].mean(1)
    return means


def _exact_select(case, state):
    count, page, tokens = case["count"], case["page"], case["tokens"]
    q, means, kv_heads = state["q"].double(), state["means"].double(), case["kv_heads"]
    group = case["heads"] // kv_heads
    pages = torch.full((len(state["sizes"]), tokens, kv_heads, count), -1, dtype=torch.int32, device=DEVICE)
    seen = torch.zeros(len(state["sizes"]), tokens, dtype=torch.int32, device=DEVICE)
    for b, n in enumerate(state["sizes"]):
        for i in range(tokens):
            have = max(0, -(-(n - tokens + 1 + i) // page))
            ids = state["table"][b, :have].tolist()
            m = means[state["table"][b, :have].long()]                            # [pages, kv_heads, dim]
            for u in range(kv_heads):
                s = torch.matmul(m[:, u], q[b, i, u * group:(u + 1) * group].T).max(1)[0].tolist() \
                    if have else []
                order = sorted(range(have), key=lambda j: (not (j < FIRST or j >= have - LAST), -s[j], j))
                got = [ids[j] for j in sorted(order[:count])]
                pages[b, i, u, :len(got)] = _ints(got)
            if have:
                seen[b, i] = n - tokens + 1 + i - page * (have - min(have, count))
    return pages, seen


def _exact_rows(q, k, v, sees):
    """One head in float64: q [m, d] over the first sees[i] of k, v [n, d]."""
    s = (q @ k.T) / math.sqrt(q.shape[1])
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= sees[:, None]
    s[hidden] = -math.inf
    l = torch.logsumexp(s, 1)
    w = torch.where(hidden, 0.0, torch.exp(s - l[:, None]))
    return w @ v, l


def _exact_attention(case, state):
    """attend and prefix: for each sequence and K/V head the keys in a row, in float64."""
    q, c, page, kv_heads, tokens = state["q"], state["cache"], case["page"], case["kv_heads"], case["tokens"]
    group = case["heads"] // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)

    def keys(ids, u, n):
        p = ids[:-(-n // page)].long()
        return _double(c[0][p, u], c[1][p, u]).flatten(0, 1)[:n], \
            _double(c[2][p, u], c[3][p, u]).transpose(1, 2).flatten(0, 1)[:n]

    def put(b, i, u, k, v, sees):
        hs = slice(u * group, (u + 1) * group)
        rows = q[b, i, hs].double().flatten(0, -2)
        o, l = _exact_rows(rows, k, v, sees)
        out[b, i, hs], lse[b, i, hs] = o.view(out[b, i, hs].shape), l.view(lse[b, i, hs].shape)

    if case["kind"] == "attend":
        for b in range(q.shape[0]):
            for i in range(tokens):
                n = state["seen"][b * tokens + i]
                for u in range(kv_heads if n else 0):
                    put(b, i, u, *keys(state["pages"][b, i, u], u, n),
                        torch.full((group,), n, device=q.device))
    else:
        owner = [p for p, n in enumerate(state["counts"]) for _ in range(n)]
        last, shared = None, None
        for u in range(kv_heads):
            for b, p in enumerate(owner):
                n, m = state["prefixes"][p], state["tails"][b]
                if last != (u, p):
                    last, shared = (u, p), keys(state["shared"][p], u, n)
                k, v = (torch.cat(t) for t in zip(shared, keys(state["table"][b], u, m)))
                sees = torch.arange(n + m - tokens + 1, n + m + 1, device=q.device).repeat_interleave(group)
                put(b, slice(None), u, k, v, sees)
    return (out, lse) if case["lse"] else out


@torch.no_grad()
def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(case, state)
    if kind == "means":
        pages = sum(-(-n // case["page"]) - lo // case["page"]
                    for lo, n in zip(state["starts"], state["sizes"]))
        return _exact_means(case, state) if pages <= 10000 else None     # walked one by one
    if len(state["q"]) * case["tokens"] * case["kv_heads"] > 6000:        # too many rows for the same
        return None
    return _exact_select(case, state) if kind == "select" else _exact_attention(case, state)
