"""Workloads of causal attention over packed prompts and of the 8-bit key/value cache.

A case is a plain dict; its "kind" names the operator that a pass goes through:

  prompt   causal_attention: whole prompts, packed, grouped heads
  write    write_cache, then read_cache of every token in the pages that the write touched
  attend   cache_attention: the newest token (or few) of each sequence over its cached tokens

`own` selects how run() computes them: the framework's entry points, or plain torch in 32 bits.

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
LEAST_EXPONENT = -100
MOST_PROMPT = 8.8e12     # operations of the largest listed prompt
MOST_TOKENS = 65536      # tokens of the largest listed write
MOST_CACHED = 524288     # cached tokens x kv heads / 8 of the largest listed cache


def _prompt(name, lengths, heads, kv_heads, dim=128, dtype="bf16", lse=False):
    return dict(name=name, kind="prompt", batch=lengths[0], shortest=lengths[1], longest=lengths[2],
                heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, lse=lse)


def _write(name, batch, held, new, kv_heads, dim=128, dtype="bf16", page=64):
    """`held` and `new`: the most tokens that a sequence has in the cache, and brings."""
    return dict(name=name, kind="write", batch=batch, held=held, new=new, kv_heads=kv_heads,
                dim=dim, dtype=dtype, page=page)


def _attend(name, lengths, heads, kv_heads, tokens=1, dim=128, dtype="bf16", page=64, lse=False):
    return dict(name=name, kind="attend", batch=lengths[0], shortest=lengths[1], longest=lengths[2],
                heads=heads, kv_heads=kv_heads, tokens=tokens, dim=dim, dtype=dtype, page=page,
                lse=lse)


def listed():
    return [
        # one long document, four query heads to a key head
        _prompt("prompt_long", (1, 32768, 32768), 32, 8),
        # a batch of ragged prompts, as a text encoder packs them in front of the block; 7 to 1
        _prompt("prompt_batch", (24, 77, 1200), 56, 8),
        # one caption: launch latency and a grid that cannot fill the card
        _prompt("prompt_caption", (1, 77, 77), 12, 2, dim=64, dtype="fp16"),
        # many short prompts with as many key heads as query heads, half precision
        _prompt("prompt_half", (64, 1, 400), 16, 16, dim=64, dtype="fp16"),
        # wide heads that share a single key head, an odd length, log-sum-exp for a later merge
        _prompt("prompt_wide", (1, 4097, 4097), 16, 1, dim=256, lse=True),
        # whole prompts go into the cache
        _write("write_prompts", 8, 0, 8192, 8),
        # a decode step: one token for each of 64 sequences into partly filled pages
        _write("write_step", 64, 8192, 1, 8),
        # pieces of prompts behind what is held, small pages, half precision
        _write("write_pieces", 16, 500, 300, 12, dim=64, dtype="fp16", page=16),
        # a decode step over ragged sequences
        _attend("attend_step", (64, 512, 8192), 40, 8),
        # one sequence with a long past: the work has to be split along it
        _attend("attend_long", (1, 131072, 131072), 56, 8, page=128),
        # the smallest step: one short sequence
        _attend("attend_caption", (1, 78, 78), 12, 2, dim=64),
        # four drafted tokens to be checked at once, small pages, log-sum-exp
        _attend("attend_draft", (16, 100, 4097), 12, 12, tokens=4, dim=64, dtype="fp16", page=16,
                lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Query and key heads: one to one, grouped (odd groups too), one for all."""
    return rng.choice(((16, 16), (12, 12), (12, 2), (32, 8), (40, 8), (56, 8), (40, 40), (16, 1), (10, 2)))


def _lengths(rng, most_batch, longest):
    batch = _log(rng, 1, most_batch)
    hi = _log(rng, 1, longest)
    return batch, hi if batch == 1 else max(1, int(hi * rng.uniform(0.02, 1.0))), hi


def draw(rng):
    kind = rng.choice(("prompt", "write", "attend"))
    dim, dtype = rng.choice((64, 128, 128, 256)), rng.choice(("bf16", "bf16", "fp16"))
    heads, kv_heads = _heads(rng)
    page = rng.choice((16, 32, 64, 64, 128, 256))
    while True:
        if kind == "prompt":
            case = _prompt("", _lengths(rng, 64, 32768), heads, kv_heads, dim, dtype,
                           rng.random() < 0.3)
            fits = work(case)["flops"] <= MOST_PROMPT
        elif kind == "write":
            new = 1 if rng.random() < 0.4 else _log(rng, 2, 32768)
            case = _write("", _log(rng, 1, 128), rng.choice((0, _log(rng, 1, 8192))), new,
                          kv_heads, dim, dtype, page)
            fits = case["batch"] * new * kv_heads * dim <= MOST_TOKENS * 1024 \
                and case["batch"] * case["held"] * kv_heads * dim <= MOST_CACHED * 1024
        else:
            tokens = rng.choice((1, 1, 1, 2, 3, 5, 8))
            case = _attend("", _lengths(rng, 128, 131072), heads, kv_heads, tokens, dim, dtype,
                           page, rng.random() < 0.3)
            fits = case["batch"] * case["longest"] * kv_heads * dim <= MOST_CACHED * 1024
        if fits:
            case.pop("name")
            return case


# ------------------------------------------------------------------------- inputs ----

def _sizes(case):
    """The sequences' lengths: spread between the shortest and the longest, both present."""
    r = random.Random(case["batch"] * 1000003 + case["longest"])
    lo, hi = case["shortest"], case["longest"]
    return [hi] + [lo] * (case["batch"] > 1) + \
        [_log(r, lo, hi) for _ in range(case["batch"] - 2)]


def _write_sizes(case):
    """Tokens that each sequence holds and brings."""
    r = random.Random(case["batch"] * 1000003 + case["new"] * 17 + case["held"])
    held = [r.randint(case["held"] // 4, case["held"]) for _ in range(case["batch"])]
    new = [case["new"]] + [max(1, int(case["new"] * r.uniform(0.1, 1.0)))
                           for _ in range(case["batch"] - 1)]
    return held, new


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _offsets(sizes):
    return _ints([0] + torch.tensor(sizes).cumsum(0).tolist())


def _projection(g, rows, heads, kv_heads, dim, dtype):
    """Q, K, V as column slices of one fused projection's output; keys carry a few loud channels."""
    qkv = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g, device=DEVICE)
    qkv[:, heads:heads + kv_heads, :dim // 32] *= 4
    qkv = qkv.to(dtype)
    return qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]


def _quantize(x, dims):
    """E4M3 codes and E8M0 bytes of x, one scale over `dims`."""
    amax = x.abs().amax(dims, keepdim=True)
    e = _exponent(amax)
    return torch.ldexp(x, -e).to(torch.float8_e4m3fn).view(torch.uint8), \
        (e + 127).to(torch.uint8).squeeze(dims[1]).squeeze(dims[0])


def _exponent(amax):
    """The least e with amax <= 448 2^e, from LEAST_EXPONENT on."""
    mantissa, exponent = torch.frexp(amax)                  # amax = mantissa 2^exponent, in [1/2, 1)
    e = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    return torch.where(amax > 0, e, LEAST_EXPONENT).clamp_min(LEAST_EXPONENT)


def _cache(g, pages, kv_heads, dim, page):
    """A filled cache: every page holds tokens of an earlier request or of these sequences."""
    parts = ([], [], [], [])
    for lo in range(0, pages, 512):
        n = min(512, pages - lo)
        k = torch.randn(n, kv_heads, page, dim, generator=g, device=DEVICE)
        k[..., :dim // 32] *= 4
        v = torch.randn(n, kv_heads, dim, page, generator=g, device=DEVICE)
        v *= torch.exp(0.5 * torch.randn(n, kv_heads, 1, 1, generator=g, device=DEVICE))
        for part, t in zip(parts, (*_quantize(k, (2, 3)), *_quantize(v, (2, 3)))):
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


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dtype, dim = case["kind"], DTYPES[case["dtype"]], case["dim"]
    kv_heads = case["kv_heads"]
    if kind == "prompt":
        sizes = _sizes(case)
        q, k, v = _projection(g, sum(sizes), case["heads"], kv_heads, dim, dtype)
        state = dict(kind=kind, q=q, k=k, v=v, sizes=sizes, lse=case["lse"])
        if own:
            from vdn_amd.causal import prepare_causal_plan
            state["plan"] = prepare_causal_plan(sizes, case["heads"], kv_heads, device=DEVICE)
        return state
    page = case["page"]
    if kind == "write":
        held, new = _write_sizes(case)
        table, pages = _tables(g, [-(-(h + n) // page) for h, n in zip(held, new)])
        cache = _cache(g, pages, kv_heads, dim, page)
        _, k, v = _projection(g, sum(new), 0, kv_heads, dim, dtype)
        # what is read back: each touched page from its first token
        first = [h // page * page for h in held]
        back = [h + n - f for h, n, f in zip(held, new, first)]
        state = dict(kind=kind, cache=cache, table=table, k=k, v=v, held=held, new=new, first=first,
                     back=back)
        if own:
            state.update(cache=_handle(cache), starts=_ints(held), offsets=_offsets(new),
                         firsts=_ints(first), back_offsets=_offsets(back), rows=sum(back))
        return state
    sizes = _sizes(case)
    table, pages = _tables(g, [-(-n // page) for n in sizes])
    cache = _cache(g, pages, kv_heads, dim, page)
    q = torch.randn(case["batch"], case["tokens"], case["heads"], dim, generator=g,
                    device=DEVICE).to(dtype)
    state = dict(kind=kind, cache=cache, table=table, q=q, sizes=sizes, lse=case["lse"])
    if own:
        state.update(cache=_handle(cache), lengths=_ints(sizes))
    return state


# --------------------------------------------------------------------- plain form ----

def _softmax(q, k, v, first, scale):
    """q [heads, m, d] over k, v [heads, n, d] in 32 bits; query i sees the keys up to first + i.
    Output and log-sum-exp; a row that sees nothing gives zeros and -inf."""
    s = q @ k.transpose(1, 2) * scale
    i = torch.arange(q.shape[1], device=q.device)[:, None] + first
    s = s.masked_fill(torch.arange(k.shape[1], device=q.device) > i, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    return p @ v / total.clamp_min(torch.finfo(s.dtype).tiny), (m + torch.log(total))[..., 0]


def _plain_prompt(state):
    q, k, v = state["q"], state["k"], state["v"]
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    start = 0
    for n in state["sizes"]:
        rows = slice(start, start + n)
        kt = k[rows].float().transpose(0, 1)
        vt = v[rows].float().transpose(0, 1)
        heads = max(1, min(k.shape[1], (1 << 29) // (n * min(n, 4096) * group)))
        for h in range(0, k.shape[1], heads):
            kk = kt[h:h + heads].repeat_interleave(group, 0)
            vv = vt[h:h + heads].repeat_interleave(group, 0)
            hs = slice(h * group, (h + heads) * group)
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                qq = q[start + a:start + b, hs].float().transpose(0, 1)
                o, l = _softmax(qq, kk[:, :b], vv[:, :b], a, scale)
                out[start + a:start + b, hs] = o.transpose(0, 1).to(q.dtype)
                lse[start + a:start + b, hs] = l.transpose(0, 1)
        start += n
    return (out, lse) if state["lse"] else out


def _values(codes, scales):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(),
                       scales.int()[:, :, None, None] - 127)


def _tokens(cache, pages, n):
    """The first n tokens of `pages` as K, V [heads, n, dim] in 32 bits."""
    k = _values(cache[0][pages], cache[1][pages]).permute(1, 0, 2, 3)
    v = _values(cache[2][pages], cache[3][pages]).permute(1, 0, 3, 2)
    return k.flatten(1, 2)[:, :n], v.flatten(1, 2)[:, :n]


def _append(codes, scales, pages, x, begin):
    """x [tokens, heads, dim] into `pages` (codes [.., page, dim]) from position `begin` of the
    first one; a page's scale only grows, and what it holds is rounded anew when it does."""
    page, x = codes.shape[2], x.float().transpose(0, 1)
    total = begin + x.shape[1]
    full = torch.zeros(x.shape[0], len(pages) * page, x.shape[2], device=x.device)
    full[:, begin:total] = x
    full = full.view(x.shape[0], len(pages), page, -1).transpose(0, 1)
    e = _exponent(full.abs().amax((2, 3)))
    fresh = torch.ldexp(full, -e[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if begin:
        held = scales[pages[:1]].int() - 127
        e[:1] = torch.maximum(e[:1], held)
        fresh[:1] = torch.ldexp(full[:1], -e[:1, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        old = torch.ldexp(codes[pages[:1]].view(torch.float8_e4m3fn).float(),
                          (held - e[:1])[:, :, None, None])
        fresh[:1, :, :begin] = old.to(torch.float8_e4m3fn).view(torch.uint8)[:, :, :begin]
    keep = codes[pages[-1:], :, (total - 1) % page + 1:]
    codes[pages] = fresh
    codes[pages[-1:], :, (total - 1) % page + 1:] = keep
    scales[pages] = (e + 127).to(torch.uint8)


def _plain_write(state):
    cache, dtype = state["cache"], state["k"].dtype
    page, at, out_k, out_v = cache[0].shape[2], 0, [], []
    for i, (held, new) in enumerate(zip(state["held"], state["new"])):
        pages = state["table"][i, held // page:-(-(held + new) // page)].long()
        _append(cache[0], cache[1], pages, state["k"][at:at + new], held % page)
        _append(cache[2].transpose(2, 3), cache[3], pages, state["v"][at:at + new], held % page)
        k, v = _tokens(cache, pages, state["back"][i])
        out_k.append(k.transpose(0, 1).to(dtype))
        out_v.append(v.transpose(0, 1).to(dtype))
        at += new
    return torch.cat(out_k), torch.cat(out_v)


def _plain_attend(state):
    q, cache = state["q"], state["cache"]
    batch, tokens, heads, dim = q.shape
    kv_heads, page = cache[0].shape[1:3]
    group = heads // kv_heads
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    for i, n in enumerate(state["sizes"]):
        k, v = _tokens(cache, state["table"][i, :-(-n // page)].long(), n)
        qq = q[i].float().transpose(0, 1)
        o, l = _softmax(qq, k.repeat_interleave(group, 0), v.repeat_interleave(group, 0), n - tokens,
                        dim ** -0.5)
        out[i] = o.transpose(0, 1).to(q.dtype)
        lse[i] = l.transpose(0, 1)
    return (out, lse) if state["lse"] else out


# ------------------------------------------------------------------------ one pass ----

@torch.no_grad()
def run(state):
    kind = state["kind"]
    if not own:
        return {"prompt": _plain_prompt, "write": _plain_write, "attend": _plain_attend}[kind](state)
    if kind == "prompt":
        from vdn_amd.causal import causal_attention
        return causal_attention(state["q"], state["k"], state["v"], state["plan"],
                                return_lse=state["lse"])
    from vdn_amd.kvcache import cache_attention, read_cache, write_cache
    if kind == "write":
        write_cache(state["cache"], state["k"], state["v"], state["table"], state["starts"],
                    state["offsets"])
        return read_cache(state["cache"], state["table"], state["firsts"], state["back_offsets"],
                          state["rows"], dtype=state["k"].dtype)
    return cache_attention(state["q"], state["cache"], state["table"], state["lengths"],
                           return_lse=state["lse"])


def work(case):
    """What a pass has to read and write (each input and output once) and to compute."""
    dim, kv_heads = case["dim"], case["kv_heads"]
    if case["kind"] == "prompt":
        sizes, heads = _sizes(case), case["heads"]
        rows = sum(sizes)
        return {"bytes": rows * (4 * (heads + kv_heads) * dim + 4 * heads * case["lse"]),
                "flops": 4.0 * dim * heads * sum(n * (n + 1) // 2 for n in sizes)}
    if case["kind"] == "write":
        held, new = _write_sizes(case)
        old = sum(h % case["page"] for h in held)
        row = 2 * kv_heads * dim          # K and V values of a token
        # new rows in, codes of the new rows out; the held part of the pages in; all of it read back
        return {"bytes": row * (3 * sum(new) + old + 2 * (sum(new) + old)),
                "flops": 4.0 * row * sum(new)}
    sizes = _sizes(case)
    rows = case["batch"] * case["tokens"] * case["heads"]
    return {"bytes": 2 * kv_heads * dim * sum(sizes) + rows * (4 * dim + 4 * case["lse"]),
            "flops": 4.0 * dim * case["heads"] * case["tokens"] * sum(sizes)}


# ---------------------------------------------------------------------- definition ----

def _double(codes, scales):
    """Codes of [heads, ...] pages as float64: sign, four exponent bits, three mantissa bits."""
    c = codes.long()
    exponent, mantissa = (c >> 3) & 15, (c & 7).double()
    value = torch.where(exponent > 0, (8 + mantissa) * torch.exp2(exponent.double() - 10),
                        mantissa * 2.0 ** -9)
    value = torch.where(c > 127, -value, value)
    return value * torch.exp2(scales.double() - 127)[..., None, None]


def _nearest(x):
    """float64 -> the nearest E4M3 value, ties to the even mantissa."""
    _, exponent = torch.frexp(x.abs())
    step = torch.exp2((exponent - 1).clamp_min(-6).double() - 3)
    return torch.where(x == 0, x, torch.round(x / step) * step)


def _exact_write(state):
    codes = state["cache"]
    page = codes[0].shape[2]
    sides = []
    for side, x in ((0, state["k"]), (2, state["v"])):
        rows, at = [], 0
        for i, (held, new) in enumerate(zip(state["held"], state["new"])):
            news, done = x[at:at + new].double(), 0
            at += new
            place = held
            while done < new:
                inside = place % page
                n = min(page - inside, new - done)
                part = news[done:done + n]                                       # [n, heads, dim]
                top = part.abs().amax((0, 2))
                e = torch.ceil(torch.log2(top / 448).clamp_min(LEAST_EXPONENT))
                if inside:
                    p = state["table"][i, place // page].long()
                    c = codes[side][p].transpose(1, 2) if side else codes[side][p]
                    byte = codes[side + 1][p]
                    e = torch.maximum(e, byte.double() - 127)
                    scale = torch.exp2(e)[:, None, None]
                    old = _nearest(_double(c, byte)[:, :inside] / scale) * scale
                    rows.append(old.transpose(0, 1))
                scale = torch.exp2(e)[None, :, None]
                rows.append(_nearest(part / scale) * scale)
                done, place = done + n, place + n
        sides.append(torch.cat(rows))
    return tuple(sides)


def _exact_attention(q, k, v, first):
    """One head group in float64: q [m, d] over k, v [n, d]."""
    out, lse = [], []
    for a in range(0, q.shape[0], 4096):
        s = (q[a:a + 4096] @ k.T) / math.sqrt(q.shape[1])
        seen = torch.arange(k.shape[0], device=q.device)[None] <= \
            torch.arange(a, a + s.shape[0], device=q.device)[:, None] + first
        s[~seen] = -math.inf
        l = torch.logsumexp(s, 1)
        w = torch.where(seen, torch.exp(s - l[:, None]), 0.0)
        out.append(w @ v)
        lse.append(l)
    return torch.cat(out), torch.cat(lse)


@torch.no_grad()
def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "write":
        if sum(state["new"]) / case["page"] > 20000:       # too many pages to walk one by one
            return None
        return _exact_write(state)
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    q = state["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float64, device=q.device)
    if case["batch"] * heads > 4000:
        return None
    start = 0
    for i, n in enumerate(state["sizes"]):
        if case["kind"] == "prompt":
            rows = slice(start, start + n)
            for h in range(heads):
                out[rows, h], lse[rows, h] = _exact_attention(
                    q[rows, h].double(), state["k"][rows, h // group].double(),
                    state["v"][rows, h // group].double(), 0)
            start += n
            continue
        p = state["table"][i, :-(-n // case["page"])].long()
        c = state["cache"]
        for u in range(case["kv_heads"]):
            k = _double(c[0][p, u], c[1][p, u]).flatten(0, 1)[:n]
            v = _double(c[2][p, u], c[3][p, u]).transpose(1, 2).flatten(0, 1)[:n]
            for h in range(u * group, (u + 1) * group):
                out[i, :, h], lse[i, :, h] = _exact_attention(q[i, :, h].double(), k, v,
                                                             n - case["tokens"])
    return (out, lse) if case["lse"] else out
