"""The operators of the 8-bit paged cache, each in its plain form and through the package.

`plan` builds block tables and slot maps from request lengths, `append` norms, rotates and stores
a step's keys and values, `attention` reads them. The plain forms are elementary torch operations
in 32 bits (64 for whole numbers); `exact` computes the same from the definitions in 64 bits.
"""

import math
import random

import torch

own = False

FLOOR = -60  # the smallest exponent a block's scale has
LARGEST = 448.0 * 2.0**40  # magnitudes above it are stored as NaN
EPS = 1e-6


# ------------------------------------------------------------------------------------- cases
def listed():
    llm = {"heads_q": 32, "heads_kv": 8, "dim": 128, "page": 64, "theta": 500000.0}
    dit = {"heads_q": 24, "heads_kv": 24, "dim": 128, "page": 16, "theta": 10000.0}
    small = {"heads_q": 12, "heads_kv": 12, "dim": 64, "page": 16, "theta": 10000.0}
    return [
        # one decode step of four chats: nothing but latency
        {"name": "plan 4 chats", "do": "plan", "page": 64, "requests": 4, "cached": 2000,
         "new": 1, "spread": "uniform", "finished": 0, "mix": 1},
        # a busy server's step: a thousand requests, prompt chunks among single tokens, some done
        {"name": "plan 1000 requests", "do": "plan", "page": 16, "requests": 1000, "cached": 8192,
         "new": 4096, "spread": "uniform", "finished": 40, "mix": 2},
        # one new token of one chat
        {"name": "append 1 token", "do": "append", **llm, "requests": 1, "cached": 4099, "new": 1,
         "spread": "same", "norm": False, "interleaved": False, "mix": 3},
        # a decode step of 256 chats, queries and keys normed
        {"name": "append 256 tokens", "do": "append", **llm, "requests": 256, "cached": 2000,
         "new": 1, "spread": "uniform", "norm": True, "interleaved": False, "mix": 4},
        # a prompt's chunk
        {"name": "append prompt", "do": "append", **llm, "requests": 1, "cached": 1000,
         "new": 8192, "spread": "same", "norm": False, "interleaved": False, "mix": 5},
        # ragged chunks of a model with heads of 64, interleaved rotation
        {"name": "append ragged d64", "do": "append", **small, "requests": 13, "cached": 777,
         "new": 611, "spread": "each", "norm": True, "interleaved": True, "mix": 6},
        # one new token of a short chat: latency
        {"name": "attend 1 token short", "do": "attention", **llm, "requests": 1, "cached": 499,
         "new": 1, "spread": "same", "mix": 7},
        # one new token after a prompt of 131071
        {"name": "attend 1 token long", "do": "attention", **llm, "requests": 1,
         "cached": 131071, "new": 1, "spread": "same", "mix": 8},
        # a decode step of 64 chats
        {"name": "attend 64 tokens", "do": "attention", **llm, "requests": 64, "cached": 16384,
         "new": 1, "spread": "uniform", "mix": 9},
        # drafts of five tokens checked for 16 chats
        {"name": "attend drafts", "do": "attention", **llm, "requests": 16, "cached": 8000,
         "new": 5, "spread": "uniform", "mix": 10},
        # the last chunk of a prompt of 131071
        {"name": "attend last chunk", "do": "attention", **llm, "requests": 1, "cached": 130047,
         "new": 1024, "spread": "same", "mix": 11},
        # a chunk among single tokens, a key head for each query head, small pages
        {"name": "attend mixed mha", "do": "attention", **dit, "requests": 11, "cached": 3001,
         "new": 1500, "spread": "uniform", "mix": 12},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        do = rng.choice(["plan", "append", "append", "attention", "attention", "attention"])
        c = {"do": do, "page": rng.choice([16, 32, 64, 128]), "mix": rng.randrange(1 << 20),
             "spread": rng.choice(["same", "uniform", "each"])}
        if do == "plan":
            c |= {"requests": _log(rng, 1, 2000), "cached": _log(rng, 1, 20000),
                  "new": _log(rng, 1, 6000), "finished": rng.randrange(0, 30)}
            c["finished"] = min(c["finished"], c["requests"] - 1)
            if c["requests"] * c["new"] > 200000:  # more tokens than a step takes
                c["spread"] = "uniform"
        else:
            kv = rng.choice([1, 2, 3, 4, 8, 12])
            c |= {"heads_kv": kv, "heads_q": kv * rng.choice([1, 1, 2, 3, 4, 5, 8]),
                  "dim": rng.choice([64, 128, 128]), "theta": rng.choice([10000.0, 500000.0])}
            c |= {"requests": _log(rng, 1, 200), "cached": _log(rng, 1, 60000),
                  "new": rng.choice([1, 1, rng.randint(2, 12), _log(rng, 1, 1500)])}
            if do == "append":
                c |= {"norm": rng.random() < 0.5, "interleaved": rng.random() < 0.5}
        if _cost(c) <= most and _plain_bytes(c) < 40e9:
            return c


def _lengths(case):
    """(tokens cached, new tokens; -1 where a request is done) of each request."""
    r, n = random.Random(case["mix"]), case["requests"]
    cached = [case["cached"]] * n
    new = [case["new"]] * n
    if case["spread"] != "same":
        cached = [case["cached"] if i == 0 else r.randint(case["cached"] // 8, case["cached"]) for i in range(n)]
    if case["spread"] == "uniform":  # one long run of new tokens, single ones for the others
        new = [case["new"] if i == 0 or case["new"] <= 12 else 1 for i in range(n)]
    if case["spread"] == "each":
        new = [case["new"] if i == 0 else r.randint(1, case["new"]) for i in range(n)]
    for i in range(case.get("finished", 0)):
        new[1 + i * (n - 1) // case["finished"]] = -1
    return cached, new


def _pages(length, page):
    return -(-length // page)


def work(case):
    cached, new = _lengths(case)
    added = [max(0, a) for a in new]
    tokens, n = sum(added), len(new)
    if case["do"] == "plan":
        page = case["page"]
        moved = sum(_pages(c + a, page) - _pages(c, page) for c, a in zip(cached, added))
        moved += sum(_pages(c, page) for c, a in zip(cached, new) if a < 0)
        # lengths and new in, lengths and starts out; positions and slots out; page numbers twice
        return {"bytes": 16 * n + 12 * tokens + 8 * moved, "flops": 0}
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    if case["do"] == "append":
        b = tokens * (hq * d * 4 + 2 * hkv * d * 3 + 4 * d)
        return {"bytes": b, "flops": tokens * (hq + 2 * hkv) * d * 8}
    keys = sum(c + a for c, a in zip(cached, added))
    pairs = sum(a * c + a * (a + 1) // 2 for c, a in zip(cached, added))
    return {"bytes": keys * hkv * 2 * d + tokens * hq * (4 * d + 4), "flops": 4 * d * hq * pairs}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 250)


def _plain_bytes(case):
    """About what the plain form holds at its largest."""
    cached, new = _lengths(case)
    if case["do"] == "plan":
        return 0
    longest, most = max(max(new), 1), max(c + max(0, a) for c, a in zip(cached, new))
    size = len(new) * most * case["heads_kv"] * case["dim"] * 8
    if case["do"] == "attention":
        size += 16 * len(new) * case["heads_q"] * longest * most
    return size


# ------------------------------------------------------------------------------------ inputs
def _exponent(amax):
    """The smallest e >= FLOOR with amax <= 448 * 2^e."""
    m, x = torch.frexp(amax)  # amax = m * 2^x, m in [0.5, 1)
    e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, FLOOR).clamp_min(FLOOR).to(torch.int32)


def _blocks(g, pages, heads, page, dim, device):
    """Codes and exponents of filled blocks: values of a unit spread, some tokens and channels of them large."""
    x = torch.randn(pages, heads, page, dim, generator=g, device=device)
    x = x * (1 + 7 * (torch.rand(pages, heads, page, 1, generator=g, device=device) < 0.01))
    x = x * torch.exp2(torch.rand(pages, heads, 1, 1, generator=g, device=device) * 3 - 1.5)
    e = _exponent(x.abs().amax(dim=(2, 3)))
    codes = (x * torch.exp2(-e.float())[:, :, None, None]).to(torch.float8_e4m3fn)
    return codes, e.to(torch.int8)


def _tables(case, g, device):
    """The requests' pages, in random order, with what is free behind them."""
    cached, new = _lengths(case)
    page, n = case["page"], len(new)
    held = [_pages(c, page) for c in cached]
    want = [_pages(c + max(0, a), page) for c, a in zip(cached, new)]
    width = max(want) + 2
    pages = sum(max(h, w) for h, w in zip(held, want)) + 7
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    held_t = torch.tensor(held, device=device)
    first = held_t.cumsum(0) - held_t
    at = torch.arange(width, device=device)
    inside = at[None, :] < held_t[:, None]
    table = torch.where(inside, order[(first[:, None] + at).clamp_max(pages - 1)], torch.tensor(-1, dtype=torch.int32, device=device))
    # a ring of page numbers: entries [head, tail) are free; the tail wraps
    head, count = pages - 3, pages - sum(held)
    free = torch.full((pages,), -1, dtype=torch.int32, device=device)
    free[(head + torch.arange(count, device=device)) % pages] = order[sum(held):]
    return {
        "table": table, "free": free, "cursor": torch.tensor([head, head + count], device=device),
        "lengths": torch.tensor(cached, dtype=torch.int32, device=device),
        "new": torch.tensor(new, dtype=torch.int32, device=device),
        "tokens": sum(max(0, a) for a in new), "longest": max(max(new), 1), "pages": pages,
    }


def _inputs(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    s = {"case": case, **_tables(case, g, device)}
    if case["do"] == "plan":
        return s
    hq, hkv, dim, page = case["heads_q"], case["heads_kv"], case["dim"], case["page"]
    # what a step has in hand: its plan, made once for all layers
    made = _plan(s["table"], s["lengths"], s["new"], s["free"], s["cursor"], s["tokens"], page)
    s |= {"after": made["lengths"], "starts": made["starts"], "positions": made["positions"], "slots": made["slots"]}
    s["key"], s["key_exponent"] = _blocks(g, s["pages"], hkv, page, dim, device)
    s["value"], s["value_exponent"] = _blocks(g, s["pages"], hkv, page, dim, device)
    s["query"] = torch.randn(s["tokens"], hq, dim, generator=g, device=device).to(torch.bfloat16)
    if case["do"] == "append":
        amp = 1 + 7 * (torch.rand(s["tokens"], hkv, 1, generator=g, device=device) < 0.01)
        s["new_key"] = (torch.randn(s["tokens"], hkv, dim, generator=g, device=device) * amp).to(torch.bfloat16)
        s["new_value"] = (torch.randn(s["tokens"], hkv, dim, generator=g, device=device) * amp * 0.5).to(torch.bfloat16)
        s["touched"] = torch.unique(s["slots"] // page)
        angle = torch.arange(s["table"].shape[1] * page, dtype=torch.float64, device=device)[:, None]
        angle = angle * case["theta"] ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
        angle = angle if case["interleaved"] else torch.cat([angle, angle], dim=1)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["norm"]:
            s["weight_q"] = 1 + 0.2 * torch.randn(dim, generator=g, device=device)
            s["weight_k"] = 1 + 0.2 * torch.randn(dim, generator=g, device=device)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from cozy_runtime_b200 import cache, rope, ulysses

        page, dim = case["page"], case.get("dim", 128)
        s["layout"] = cache.Layout(heads_q=case.get("heads_q", 32), heads_kv=case.get("heads_kv", 8), head_dim=dim, page=page)
        if case["do"] != "plan":
            s["plan"] = cache.plan(s["layout"], s["table"], s["lengths"], s["new"], s["free"], s["cursor"],
                                   tokens=s["tokens"], longest=s["longest"])
            s["store"] = cache.Cache(s["key"], s["value"], s["key_exponent"], s["value_exponent"])
        if case["do"] == "append":
            s["rope"] = rope.RopeSpec(s["cos"], s["sin"], s["cos"].shape[1], 1, dim, case["interleaved"])
            s["norm_q"] = ulysses.Norm(weight=s["weight_q"], eps=EPS) if case["norm"] else None
            s["norm_k"] = ulysses.Norm(weight=s["weight_k"], eps=EPS) if case["norm"] else None
    return s


# ------------------------------------------------------------------------------------- plain
def _plan(table, lengths, new, free, cursor, tokens, page):
    """Gives pages to the requests that grow and takes those of the finished ones; `table` and
    `free` are written in place, on entries that held nothing."""
    n, width = table.shape
    pages, device = free.numel(), table.device
    length, done = lengths.long(), new < 0
    added = new.long().clamp_min(0)
    held = (length + page - 1) // page
    need = (length + added + page - 1) // page - held
    at = torch.arange(width, device=device)
    place = at[None, :] - held[:, None]
    fresh = (place >= 0) & (place < need[:, None])
    source = cursor[0] + (need.cumsum(0) - need)[:, None] + place
    back = torch.where(done, held, 0)
    target = cursor[1] + (back.cumsum(0) - back)[:, None] + at[None, :]
    given = done[:, None] & (at[None, :] < held[:, None])
    before = table.clone()
    table.copy_(torch.where(fresh, free[source % pages], table))
    spare = torch.cat([free, free.new_empty(1)])
    spare[torch.where(given, target % pages, pages)] = before
    free.copy_(spare[:pages])
    ends = added.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(tokens, device=device)
    request = torch.searchsorted(ends, t, right=True)
    position = length[request] + t - starts[request]
    slots = table[request, position // page].long() * page + position % page
    return {
        "lengths": torch.where(done, 0, length + added).to(torch.int32), "starts": starts.to(torch.int32),
        "cursor": torch.stack([cursor[0] + need.sum(), cursor[1] + back.sum()]),
        "positions": position.to(torch.int32), "slots": slots,
    }


def _turn(x, weight, s):
    """Per-head norm (with `weight`), then rotation by the tokens' positions."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * weight
    cos, sin = (s[k][s["positions"].long()][:, None, :] for k in ("cos", "sin"))
    if s["case"]["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _store(x, codes, exponent, s):
    """Puts rows `x` [tokens, heads, dim] in their slots; a block's scale grows to its largest
    value and what the block holds already is rounded to the grown scale."""
    page, touched = s["case"]["page"], s["touched"]
    where, offset = s["slots"] // page, s["slots"] % page
    fits = x.abs() <= LARGEST
    size = torch.where(fits, x.abs(), 0).amax(dim=-1)
    largest = torch.zeros(exponent.shape, dtype=x.dtype, device=x.device)
    largest.index_reduce_(0, where, size, "amax")
    first = torch.full((exponent.shape[0],), page, device=x.device)
    first.index_reduce_(0, where, offset, "amin")  # a block's rows in front of it are held already
    old = torch.where(first[:, None] == 0, FLOOR, exponent.to(torch.int32))
    grown = torch.maximum(old, _exponent(largest))[touched]
    shift = torch.exp2((old[touched] - grown).to(x.dtype))[:, :, None, None]
    raw = codes.view(torch.uint8)
    before = raw[touched]
    after = (before.view(torch.float8_e4m3fn).to(x.dtype) * shift).to(torch.float8_e4m3fn).view(torch.uint8)
    held = torch.arange(page, device=x.device) < first[touched][:, None]
    raw[touched] = torch.where(held[:, None, :, None], after, before)
    exponent[touched] = grown.to(torch.int8)
    scale = torch.exp2(-exponent[where].to(x.dtype))[:, :, None]
    row = torch.where(fits, x * scale, math.nan).to(torch.float8_e4m3fn)
    raw[where, :, offset] = row.view(torch.uint8)


def _append(s):
    q = _turn(s["query"].float(), s.get("weight_q"), s).to(torch.bfloat16)
    k = _turn(s["new_key"].float(), s.get("weight_k"), s).to(torch.bfloat16)
    _store(k.float(), s["key"], s["key_exponent"], s)
    _store(s["new_value"].float(), s["value"], s["value_exponent"], s)
    return q


def _widened(codes, exponent, pages, dtype):
    """Blocks `pages` [requests, width] as [requests, heads, width * page, dim]."""
    x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(dtype)
    x = x * torch.exp2(exponent[pages].to(dtype))[..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    """Every request padded to the longest; rows in a request's group of heads together."""
    c, device = s["case"], s["query"].device
    n, longest, group = len(s["new"]), s["longest"], c["heads_q"] // c["heads_kv"]
    new, after, starts = s["new"].long(), s["after"].long(), s["starts"].long()
    width = -(-(c["cached"] + c["new"]) // c["page"])
    pages = s["table"][:, :width].long().clamp_min(0)
    k = _widened(s["key"], s["key_exponent"], pages, torch.float32)
    v = _widened(s["value"], s["value_exponent"], pages, torch.float32)
    i = torch.arange(longest, device=device)
    row = (starts[:-1, None] + i).clamp_max(s["tokens"] - 1)
    q = s["query"].float()[row].unflatten(2, (c["heads_kv"], group))  # [n, longest, kv, group, dim]
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(c["dim"])
    score = score.unflatten(2, (group, longest))
    seen = torch.arange(k.shape[2], device=device) <= (after - new)[:, None, None] + i[:, None]
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(dim=-1, keepdim=True)
    v = torch.where((torch.arange(k.shape[2], device=device) < after[:, None])[:, None, :, None], v, 0)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, longest)) / total
    lse = (top + torch.log(total))[..., 0]
    t = torch.arange(s["tokens"], device=device)
    request = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    index = (request, slice(None), slice(None), t - starts[request])
    return out[index].flatten(1, 2).to(torch.bfloat16), lse[index].flatten(1, 2)


def run(s):
    do = s["case"]["do"]
    if own:
        from cozy_runtime_b200 import cache

        if do == "plan":
            made = cache.plan(s["layout"], s["table"], s["lengths"], s["new"], s["free"], s["cursor"],
                              tokens=s["tokens"], longest=s["longest"])
            return [s["table"], s["free"], made.lengths, made.starts, made.cursor, made.positions, made.slots]
        if do == "append":
            q = cache.append(s["store"], s["plan"], s["new_key"], s["new_value"], query=s["query"],
                             rope=s["rope"], norm_q=s["norm_q"], norm_k=s["norm_k"])
            return [q, s["key"], s["value"], s["key_exponent"], s["value_exponent"]]
        out, lse = cache.attention(s["store"], s["plan"], s["query"], return_lse=True)
        return [out, lse]
    if do == "plan":
        p = _plan(s["table"], s["lengths"], s["new"], s["free"], s["cursor"], s["tokens"], s["case"]["page"])
        return [s["table"], s["free"], p["lengths"], p["starts"], p["cursor"], p["positions"], p["slots"]]
    if do == "append":
        q = _append(s)
        return [q, s["key"], s["value"], s["key_exponent"], s["value_exponent"]]
    return list(_attend(s))


# ------------------------------------------------------------------------------------- exact
def _round_e4m3(x):
    """The nearest e4m3 value (ties to the even one) of 64-bit |x| <= 448."""
    step = torch.exp2((torch.frexp(x.abs())[1] - 1).clamp_min(-6).to(x.dtype) - 3)
    return torch.round(x / step) * step


def _exact_store(x, codes, exponent, s, cached, new):
    page = s["case"]["page"]
    codes, exponent, t = codes.double(), exponent.long(), 0
    for n, (c, a) in enumerate(zip(cached, new)):
        for b in range(c // page, _pages(c + a, page)):
            p = int(s["table"][n, b])
            first, last = max(c, b * page), min(c + a, (b + 1) * page)
            rows = x[t + first - c:t + last - c].transpose(0, 1)  # [heads, rows, dim]
            fits = rows.abs() <= LARGEST
            largest = torch.where(fits, rows.abs(), 0).amax(dim=(1, 2))
            e = torch.ceil(torch.log2(largest / 448)).clamp_min(FLOOR).long()
            held = first - b * page
            if held > 0:
                e = torch.maximum(e, exponent[p])
                codes[p, :, :held] = _round_e4m3(codes[p, :, :held] * torch.exp2((exponent[p] - e).double())[:, None, None])
            exponent[p] = e
            stored = _round_e4m3(torch.where(fits, rows, 0) * torch.exp2(-e.double())[:, None, None])
            codes[p, :, first - b * page:last - b * page] = torch.where(fits, stored, math.nan)
        t += a
    return codes, exponent


def _exact_turn(x, weight, s):
    """The pairs of channels as complex numbers, turned by cos + i sin."""
    x, pairs = x.double(), x.shape[-1] // 2
    if weight is not None:
        x = x * weight.double() / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / x.shape[-1] + EPS)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long(), None, :pairs]
    if s["case"]["interleaved"]:
        return torch.view_as_real(torch.complex(x[..., ::2], x[..., 1::2]) * turn).flatten(-2)
    x = torch.complex(x[..., :pairs], x[..., pairs:]) * turn
    return torch.cat([x.real, x.imag], dim=-1)


def exact(case, seed):
    if case["do"] == "plan":
        return None
    s, (cached, new) = _inputs(case, seed), _lengths(case)
    if case["do"] == "append":
        if sum(new) // case["page"] + len(new) > 3000:
            return None
        q = _exact_turn(s["query"], s.get("weight_q"), s)
        k = _exact_turn(s["new_key"], s.get("weight_k"), s).to(torch.bfloat16).double()
        kc, ke = _exact_store(k, s["key"], s["key_exponent"], s, cached, new)
        vc, ve = _exact_store(s["new_value"].double(), s["value"], s["value_exponent"], s, cached, new)
        return [q, kc, vc, None, None]
    group, t, outs, sums = case["heads_q"] // case["heads_kv"], 0, [], []
    for n, (c, a) in enumerate(zip(cached, new)):
        pages = s["table"][n, :_pages(c + a, case["page"])].long()
        out = torch.empty(a, case["heads_q"], case["dim"], dtype=torch.float64, device="cuda")
        lse = torch.empty(a, case["heads_q"], dtype=torch.float64, device="cuda")
        for h in range(case["heads_kv"]):
            k, v = (
                (x[pages, h].double() * torch.exp2(e[pages, h].double())[:, None, None]).flatten(0, 1)[:c + a]
                for x, e in ((s["key"], s["key_exponent"]), (s["value"], s["value_exponent"]))
            )
            heads = slice(h * group, (h + 1) * group)
            score = torch.einsum("tgd,kd->gtk", s["query"][t:t + a, heads].double(), k) / math.sqrt(case["dim"])
            hidden = torch.arange(c + a, device="cuda") > c + torch.arange(a, device="cuda")[:, None]
            score.masked_fill_(hidden, -math.inf)
            lse[:, heads] = torch.logsumexp(score, dim=-1).T
            out[:, heads] = torch.einsum("gtk,kd->tgd", torch.softmax(score, dim=-1), v)
        outs.append(out)
        sums.append(lse)
        t += a
    return [torch.cat(outs), torch.cat(sums)]
