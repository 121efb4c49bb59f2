"""The 8-bit paged cache's laws, restated plainly: whole numbers in Python, values in 64 bits.

Test infrastructure only. Blocks hold e4m3 codes under a power of two: `plan_step` gives pages,
`append_step` stores rows, `attend_step` reads them.
"""

from __future__ import annotations

import math

import torch

FLOOR = -60
LARGEST = 448.0 * 2.0**40


def plan_step(table, lengths, new, free, cursor, *, tokens, longest, page, reached=None):
    """Lists in (table: list of rows; copies are changed), a dict out. `reached`: lengths that the
    rows held pages for, where they were set back since."""
    reached = lengths if reached is None else reached
    table, free = [list(r) for r in table], list(free)
    pages, width, (head, tail) = len(free), len(table[0]), cursor
    up = lambda x: -(-x // page)  # noqa: E731
    status, need, back, total = 0, 0, 0, 0
    for length, a, r in zip(lengths, new, reached):
        held, want = up(max(length, r)), up(length + a) if a >= 0 else 0
        if length < 0 or a < -1 or r < 0:
            status |= 8
            continue
        status |= 2 * (max(held, want) > width) | 4 * (a > longest)
        need += max(0, want - held)
        back += max(0, held - want)
        total += max(a, 0)
    if head < 0 or tail < head or tail - head > pages:
        status |= 8
    elif need > tail - head:
        status |= 1
    elif tail - head + back > pages:
        status |= 8
    status |= 4 * (total > tokens)
    if not status:  # numbers outside the pool do not come into the ring
        gone = (p for row, length, a, r in zip(table, lengths, new, reached)
                for p in row[up(length + a) if a >= 0 else 0:up(max(length, r))])
        status = 16 * any(not 0 <= p < pages for p in gone)
    out = {"status": status, "table": table, "free": free, "lengths": [max(x, 0) for x in lengths],
           "cursor": [head, tail], "starts": [0] * (len(new) + 1), "positions": [-1] * tokens,
           "slots": [-1] * tokens}
    if status:
        return out
    before, t = [list(r) for r in table], 0
    for n, (length, a, r) in enumerate(zip(lengths, new, reached)):
        held = up(max(length, r))
        for i in range(up(length + a) if a >= 0 else 0, held):
            free[tail % pages] = before[n][i]
            tail += 1
        if a < 0:
            out["lengths"][n] = 0
        else:
            for b in range(held, up(length + a)):
                table[n][b] = free[head % pages]
                head += 1
            for x in range(length, length + a):
                p = table[n][x // page]
                if 0 <= p < pages:
                    out["positions"][t], out["slots"][t] = x, p * page + x % page
                else:
                    out["status"] |= 16
                t += 1
            out["lengths"][n] = length + a
        out["starts"][n + 1] = t
    out["cursor"] = [head, tail]
    return out


def exponent(amax: float) -> int:
    """The smallest e >= FLOOR with amax <= 448 * 2^e."""
    e = FLOOR
    while amax > 448.0 * 2.0**e:
        e += 1
    return e


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to the even one (|x| <= 448; NaN stays)."""
    step = torch.exp2((torch.frexp(x.abs())[1] - 1).clamp_min(-6).double() - 3)
    return torch.round(x / step) * step


def ready(x, weight, offset, eps, cos, sin, interleaved, rotary):
    """Per-head norm (`eps` None: none) and rotation of rows [tokens, heads, dim] in 64 bits;
    cos and sin [tokens, columns]."""
    x = x.double()
    if eps is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            x = x * (weight.double() + offset)
    if cos is None:
        return x
    y, half = x.clone(), rotary // 2
    for i in range(half):
        a, b, ca, cb = (2 * i, 2 * i + 1, i, i) if interleaved else (i, i + half, i, i + half)
        y[..., a] = x[..., a] * cos[:, None, ca].double() - x[..., b] * sin[:, None, ca].double()
        y[..., b] = x[..., b] * cos[:, None, cb].double() + x[..., a] * sin[:, None, cb].double()
    return y


def append_step(codes, exponents, table, lengths, new, rows, page):
    """Codes [pages, heads, page, dim] (64-bit values of the codes) and exponents [pages, heads]
    with rows [tokens, heads, dim] of a step put in; copies."""
    codes, exponents, t = codes.clone(), exponents.clone().long(), 0
    for n, (length, a) in enumerate(zip(lengths, new)):
        a = max(a, 0)
        for b in range(length // page, -(-(length + a) // page) if a else 0):
            low, high, p = max(length, b * page), min(length + a, (b + 1) * page), table[n][b]
            if not 0 <= p < codes.shape[0]:  # tokens of a page that is not there are left out
                continue
            for h in range(codes.shape[1]):
                x = rows[t + low - length:t + high - length, h].double()
                fits = x.abs() <= LARGEST
                e = exponent(float(torch.where(fits, x.abs(), 0).max()))
                held = low - b * page
                if held:
                    e = max(e, int(exponents[p, h]))
                    moved = codes[p, h, :held] * 2.0 ** (int(exponents[p, h]) - e)
                    codes[p, h, :held] = round_e4m3(moved)
                exponents[p, h] = e
                stored = torch.where(fits, round_e4m3(torch.where(fits, x, 0) * 2.0**-e), math.nan)
                codes[p, h, held:high - b * page] = stored
        t += a
    return codes, exponents


def attend_step(key, value, table, lengths, new, query, page, scale):
    """out, lse, and for the tolerances: the mean of |v| under each row's weights, and the largest
    sum of |q k| * scale of a key that the row sees. key and value [pages, heads, page, dim] are
    stored values (code * 2^exponent) in 64 bits; lengths before the step."""
    tokens, heads_q, dim = query.shape
    group = heads_q // key.shape[1]
    out = torch.zeros(tokens, heads_q, dim, dtype=torch.float64)
    lse = torch.full((tokens, heads_q), -math.inf, dtype=torch.float64)
    weight, size = torch.zeros_like(out), torch.zeros_like(lse)
    t = 0
    for n, (length, a) in enumerate(zip(lengths, new)):
        for i in range(max(a, 0)):
            x = length + i + 1
            pages = table[n][:-(-x // page)]
            good = torch.tensor([0 <= p < key.shape[0] for p in pages]).repeat_interleave(page)[:x]
            at = torch.tensor([p if 0 <= p < key.shape[0] else 0 for p in pages])
            for h in range(key.shape[1]):
                k, v = (c[at, h].flatten(0, 1)[:x][good] for c in (key, value))
                if not len(k):
                    continue
                q = query[t, h * group:(h + 1) * group].double()
                s = q @ k.T * scale
                p = torch.softmax(s, -1)
                rows = slice(h * group, (h + 1) * group)
                lse[t, rows], out[t, rows] = torch.logsumexp(s, -1), p @ v
                weight[t, rows] = p @ v.abs()
                size[t, rows] = (q.abs() @ k.abs().T * scale).amax(-1)
            t += 1
    return out, lse, weight, size
