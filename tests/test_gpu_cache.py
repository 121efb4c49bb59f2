"""The 8-bit paged cache on the GPU against its 64-bit restatement (oracle/cache_oracle.py).

Tolerances, in the terms that `attend_step` returns beside the outputs:
* codes of values that no arithmetic touched, exponents and whole numbers: equal;
* rows after norm and rotation: one bf16 rounding, 2^-8 of the value (half a step relative), and
  fp32 arithmetic on a row of up to 128 channels, below 2^-18 of the row's largest value;
* codes of such rows: a bf16 rounding that fell the other way may move a code by one step, 2^-3 of
  the value, or one subnormal step;
* attention: a score has the error of 128 fp32 products and sums of a tensor core (2^-16 of the
  sum of magnitudes `size`, the rounding of a query split into 8-bit parts among it), which moves
  every weight by that relative amount; weights are rounded to 11 bits (2^-11); the output to
  bf16 (2^-8 of the value): |out error| <= 2^-8 |out| + (2^-10 + 2 * 2^-16 * size) * weight, and
  |lse error| <= 2^-16 * size + 2^-20 * (8 + |lse|). An f16 weight has 11 bits down to 2^-14 and an
  absolute error of 2^-25 below; the row's largest is at least 2^7, so n keys of values up to
  448 * 2^e add at most n * 448 * 2^e * 2^-32 to the output (`floor`: it shows where the heavy
  keys' values are exactly zero).
"""

import math

import pytest
import torch

from oracle import cache_oracle as law

pytestmark = pytest.mark.gpu


def make(lengths, new, page, g, *, spare=5, tokens=None, longest=None):
    """A table in random page order, a ring whose free entries wrap, and the plan's arguments."""
    up = lambda x: -(-x // page)  # noqa: E731
    held, want = [up(x) for x in lengths], [up(x + max(a, 0)) for x, a in zip(lengths, new)]
    pages = sum(max(h, w) for h, w in zip(held, want)) + spare
    order = torch.randperm(pages, generator=g).tolist()
    width, at, table = max(want + held) + 1, 0, []
    for h in held:
        table.append(order[at:at + h] + [-1] * (width - h))
        at += h
    head, count = pages - 2, pages - at
    free = [-1] * pages
    for i, p in enumerate(order[at:]):
        free[(head + i) % pages] = p
    return {"table": table, "lengths": lengths, "new": new, "free": free,
            "cursor": [head, head + count],
            "tokens": sum(max(a, 0) for a in new) if tokens is None else tokens,
            "longest": max(new + [0]) if longest is None else longest}


def on_gpu(m, layout):
    from cozy_runtime_b200 import cache

    t = {k: torch.tensor(m[k], dtype=torch.int64 if k == "cursor" else torch.int32, device="cuda")
         for k in ("table", "lengths", "new", "free", "cursor")}
    step = cache.plan(layout, t["table"], t["lengths"], t["new"], t["free"], t["cursor"],
                      tokens=m["tokens"], longest=m["longest"])
    return step, t


def want_plan(m, page):
    return law.plan_step(m["table"], m["lengths"], m["new"], m["free"], m["cursor"],
                         tokens=m["tokens"], longest=m["longest"], page=page)


def fill(pages, heads, page, dim, g, *, outliers=True):
    """Codes and exponents of random blocks, and the values they stand for in 64 bits."""
    from cozy_runtime_b200 import cache  # noqa: F401

    x = torch.randn(pages, heads, page, dim, generator=g)
    if outliers:
        x *= 1 + 7 * (torch.rand(pages, heads, page, 1, generator=g) < 0.02)
    codes = (x * 50).clamp(-448, 448).to(torch.float8_e4m3fn)
    e = torch.randint(-8, -3, (pages, heads), generator=g).to(torch.int8)
    return codes, e


def values(codes, e):
    return codes.double() * torch.exp2(e.double())[..., None, None]


def store_on_gpu(k, ke, v, ve):
    from cozy_runtime_b200 import cache

    return cache.Cache(k.cuda(), v.cuda(), ke.cuda(), ve.cuda())


# ------------------------------------------------------------------------------------------ plan
PLANS = [
    ([0], [1], 16), ([5], [1], 64), ([16], [1], 16), ([15], [1], 16), ([0, 0, 0], [0, 0, 0], 32),
    ([0, 33, 64, 7], [64, 31, 1, 0], 32), ([100, 1, 50, 0], [-1, 3, -1, -1], 16),
    ([127, 128, 129], [129, 128, 127], 128), ([3] * 1500, [1] * 1500, 16),
    ([17 * i % 300 for i in range(2050)], [(7 * i) % 9 - 1 for i in range(2050)], 64),
    ([0, 4000], [9000, 1], 16),
]


@pytest.mark.parametrize("lengths,new,page", PLANS)
def test_plan_matches_the_law(lengths, new, page):
    from cozy_runtime_b200 import cache

    m = make(lengths, new, page, torch.Generator().manual_seed(1))
    m["tokens"] += 3  # rows of nobody behind the last
    want = want_plan(m, page)
    assert want["status"] == 0
    for _ in range(2):  # planning the same tensors again gives the same plan
        step, t = on_gpu(m, cache.Layout(8, 2, 128, page))
        step = cache.plan(step.layout, t["table"], t["lengths"], t["new"], t["free"], t["cursor"],
                          tokens=m["tokens"], longest=m["longest"])
        step.check()
        for name in ("lengths", "starts", "cursor", "positions", "slots"):
            assert getattr(step, name).tolist() == want[name], name
        assert t["table"].tolist() == want["table"] and t["free"].tolist() == want["free"]
        assert t["lengths"].tolist() == lengths and t["cursor"].tolist() == m["cursor"]


@pytest.mark.parametrize("change,bit", [
    ({"cursor": [0, 1]}, 1), ({"new": [100, 900]}, 2), ({"tokens": 4}, 4), ({"longest": 3}, 4),
    ({"lengths": [-5, 40]}, 8), ({"new": [-2, 1]}, 8), ({"cursor": [5, 3]}, 8),
    ({"cursor": [0, 10**6]}, 8), ({"cursor": [-3, 2]}, 8),
    ({"lengths": [2**31 - 1, 1], "new": [2**31 - 1, 1], "longest": 2**31 - 1}, 2),
])
def test_plan_refuses_whole_steps(change, bit):
    from cozy_runtime_b200 import cache

    m = make([20, 40], [40, 2], 16, torch.Generator().manual_seed(2))
    m |= change
    step, t = on_gpu(m, cache.Layout(4, 4, 64, 16))
    want = want_plan(m, 16)
    assert want["status"] & bit and int(step.status) == want["status"]
    with pytest.raises(RuntimeError, match="cache plan"):
        step.check()
    assert t["table"].tolist() == m["table"] and t["free"].tolist() == m["free"]
    assert step.starts.tolist() == [0, 0, 0] and step.cursor.tolist() == m["cursor"]
    assert set(step.positions.tolist()) <= {-1} and set(step.slots.tolist()) <= {-1}
    # and nothing is stored or attended
    k, ke = fill(step.pages, 4, 16, 64, torch.Generator().manual_seed(3))
    store = store_on_gpu(k, ke, k, ke)
    x = torch.ones(m["tokens"], 4, 64, dtype=torch.bfloat16, device="cuda")
    cache.append(store, step, x, x)
    out = cache.attention(store, step, x, out=x.clone())
    assert torch.equal(out, x)
    assert torch.equal(store.key.cpu().view(torch.uint8), k.view(torch.uint8))


def test_plan_leaves_out_bad_pages():
    from cozy_runtime_b200 import cache

    m = make([20, 40], [40, 2], 16, torch.Generator().manual_seed(2))
    m["table"][0][1] = 10**6  # the page that the first request is filling
    m["free"][m["cursor"][0] % len(m["free"])] = -7  # and the first that it is given
    step, _ = on_gpu(m, cache.Layout(4, 4, 64, 16))
    want = want_plan(m, 16)
    assert int(step.status) == want["status"] == 16
    assert step.slots.tolist() == want["slots"] and step.positions.tolist() == want["positions"]


# ---------------------------------------------------------------------------------------- append
APPENDS = [
    # lengths, new, page, heads_q, heads_kv, dim, norm, rotary, interleaved
    ([0], [1], 64, 1, 1, 128, False, 0, False),
    ([70], [1], 64, 8, 2, 128, True, 128, False),
    ([5, 0, 64, 63], [3, 17, 1, 2], 64, 6, 2, 128, True, 128, True),
    ([130, 7], [300, 1], 128, 4, 4, 128, False, 128, False),
    ([130, 7, 0], [300, 0, 90], 16, 5, 5, 64, True, 64, True),
    ([33], [31], 32, 14, 2, 64, True, 32, False),
    ([1] * 40, [1] * 40, 16, 8, 8, 128, True, 96, True),
]


@pytest.mark.parametrize("lengths,new,page,hq,hkv,dim,norm,rotary,interleaved", APPENDS)
def test_append_matches_the_law(lengths, new, page, hq, hkv, dim, norm, rotary, interleaved):
    from cozy_runtime_b200 import cache, rope, ulysses

    g = torch.Generator().manual_seed(4 + len(new))
    layout = cache.Layout(hq, hkv, dim, page)
    m = make(lengths, new, page, g)
    used = m["tokens"]
    m["tokens"] += 2
    step, t = on_gpu(m, layout)
    step.check()
    k0, ke0 = fill(step.pages, hkv, page, dim, g)
    v0, ve0 = fill(step.pages, hkv, page, dim, g)
    # a packed projection: rows of q, k and v beside each other, some far out of scale
    qkv = torch.randn(m["tokens"], hq + 2 * hkv, dim, generator=g)
    qkv *= torch.exp2(torch.randint(-6, 7, (m["tokens"], 1, 1), generator=g).float())
    qkv = qkv.to(torch.bfloat16)
    q, k, v = qkv.split([hq, hkv, hkv], dim=1)
    columns = rotary // 2 if interleaved else rotary
    angle = torch.rand(t["table"].shape[1] * page, max(columns, 1), generator=g) * 6
    spec = rope.RopeSpec(angle.cos().cuda(), angle.sin().cuda(), max(columns, 1), 1, rotary,
                         interleaved) if rotary else None
    weights = [torch.randn(dim, generator=g) for _ in "qk"]
    norms = [ulysses.Norm(w, offset=0.5, eps=1e-5) if norm else None for w in weights]
    store = store_on_gpu(k0, ke0, v0, ve0)
    kept = torch.full((m["tokens"], hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    on = qkv.cuda().split([hq, hkv, hkv], dim=1)
    positions = step.positions.cpu().long()[:used]
    cos, sin = (angle.cos()[positions], angle.sin()[positions]) if rotary else (None, None)
    want = [law.ready(x[:used], w, 0.5, 1e-5 if norm else None, cos, sin, interleaved, rotary)
            for x, w in zip((q, k), weights)]
    table = t["table"].tolist()
    kc, ke = law.append_step(k0.double(), ke0, table, lengths, new,
                             want[1].to(torch.bfloat16).double(), page)
    vc, ve = law.append_step(v0.double(), ve0, table, lengths, new, v[:used].double(), page)
    for _ in range(2):  # the same step again stores the same
        got = cache.append(store, step, on[1], on[2], query=on[0], rope=spec, norm_q=norms[0],
                           norm_k=norms[1], out=kept)
        err = (got[:used].cpu().double() - want[0]).abs()
        bound = 2**-8 * want[0].abs() + 2**-18 * want[0].abs().amax(-1, keepdim=True)
        assert (err <= bound).all(), (err / bound).max()
        assert (got[used:] == 7).all()
        assert torch.equal(store.value.cpu().double(), vc)
        assert torch.equal(store.value_exponent.cpu().long(), ve)
        assert torch.equal(store.key_exponent.cpu().long(), ke)
        err = (store.key.cpu().double() - kc).abs()
        if norm or rotary:
            assert (err <= 2**-3 * kc.abs() + 2**-9).all()
            assert (err > 0).float().mean() < 1e-3
        else:
            assert (err == 0).all()
    step.check()


@pytest.mark.parametrize("dim", [64, 128])
def test_append_grows_a_block_token_by_token(dim):
    """A block filled by single tokens of growing and shrinking size: its exponent grows only, and
    a token of NaN, infinities or too large a magnitude is stored as NaN beside the others."""
    from cozy_runtime_b200 import cache

    g = torch.Generator().manual_seed(9)
    page, hkv = 16, 3
    rows = torch.randn(20, hkv, dim, generator=g)
    rows *= torch.tensor([1, 1e-30, 0, 300, 2, 1e-4, 6e5, 1, 0, 7, 1e9, 3, 448, 449, 450, 1, 1, 2, 3, 4])[:, None, None]
    rows = rows.to(torch.bfloat16)
    rows[4, 0, 5], rows[5, 1, 0], rows[6, 2, 9], rows[7, 0, 1] = math.nan, math.inf, -math.inf, 3e38
    rows[11, 0], rows[12, 1] = 0, torch.tensor(448.0 * 2**40)
    layout = cache.Layout(hkv, hkv, dim, page)
    k0, ke0 = fill(4, hkv, page, dim, g)
    store = store_on_gpu(k0, ke0, k0, ke0)
    codes, e = k0.double(), ke0.long()
    for i in range(20):
        m = {"table": [[2, 1]], "lengths": [i], "new": [1], "free": [0, 1, 2, 3],
             "cursor": [2 if i == 0 else 1, 3], "tokens": 1, "longest": 1}
        step, t = on_gpu(m, layout)
        x = rows[i:i + 1].cuda()
        cache.append(store, step, x, x)
        codes, e = law.append_step(codes, e, t["table"].tolist(), [i], [1], rows[i:i + 1], page)
        for got, ge in ((store.key, store.key_exponent), (store.value, store.value_exponent)):
            assert torch.equal(ge.cpu().long(), e)
            assert torch.equal(got.cpu().double().nan_to_num(9999), codes.nan_to_num(9999))
            assert torch.equal(got.cpu().float().isnan(), codes.isnan())


# ------------------------------------------------------------------------------------- attention
ATTENDS = [
    # lengths, new, page, heads_q, heads_kv, dim
    ([0], [1], 64, 1, 1, 128),
    ([63], [1], 64, 4, 1, 128),
    ([64], [1], 64, 32, 8, 128),
    ([700, 0, 15, 16, 17, 300], [1, 1, 1, 1, 1, 0], 16, 8, 2, 128),
    ([1000, 3, 129], [1, 1, 1], 128, 16, 1, 64),
    ([500, 127, 64], [4, 1, 3], 32, 8, 2, 128),  # a few rows a head, some requests fewer
    ([90, 0, 5], [5, 16, 0], 16, 3, 3, 64),
    ([200, 31], [9, 2], 32, 10, 2, 128),
    ([0], [130], 64, 4, 4, 128),
    ([0, 77, 513], [300, 1, 40], 16, 8, 2, 64),
    ([1000, 256, 255], [257, 64, 1], 128, 12, 3, 128),
    ([33, 5], [70, 3], 32, 21, 3, 128),  # a group of 7
    ([40], [5], 16, 128, 1, 64),  # a group of 128
]


def floor_of(keys, ve):
    return keys * 448.0 * 2.0 ** (int(ve.max()) - 32)


def check_attention(out, lse, want, used, floor):
    ref, rlse, weight, size = (x[:used] for x in want)
    err = (out[:used].cpu().double() - ref).abs()
    bound = 2**-8 * ref.abs() + (2**-10 + 2**-15 * size[..., None]) * weight + floor
    assert (err <= bound).all(), (err / bound).max()
    if lse is not None:
        seen = rlse > -math.inf
        err = (lse[:used].cpu().double() - rlse)[seen].abs()
        assert (err <= (2**-16 * size + 2**-20 * (8 + rlse.abs()))[seen]).all(), err.max()
        assert (lse[:used].cpu()[~seen] == -math.inf).all()


@pytest.mark.parametrize("amp", [1.0, 6.0])
@pytest.mark.parametrize("lengths,new,page,hq,hkv,dim", ATTENDS)
def test_attention_matches_the_law(lengths, new, page, hq, hkv, dim, amp):
    from cozy_runtime_b200 import cache

    g = torch.Generator().manual_seed(hq + dim)
    m = make(lengths, new, page, g)
    used = m["tokens"]
    m["tokens"] += 2
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    # what no row sees is NaN: pages of nobody and rows behind a sequence's end
    seen = torch.zeros(step.pages, page, dtype=torch.bool)
    table = t["table"].tolist()
    for n, (x, a) in enumerate(zip(lengths, new)):
        for i in range(x + max(a, 0)):
            seen[table[n][i // page], i % page] = True
    hidden = ~seen[:, None, :, None]
    k, v = (torch.where(hidden, math.nan, x.float()).to(torch.float8_e4m3fn) for x in (k, v))
    q = (torch.randn(m["tokens"], hq, dim, generator=g) * amp).to(torch.bfloat16)
    store = store_on_gpu(k, ke, v, ve)
    scale = 1 / math.sqrt(dim)
    want = law.attend_step(values(k, ke), values(v, ve), table, lengths, new, q, page, scale)
    kept = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = cache.attention(store, step, q.cuda(), out=kept, return_lse=True)
    floor = floor_of(max(x + max(a, 0) for x, a in zip(lengths, new)), ve)
    check_attention(out, lse, want, used, floor)
    assert (out[used:] == 7).all()
    again = cache.attention(store, step, q.cuda())
    assert torch.equal(again[:used], out[:used])
    step.check()
