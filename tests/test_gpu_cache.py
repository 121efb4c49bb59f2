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


@pytest.mark.parametrize("requests", [3, 1500])
def test_plan_refuses_to_release_what_is_not_in_the_pool(requests):
    """A finished or shortened row with a number outside the pool: the step changes nothing, and
    the ring holds pages of the pool only; without that row it is served."""
    from cozy_runtime_b200 import cache

    layout = cache.Layout(4, 4, 64, 16)
    lengths = [20 + 37 * i % 90 for i in range(requests)]
    for bad, new_there in ((-1, -1), (10**6, -1), (-1, 0)):
        new = [-1 if i % 7 == 0 else 1 for i in range(requests)]
        m = make(lengths, new, 16, torch.Generator().manual_seed(2))
        who = requests - 2
        new[who] = new_there
        m["new"], set_back = new, list(lengths)
        if new_there == 0:  # a row set back to where its last page is not needed
            set_back[who] = 16 * ((lengths[who] - 1) // 16)
        m["table"][who][(lengths[who] - 1) // 16] = bad
        t = {k: torch.tensor(m[k], dtype=torch.int64 if k == "cursor" else torch.int32, device="cuda")
             for k in ("table", "lengths", "new", "free", "cursor")}
        t["lengths"].copy_(torch.tensor(set_back, dtype=torch.int32))
        reached = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want = law.plan_step(m["table"], set_back, new, m["free"], m["cursor"], tokens=requests, longest=1, page=16,
                             reached=lengths)
        step = cache.plan(layout, *t.values(), tokens=requests, longest=1, reached=reached)
        assert int(step.status) == want["status"] == 16
        assert t["table"].tolist() == m["table"] and t["free"].tolist() == m["free"]
        assert step.starts.tolist() == [0] * (requests + 1) and step.cursor.tolist() == m["cursor"]
        assert step.lengths.tolist() == set_back
        t["lengths"][who] = reached[who] = 0  # the host hands the row on instead
        step = cache.plan(layout, *t.values(), tokens=requests, longest=1, reached=reached)
        step.check()


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


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_reads_tables_and_weights_of_any_alignment(interleaved):
    """Tables and weights 4 bytes behind a 16-byte boundary, strided tables: the same bits."""
    from cozy_runtime_b200 import cache, rope, ulysses

    dim, page, hkv, hq, new = 64, 32, 2, 6, [70, 1, 9]
    g = torch.Generator().manual_seed(15)
    m = make([3, 40, 0], new, page, g)
    layout = cache.Layout(hq, hkv, dim, page)
    step, t = on_gpu(m, layout)
    columns = dim // 2 if interleaved else dim
    angle = torch.rand(t["table"].shape[1] * page, columns, generator=g).cuda() * 6
    weight = torch.randn(dim, generator=g).cuda()
    q, k = (torch.randn(m["tokens"], h, dim, generator=g).to(torch.bfloat16).cuda() for h in (hq, hkv))

    def behind(x):
        whole = x.new_empty(x.numel() + 1)
        whole[1:] = x.flatten()
        return whole[1:].view(x.shape)

    def apart(x):
        whole = x.new_zeros(x.shape[0], 2 * x.shape[1] + 3)
        whole[:, 0:2 * x.shape[1]:2] = x
        return whole

    cos, sin = angle.cos(), angle.sin()
    got = []
    for c, s, strides, w in ((cos, sin, (columns, 1), weight),
                             (behind(cos), behind(sin), (columns, 1), behind(weight)),
                             (apart(cos), apart(sin), (2 * columns + 3, 2), behind(weight))):
        spec = rope.RopeSpec(c, s, *strides, dim, interleaved)
        store = cache.Cache.empty(layout, step.pages)
        for codes in (store.key, store.value):
            codes.view(torch.uint8).zero_()
        norm = ulysses.Norm(w, offset=0.25, eps=1e-6)
        out = cache.append(store, step, k, k, query=q, rope=spec, norm_q=norm, norm_k=norm)
        got.append((out, store.key.view(torch.uint8), store.key_exponent, store.value.view(torch.uint8)))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_keeps_what_is_not_finite_to_its_pair(interleaved):
    """NaN and infinities reach the channels that the rotation pairs them with, no others."""
    from cozy_runtime_b200 import cache, rope

    dim, rotary, page, hkv, tokens = 64, 32, 16, 2, 5
    g = torch.Generator().manual_seed(14)
    m = make([3], [tokens], page, g)
    step, t = on_gpu(m, cache.Layout(4, hkv, dim, page))
    columns = rotary // 2 if interleaved else rotary
    angle = torch.rand(t["table"].shape[1] * page, columns, generator=g) + 0.3
    spec = rope.RopeSpec(angle.cos().cuda(), angle.sin().cuda(), columns, 1, rotary, interleaved)
    x = torch.randn(tokens, 4, dim, generator=g).to(torch.bfloat16)
    spots = {0: math.inf, 1: math.nan, 9: -math.inf, 33: math.inf, 40: math.nan, 63: -math.inf}
    touched = torch.zeros(dim, dtype=torch.bool)
    for d, v in spots.items():
        x[2, 1, d] = v
        other = d if d >= rotary else d ^ 1 if interleaved else (d + rotary // 2) % rotary
        touched[[d, other]] = True
    k, ke = fill(step.pages, hkv, page, dim, g)
    store = store_on_gpu(k, ke, k, ke)
    out = cache.append(store, step, x[:, :hkv].cuda(), x[:, :hkv].cuda(), query=x.cuda(), rope=spec)
    clean = torch.ones(tokens, 4, dim, dtype=torch.bool)
    clean[2, 1] = ~touched
    assert torch.equal(out.isfinite().cpu(), clean)
    slot = int(step.slots[2])
    stored = store.key[slot // page, :, slot % page].float().cpu()
    assert torch.equal(stored.isnan(), ~clean[2, :hkv])


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


@pytest.mark.parametrize("lengths,new,page,hq,hkv,dim", [
    ([20000], [1], 64, 8, 2, 128),  # one row's keys over every worker
    ([9000, 40], [3, 1], 128, 4, 2, 64),
    ([3000, 0], [200, 1], 32, 6, 2, 128),  # an item's tiles over several workers
    ([2500], [90], 64, 2, 1, 64),
])
def test_attention_over_long_contexts(lengths, new, page, hq, hkv, dim):
    from cozy_runtime_b200 import cache

    g = torch.Generator().manual_seed(sum(lengths))
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16)
    out, lse = cache.attention(store_on_gpu(k, ke, v, ve), step, q.cuda(), scale=0.2, return_lse=True)
    want = law.attend_step(values(k, ke), values(v, ve), t["table"].tolist(), lengths, new, q, page, 0.2)
    check_attention(out, lse, want, m["tokens"], floor_of(max(lengths) + max(new), ve))


@pytest.mark.parametrize("dim,hq", [(64, 20), (128, 20), (128, 24)])
def test_attention_of_many_short_items(dim, hq):
    """Items of one and two query tiles that follow one another in a worker, each with its output
    staged where the next one's queries come: every repetition gives the same bits."""
    from cozy_runtime_b200 import cache

    hkv, page, requests = 4, 16, 240
    g = torch.Generator().manual_seed(dim + hq)
    lengths = torch.randint(0, 200, (requests,), generator=g).tolist()
    new = torch.randint(7, 60, (requests,), generator=g).tolist()
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16)
    store, mine = store_on_gpu(k, ke, v, ve), q.cuda()
    out, lse = cache.attention(store, step, mine, return_lse=True)
    want = law.attend_step(values(k, ke), values(v, ve), t["table"].tolist(), lengths, new, q, page, dim**-0.5)
    check_attention(out, lse, want, m["tokens"], floor_of(300, ve))
    for _ in range(200):
        again, again_lse = cache.attention(store, step, mine, return_lse=True)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_whose_second_query_tile_skips_items(dim):
    """Workers whose items are of one query tile for many tiles of keys, then of two: the second
    tile's rows meet the scales of their own keys."""
    from cozy_runtime_b200 import cache

    hq, hkv, page, requests = 2, 2, 16, 200
    g = torch.Generator().manual_seed(dim)
    lengths = torch.randint(300, 700, (requests,), generator=g).tolist()
    new = [142 if n % 13 == 12 else 30 + n % 60 for n in range(requests)]
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16)
    store, mine, table = store_on_gpu(k, ke, v, ve), q.cuda(), t["table"].tolist()
    two = [n for n in range(requests) if new[n] > 128]
    rows = torch.cat([sum(new[:n]) + torch.arange(new[n]) for n in two])
    want = law.attend_step(values(k, ke), values(v, ve), [table[n] for n in two], [lengths[n] for n in two],
                           [new[n] for n in two], q[rows], page, dim**-0.5)
    for _ in range(5):
        out, lse = cache.attention(store, step, mine, return_lse=True)
        check_attention(out[rows], lse[rows], want, len(rows), floor_of(850, ve))


@pytest.mark.parametrize("lengths,new,hq,hkv,dim", [
    ([100, 30], [1, 1], 4, 2, 128), ([100, 30], [5, 3], 2, 1, 64), ([100, 30], [150, 90], 4, 2, 128),
    ([100, 30], [150, 90], 3, 1, 64),
])
def test_attention_nan_reaches_the_rows_that_see_it(lengths, new, hq, hkv, dim):
    """A NaN value reaches its own channels, a NaN key whole rows, of those rows only that see it."""
    from cozy_runtime_b200 import cache

    page = 32
    g = torch.Generator().manual_seed(3)
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16).cuda()
    plain, plain_lse = cache.attention(store_on_gpu(k, ke, v, ve), step, q, return_lse=True)
    table, group = t["table"].tolist(), hq // hkv
    kf, vf = k.float(), v.float()
    spots = [(0, lengths[0] + new[0] - 1, "v"), (0, 7, "v"), (1, lengths[1] + new[1] // 2, "k")]
    for n, x, which in spots:
        to = (kf if which == "k" else vf)[table[n][x // page], hkv - 1, x % page]
        to[dim - 3] = math.nan
    got, lse = cache.attention(
        store_on_gpu(kf.to(torch.float8_e4m3fn), ke, vf.to(torch.float8_e4m3fn), ve), step, q, return_lse=True)
    hit = torch.zeros(got.shape, dtype=torch.bool)
    t0 = 0
    for n, (length, a) in enumerate(zip(lengths, new)):
        for i in range(a):
            for which_n, x, which in spots:
                if which_n == n and x <= length + i:
                    channels = slice(None) if which == "k" else slice(dim - 3, dim - 2)
                    hit[t0 + i, (hkv - 1) * group:, channels] = True
        t0 += a
    assert torch.equal(got.isnan().cpu(), hit)
    assert torch.equal(got.cpu()[~hit], plain.cpu()[~hit])
    rows = hit.all(-1)
    assert torch.equal(lse.cpu()[~rows], plain_lse.cpu()[~rows]) and lse.cpu()[rows].isnan().all()


@pytest.mark.parametrize("spot", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("lengths,new,dim", [
    ([100, 30], [1, 1], 128), ([100, 30], [3, 2], 64), ([20000, 30], [1, 1], 128),  # the last: joined parts
    ([100, 30], [150, 90], 128), ([100, 30], [80, 1], 64),
])
def test_attention_of_a_query_that_is_not_finite_is_nan(lengths, new, dim, spot):
    """An infinity's scores are infinite or NaN, of one sign too where the keys are: no softmax."""
    from cozy_runtime_b200 import cache

    page, hq, hkv = 32, 4, 2
    g = torch.Generator().manual_seed(3)
    m = make(lengths, new, page, g)
    step, _ = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    k[..., 5] = 3.0  # every key's share of an infinity here has its sign
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16)
    store = store_on_gpu(k, ke, v, ve)
    plain, plain_lse = cache.attention(store, step, q.cuda(), return_lse=True)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool)
    for t, h in ((0, 1), (m["tokens"] - 1, 3), (m["tokens"] // 2, 2)):
        q[t, h, 5], hit[t, h] = spot, True
    out, lse = cache.attention(store, step, q.cuda(), return_lse=True)
    assert torch.equal(out.isnan().cpu(), hit[..., None].expand(q.shape)) and torch.equal(lse.isnan().cpu(), hit)
    assert torch.equal(out.cpu()[~hit], plain.cpu()[~hit]) and torch.equal(lse.cpu()[~hit], plain_lse.cpu()[~hit])


@pytest.mark.parametrize("new,dim", [([1, 1, 1], 128), ([4, 1, 2], 64), ([200, 1, 60], 128), ([70, 70, 1], 64)])
def test_attention_leaves_out_bad_pages(new, dim):
    """Page numbers outside the pool (written into the table behind the plan): their keys are left
    out and the status says so; a row without any key is zero, its lse -inf."""
    from cozy_runtime_b200 import cache

    lengths, page, hq, hkv = [130, 75, 20], 16, 4, 2
    g = torch.Generator().manual_seed(8)
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    table = t["table"].tolist()
    table[0][2], table[0][5], table[0][8], table[2] = step.pages, -1, 2**31 - 1, [-5] * len(table[2])
    t["table"].copy_(torch.tensor(table, dtype=torch.int32))
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16)
    out, lse = cache.attention(store_on_gpu(k, ke, v, ve), step, q.cuda(), return_lse=True)
    want = law.attend_step(values(k, ke), values(v, ve), table, lengths, new, q, page, dim**-0.5)
    check_attention(out, lse, want, m["tokens"], floor_of(500, ve))
    assert (out[-new[2]:] == 0).all()
    assert int(step.status) == 16


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_step_with_bad_pages_among_good_ones(interleaved):
    """Tokens whose own page number is outside the pool: nothing of them is stored, their ready
    queries are zeros, and every other row and block is what the law gives."""
    from cozy_runtime_b200 import cache, rope

    lengths, new, page, hq, hkv, dim = [20, 40, 7], [40, 2, 1], 16, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    m = make(lengths, new, page, g)
    used = m["tokens"]
    m["tokens"] += 2
    m["table"][0][1] = 10**6  # the page that the first request is filling
    m["free"][m["cursor"][0] % len(m["free"])] = -7  # and the first that it is given
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    positions, table = step.positions.cpu().long()[:used], t["table"].tolist()
    bad = positions < 0
    assert bad.tolist() == [i < 28 for i in range(used)]
    k0, ke0 = fill(step.pages, hkv, page, dim, g)
    v0, ve0 = fill(step.pages, hkv, page, dim, g)
    store = store_on_gpu(k0, ke0, v0, ve0)
    columns = dim // 2 if interleaved else dim
    angle = torch.rand(t["table"].shape[1] * page, columns, generator=g) * 6
    spec = rope.RopeSpec(angle.cos().cuda(), angle.sin().cuda(), columns, 1, dim, interleaved)
    q, k, v = (torch.randn(m["tokens"], h, dim, generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv))
    kept = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    got = cache.append(store, step, k.cuda(), v.cuda(), query=q.cuda(), rope=spec, out=kept)
    assert (got[:used][bad.cuda()] == 0).all() and (got[used:] == 7).all()
    cos, sin = angle.cos()[positions.clamp_min(0)], angle.sin()[positions.clamp_min(0)]
    want_q, want_k = (law.ready(x[:used], None, 0.0, None, cos, sin, interleaved, dim) for x in (q, k))
    err = (got[:used].cpu().double() - want_q).abs()
    assert (err <= 2**-8 * want_q.abs() + 2**-18 * want_q.abs().amax(-1, keepdim=True))[~bad].all()
    kc, ke = law.append_step(k0.double(), ke0, table, lengths, new, want_k.to(torch.bfloat16).double(), page)
    vc, ve = law.append_step(v0.double(), ve0, table, lengths, new, v[:used].double(), page)
    assert torch.equal(store.value.cpu().double(), vc) and torch.equal(store.value_exponent.cpu().long(), ve)
    assert torch.equal(store.key_exponent.cpu().long(), ke)
    assert ((store.key.cpu().double() - kc).abs() <= 2**-3 * kc.abs() + 2**-9).all()
    out, lse = cache.attention(store, step, got, return_lse=True)
    stored = [values(c.cpu(), e.cpu()) for c, e in ((store.key, store.key_exponent), (store.value, store.value_exponent))]
    want = law.attend_step(*stored, table, lengths, new, got.cpu(), page, dim**-0.5)
    check_attention(out, lse, want, used, floor_of(60, store.value_exponent))
    assert int(step.status) == 16


@pytest.mark.parametrize("new", [[1, 2], [70, 90]])
def test_attention_over_the_whole_range_of_scales(new):
    """Value exponents from the floor to the ceiling in one row, keys of tiny blocks, zero queries."""
    from cozy_runtime_b200 import cache

    lengths, page, hq, hkv, dim = [200, 90], 16, 2, 1, 64
    g = torch.Generator().manual_seed(5)
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, _ = fill(step.pages, hkv, page, dim, g)
    ve = torch.randint(-60, 41, (step.pages, hkv), generator=g).to(torch.int8)
    ke[::3] = -60
    k[1::5] = 0
    q = torch.randn(m["tokens"], hq, dim, generator=g)
    q[::4] = 0
    q[1::4] *= 1e-20
    q = q.to(torch.bfloat16)
    out, lse = cache.attention(store_on_gpu(k, ke, v, ve), step, q.cuda(), return_lse=True)
    want = law.attend_step(values(k, ke), values(v, ve), t["table"].tolist(), lengths, new, q, page, dim**-0.5)
    check_attention(out, lse, want, m["tokens"], floor_of(300, ve))


@pytest.mark.parametrize("new", [[2, 1, 3], [70, 90, 60]])
def test_attention_over_the_scales_of_a_rows_own_blocks(new):
    """Requests and heads whose values are all tiny, all ordinary or all huge, in one step: the
    absolute error of a row is that of the scales it sees, not of the pool's largest."""
    from cozy_runtime_b200 import cache

    lengths, page, hq, hkv, dim = [200, 90, 133], 16, 4, 2, 64
    g = torch.Generator().manual_seed(21)
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g)
    v, ve = fill(step.pages, hkv, page, dim, g)
    floor, table, t0 = torch.zeros(m["tokens"], hq, 1, dtype=torch.float64), t["table"].tolist(), 0
    for n, (length, a) in enumerate(zip(lengths, new)):
        for h in range(hkv):
            low = [-60, -8, 34][(n + h) % 3]
            pages = table[n][:-(-(length + a) // page)]
            ve[pages, h] = torch.randint(low, low + 7, (len(pages),), generator=g).to(torch.int8)
            floor[t0:t0 + a, h * hq // hkv:(h + 1) * hq // hkv] = floor_of(length + a, ve[pages, h])
        t0 += a
    q = torch.randn(m["tokens"], hq, dim, generator=g).to(torch.bfloat16)
    out, lse = cache.attention(store_on_gpu(k, ke, v, ve), step, q.cuda(), return_lse=True)
    want = law.attend_step(values(k, ke), values(v, ve), table, lengths, new, q, page, dim**-0.5)
    check_attention(out, lse, want, m["tokens"], floor)


@pytest.mark.parametrize("new,dim", [([1, 3], 128), ([2, 1], 64), ([60, 90], 128), ([130, 40], 64)])
def test_attention_of_queries_with_one_large_channel(new, dim):
    """One channel of a query 2000 times the others and the keys zero in it. In a chunk a query is two
    e4m3 parts whose largest value is scaled into (224, 448]: each channel is off by half a
    subnormal step, 2^-10, or less, so a score by amax(q) · 2^-10 / 224 · sum |k| · scale on top of
    the usual 2^-16 of its sum of magnitudes. Single tokens and drafts do without that."""
    from cozy_runtime_b200 import cache

    lengths, page, hq, hkv = [150, 77], 16, 4, 2
    g = torch.Generator().manual_seed(dim + len(new))
    m = make(lengths, new, page, g)
    step, t = on_gpu(m, cache.Layout(hq, hkv, dim, page))
    k, ke = fill(step.pages, hkv, page, dim, g, outliers=False)
    v, ve = fill(step.pages, hkv, page, dim, g)
    k[..., 7] = 0
    q = torch.randn(m["tokens"], hq, dim, generator=g) * 0.05
    q[..., 7] = torch.where(torch.rand(q.shape[:2], generator=g) < 0.5, -1, 1) * (60 + 60 * torch.rand(q.shape[:2], generator=g))
    q = q.to(torch.bfloat16)
    out, lse = cache.attention(store_on_gpu(k, ke, v, ve), step, q.cuda(), return_lse=True)
    scale, kv, table = dim**-0.5, values(k, ke), t["table"].tolist()
    ref, rlse, weight, size = law.attend_step(kv, values(v, ve), table, lengths, new, q, page, scale)
    off, t0 = 2**-16 * size, 0
    for n, (length, a) in enumerate(zip(lengths, new)):
        if a * hq // hkv > 24:
            rows = kv[table[n][:-(-(length + a) // page)]].abs().sum(-1).amax((0, 2))  # of each key head
            amax = q[t0:t0 + a].double().abs().amax(-1)
            off[t0:t0 + a] += amax * 2**-10 / 224 * rows.repeat_interleave(hq // hkv) * scale
        t0 += a
    assert off.max() < 0.04  # e^(2 off) - 1 < 2.1 off
    err = (out.cpu().double() - ref).abs()
    bound = 2**-8 * ref.abs() + (2**-10 + 2.1 * off[..., None]) * weight + floor_of(300, ve)
    assert (err <= bound).all(), (err / bound).max()
    err = (lse.cpu().double() - rlse).abs()
    assert (err <= off + 2**-20 * (8 + rlse.abs())).all(), err.max()


def test_attention_far_into_a_large_pool():
    """Blocks behind the first 4 GB of a pool, rows of a packed projection, a strided output."""
    from cozy_runtime_b200 import cache

    page, hkv, hq, dim, pages = 128, 8, 16, 128, 40000
    g = torch.Generator().manual_seed(6)
    for lengths, new in (([300, 77], [1, 1]), ([300, 77], [60, 40])):  # 3 pages and 1
        layout = cache.Layout(hq, hkv, dim, page)
        large = cache.Cache.empty(layout, pages)
        table = torch.tensor([[pages - 1, 5, pages - 2, pages - 7], [pages - 4, pages - 3, 0, 1]], dtype=torch.int32)
        small_table = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7]], dtype=torch.int32)
        k, ke = fill(8, hkv, page, dim, g)
        v, ve = fill(8, hkv, page, dim, g)
        small = store_on_gpu(k, ke, v, ve)
        at = table.reshape(-1).long().cuda()
        for to, of in ((large.key, small.key), (large.value, small.value)):
            to.view(torch.uint8)[at] = of.view(torch.uint8)
        for to, of in ((large.key_exponent, small.key_exponent), (large.value_exponent, small.value_exponent)):
            to[at] = of
        T = sum(new)
        qkv = torch.randn(T, hq + 2 * hkv, dim, generator=g).to(torch.bfloat16).cuda()
        q = qkv[:, :hq]
        outs = []
        for store, tab, n_pages in ((large, table, pages), (small, small_table, 8)):
            # no request needs a page that its row does not name already
            step = cache.plan(layout, tab.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                              torch.tensor(new, dtype=torch.int32).cuda(),
                              torch.zeros(n_pages, dtype=torch.int32).cuda(),
                              torch.zeros(2, dtype=torch.int64).cuda(), tokens=T, longest=max(new))
            outs.append((store, step))
        results = []
        for store, step in outs:
            step.check()
            cache.append(store, step, qkv[:, hq:hq + hkv], qkv[:, hq + hkv:])
            out = torch.zeros(T, 2 * hq, dim, dtype=torch.bfloat16, device="cuda")
            cache.attention(store, step, q, out=out[:, ::2])
            assert (out[:, 1::2] == 0).all()
            results.append(out)
        assert torch.equal(results[0], results[1])
        assert torch.equal(large.key.view(torch.uint8)[at], small.key.view(torch.uint8))


# --------------------------------------------------------------------------------------- together
def test_requests_come_grow_and_go():
    """Steps as a server makes them: prompts in chunks, single tokens, drafts, finished requests
    whose pages go to others, two layers. Lengths and cursor go from step to step."""
    from cozy_runtime_b200 import cache, rope, ulysses

    g = torch.Generator().manual_seed(12)
    layout = cache.Layout(6, 2, 64, 16)
    pages, width = 40, 20
    table = torch.zeros(3, width, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=g).to(torch.int32).cuda()
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    cursor = torch.tensor([0, pages], device="cuda")
    stores = [cache.Cache.empty(layout, pages) for _ in "ab"]
    spec = rope.llama(width * 16, 64).to("cuda")
    norm = ulysses.Norm(torch.rand(64, generator=g) + 0.5)
    steps = [[70, 5, 0], [33, 1, 90], [1, 1, 1], [4, -1, 1], [1, 200, 3], [-1, 1, 1], [120, -1, -1], [1, 0, 40]]
    held = [0, 0, 0]
    for new in steps:
        t = sum(max(a, 0) for a in new)
        step = cache.plan(layout, table, lengths, torch.tensor(new, dtype=torch.int32).cuda(), free, cursor,
                          tokens=t + 3, longest=max(new))
        step.check()
        lengths, cursor = step.lengths, step.cursor
        for store in stores:
            qkv = torch.randn(t + 3, 10, 64, generator=g).to(torch.bfloat16).cuda()
            q, k, v = qkv.split([6, 2, 2], dim=1)
            q = cache.append(store, step, k, v, query=q, rope=spec, norm_q=norm, norm_k=norm)
            out, lse = cache.attention(store, step, q, return_lse=True)
            step.check()
            kv, vv = (x.double().cpu() for x in store.read(torch.arange(pages, device="cuda")))
            want = law.attend_step(kv, vv, table.tolist(), held, new, q.cpu(), 16, 0.125)
            check_attention(out, lse, want, t, floor_of(400, store.value_exponent))
        held = [0 if a < 0 else x + a for x, a in zip(held, new)]
        assert lengths.tolist() == held
        free_now = sum(-(-x // 16) for x in held)
        assert int(cursor[1] - cursor[0]) == pages - free_now


def test_a_draft_over_a_pages_end_is_rejected_again_and_again():
    from cozy_runtime_b200 import cache

    layout, pages = cache.Layout(2, 1, 64, 16), 3
    table, free, new = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, -1, -1]], [0, 1, 2], [5]))
    lengths = reached = torch.tensor([15], dtype=torch.int32, device="cuda")
    cursor = torch.tensor([1, 3], device="cuda")
    for _ in range(50):
        step = cache.plan(layout, table, lengths, new, free, cursor, tokens=5, longest=5, reached=reached)
        step.check()
        reached, cursor = step.lengths, step.cursor
        held = table[0, :2].tolist()
        left = [int(free[i % pages]) for i in range(*cursor.tolist())]
        assert sorted(held + left) == [0, 1, 2] and step.slots.tolist()[1] == held[1] * 16
    step = cache.plan(layout, table, lengths, new - 6, free, cursor, tokens=5, longest=5, reached=reached)
    step.check()
    assert int(step.cursor[1] - step.cursor[0]) == pages and sorted(free.tolist()) == [0, 1, 2]


@pytest.mark.parametrize("page,longest", [(16, 40), (32, 7), (64, 200)])
def test_lengths_set_back_give_their_pages_back(page, longest):
    """Steps whose requests come, bring drafts, lose some of them (whole pages too) and go: each plan
    is the law's, eager and captured, the rows and the ring hold every page once, and the attention
    sees what was accepted."""
    import random

    from cozy_runtime_b200 import cache

    r, g = random.Random(page), torch.Generator().manual_seed(page)
    layout, requests, tokens = cache.Layout(4, 2, 64, page), 5, 300
    width = 6 * longest // page + 8
    pages = requests * width
    state = {"table": torch.full((requests, width), -1, dtype=torch.int32), "lengths": torch.zeros(requests, dtype=torch.int32),
             "new": torch.zeros(requests, dtype=torch.int32), "reached": torch.zeros(requests, dtype=torch.int32),
             "free": torch.randperm(pages, generator=g).to(torch.int32), "cursor": torch.tensor([0, pages])}
    state = {k: x.cuda() for k, x in state.items()}
    captured = {k: x.clone() for k, x in state.items()}

    def plan(s):
        return cache.plan(layout, s["table"], s["lengths"], s["new"], s["free"], s["cursor"], tokens=tokens,
                          longest=longest, reached=s["reached"])

    plan({k: x.clone() for k, x in state.items()})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured_plan = plan(captured)
    store = cache.Cache.empty(layout, pages)
    lengths = [0] * requests
    for i in range(40):
        reached = state["reached"].tolist()
        # what was rejected of the last step, and what this one brings
        lengths = [0 if not x else x - r.choice([0, 0, 1, r.randint(0, min(x, longest))]) for x in reached]
        new = [-1 if x and r.random() < 0.1 else r.choice([0, 1, r.randint(1, longest)]) if x + longest <= page * (width - 1) else -1
               for x in lengths]
        while sum(max(a, 0) for a in new) > tokens:
            new[r.randrange(requests)] = 0
        want = law.plan_step(state["table"].tolist(), lengths, new, state["free"].tolist(), state["cursor"].tolist(),
                             tokens=tokens, longest=longest, page=page, reached=reached)
        assert want["status"] == 0
        for s in (state, captured):
            s["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
            s["new"].copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        step = plan(state)
        for p, s in ((step, state), (captured_plan, captured)):
            p.check()
            for name in ("lengths", "starts", "cursor", "positions", "slots"):
                assert getattr(p, name).tolist() == want[name], (i, name)
            assert s["table"].tolist() == want["table"] and s["free"].tolist() == want["free"]
        head, tail = want["cursor"]
        rows = [p for row, x in zip(want["table"], want["lengths"]) for p in row[:-(-x // page)]]
        assert sorted(rows + [want["free"][j % pages] for j in range(head, tail)]) == list(range(pages))
        qkv = torch.randn(tokens, 8, 64, generator=g).to(torch.bfloat16).cuda()
        cache.append(store, step, qkv[:, 4:6], qkv[:, 6:])
        out, lse = cache.attention(store, step, qkv[:, :4], return_lse=True)
        if i % 8 == 7:
            kv = [values(c.cpu(), e.cpu()) for c, e in ((store.key, store.key_exponent), (store.value, store.value_exponent))]
            ref = law.attend_step(*kv, want["table"], lengths, new, qkv[:, :4].cpu(), page, 0.125)
            check_attention(out, lse, ref, sum(max(a, 0) for a in new), floor_of(pages * page, store.value_exponent))
        for p, s in ((step, state), (captured_plan, captured)):
            s["reached"].copy_(p.lengths)
            s["cursor"].copy_(p.cursor)


@pytest.mark.parametrize("reached,bit", [([-1, 40], 8), ([16 * 8, 40], 2), ([20, 2**31 - 1], 2)])
def test_plan_refuses_an_impossible_reach(reached, bit):
    from cozy_runtime_b200 import cache

    m = make([20, 40], [40, 2], 16, torch.Generator().manual_seed(2))
    t = {k: torch.tensor(m[k], dtype=torch.int64 if k == "cursor" else torch.int32, device="cuda")
         for k in ("table", "lengths", "new", "free", "cursor")}
    step = cache.plan(cache.Layout(4, 4, 64, 16), *t.values(), tokens=m["tokens"], longest=m["longest"],
                      reached=torch.tensor(reached, dtype=torch.int32, device="cuda"))
    assert int(step.status) & bit and step.starts.tolist() == [0, 0, 0]
    assert t["table"].tolist() == m["table"] and t["free"].tolist() == m["free"]


def test_a_captured_step_plans_anew_at_each_replay():
    from cozy_runtime_b200 import cache, rope

    g = torch.Generator().manual_seed(13)
    layout = cache.Layout(8, 2, 128, 32)
    spec = rope.llama(40 * 32, 128).to("cuda")
    for longest, news in ((1, ([1, 1, 0], [1, 1, 1], [0, 1, 1])), (100, ([100, 3, 1], [1, 0, 60], [7, 80, 0]))):
        T = 200
        m = make([40, 1000, 333], [longest] * 3, 32, g, spare=40)
        state = {k: torch.tensor(m[k], dtype=torch.int64 if k == "cursor" else torch.int32, device="cuda")
                 for k in ("table", "lengths", "new", "free", "cursor")}
        state["table"] = torch.cat([state["table"], state["table"].new_full((3, 4), -1)], dim=1)
        pages = len(m["free"])
        k, ke = fill(pages, 2, 32, 128, g)
        stores = [store_on_gpu(k, ke, k, ke) for _ in "ab"]
        qkv = torch.empty(T, 12, 128, dtype=torch.bfloat16, device="cuda")

        def step(store, s):
            p = cache.plan(layout, s["table"], s["lengths"], s["new"], s["free"], s["cursor"], tokens=T, longest=longest)
            q = cache.append(store, p, qkv[:, 8:10], qkv[:, 10:], query=qkv[:, :8], rope=spec)
            out = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device="cuda")
            cache.attention(store, p, q, out=out)
            s["lengths"].copy_(p.lengths)
            s["cursor"].copy_(p.cursor)
            return out, p

        captured, eager = ({k: v.clone() for k, v in state.items()} for _ in "ab")
        warm = {k: v.clone() for k, v in state.items()}
        warm["new"].zero_()
        step(cache.Cache.empty(layout, pages), warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured_out, captured_plan = step(stores[0], captured)
        for new in news:
            qkv.copy_(torch.randn(T, 12, 128, generator=g))
            for s in (captured, eager):
                s["new"].copy_(torch.tensor(new, dtype=torch.int32))
            graph.replay()
            out, p = step(stores[1], eager)
            p.check()
            captured_plan.check()
            assert torch.equal(captured["lengths"], eager["lengths"]) and torch.equal(captured["table"], eager["table"])
            assert torch.equal(captured_out, out)
            for a, b in ((stores[0].key, stores[1].key), (stores[0].value, stores[1].value)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert (out[sum(new):] == 0).all()


def test_norm_weights_as_models_ship_them():
    """bf16 and strided weights give what their fp32 values give, captured too; a weight that is not
    on the GPU is refused in a captured step, which goes on without it."""
    from cozy_runtime_b200 import cache, ulysses

    g = torch.Generator().manual_seed(16)
    layout = cache.Layout(4, 2, 128, 16)
    m = make([5, 40], [20, 3], 16, g)
    step, _ = on_gpu(m, layout)
    store = cache.Cache.empty(layout, step.pages)
    q, k = (torch.randn(23, h, 128, generator=g).to(torch.bfloat16).cuda() for h in (4, 2))
    weight = torch.randn(128, generator=g).to(torch.bfloat16)
    strided = weight.float().repeat_interleave(2).cuda()[::2]

    def append(w):
        return cache.append(store, step, k, k, query=q, norm_q=ulysses.Norm(w, 0.5), norm_k=ulysses.Norm(w, 0.5))

    want, codes = append(weight.float().cuda()), store.key.view(torch.uint8).clone()
    on_cuda = weight.cuda()
    for w in (on_cuda, strided, weight, weight.double()):
        assert torch.equal(append(w), want) and torch.equal(store.key.view(torch.uint8), codes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured"):
            append(weight)
        got = append(on_cuda)
    got.zero_()
    graph.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [[1] * 20, [60, 1, 9] + [1] * 17])
def test_calls_side_by_side_on_two_streams(new):
    """Two layers of one step on two streams: the same plan, caches of their own."""
    from cozy_runtime_b200 import cache

    g = torch.Generator().manual_seed(14)
    lengths = [137 * i % 900 for i in range(20)]
    m = make(lengths, new, 64, g)
    step, _ = on_gpu(m, cache.Layout(8, 2, 128, 64))
    made = []
    for _ in "ab":
        k, ke = fill(step.pages, 2, 64, 128, g)
        v, ve = fill(step.pages, 2, 64, 128, g)
        q = torch.randn(m["tokens"], 8, 128, generator=g).to(torch.bfloat16).cuda()
        made.append((store_on_gpu(k, ke, v, ve), q))
    alone = [cache.attention(s, step, q) for s, q in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    outs = [[], []]
    for _ in range(10):
        for i, (stream, (s, q)) in enumerate(zip(streams, made)):
            with torch.cuda.stream(stream):
                outs[i].append(cache.attention(s, step, q))
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        assert all(torch.equal(want, x) for x in got)


def test_a_step_that_brings_nothing_with_rows_to_spare():
    from cozy_runtime_b200 import cache

    layout = cache.Layout(4, 2, 64, 16)
    m = make([5, 0], [0, 0], 16, torch.Generator().manual_seed(1), tokens=7)
    for longest in (0, 1, 60):
        m["longest"] = longest
        step, _ = on_gpu(m, layout)
        store = cache.Cache.empty(layout, step.pages)
        q, k = (torch.ones(7, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
        assert cache.append(store, step, k, k, query=q, out=q).data_ptr() == q.data_ptr()
        out = cache.attention(store, step, q, out=torch.full_like(q, 3))
        assert (q == 1).all() and (out == 3).all()
        step.check()


def test_append_in_place():
    from cozy_runtime_b200 import cache, rope

    g = torch.Generator().manual_seed(2)
    layout = cache.Layout(6, 2, 128, 16)
    m = make([5, 40], [20, 3], 16, g)
    step, t = on_gpu(m, layout)
    store = cache.Cache.empty(layout, step.pages)
    spec = rope.llama(t["table"].shape[1] * 16, 128).to("cuda")
    qkv = torch.randn(23, 10, 128, generator=g).to(torch.bfloat16).cuda()
    want = cache.append(store, step, qkv[:, 6:8], qkv[:, 8:], query=qkv[:, :6], rope=spec)
    rest = qkv[:, 6:].clone()
    got = cache.append(store, step, qkv[:, 6:8], qkv[:, 8:], query=qkv[:, :6], rope=spec, out=qkv[:, :6])
    assert torch.equal(got, want) and torch.equal(qkv[:, 6:], rest)
    with pytest.raises(ValueError):
        cache.append(store, step, qkv[:, 6:8], qkv[:, 8:], query=qkv[:, :6], rope=spec, out=qkv[:, 1:7])


def test_append_refuses_an_out_over_keys_or_values():
    """Keys and values are read while queries are written: an `out` over a row of theirs is refused
    and nothing is stored; one between their rows is served."""
    from cozy_runtime_b200 import cache

    g = torch.Generator().manual_seed(2)
    layout = cache.Layout(4, 4, 64, 16)
    m = make([5, 40], [20, 3], 16, g)
    step, _ = on_gpu(m, layout)
    k0, ke0 = fill(step.pages, 4, 16, 64, g)
    store = store_on_gpu(k0, ke0, k0, ke0)
    qkv = torch.randn(23, 16, 64, generator=g).to(torch.bfloat16).cuda()
    q, k, v, rest = qkv.split(4, dim=1)
    was = qkv.clone()
    for out in (k, v, qkv[:, 6:10], qkv[:, 11:15], qkv[:, 5:13:2]):
        for query in (q, q.clone()):
            with pytest.raises(ValueError, match="out"):
                cache.append(store, step, k, v, query=query, out=out)
    assert torch.equal(qkv, was) and torch.equal(store.key.cpu().view(torch.uint8), k0.view(torch.uint8))
    got = cache.append(store, step, k, v, query=q.clone(), out=rest)
    assert torch.equal(got, q) and torch.equal(qkv[:, :12], was[:, :12])
    want = cache.append(store, step, k, v, query=q)
    assert torch.equal(want, q)


def test_an_empty_step():
    from cozy_runtime_b200 import cache

    layout = cache.Layout(4, 2, 64, 16)
    m = make([5, 0], [0, 0], 16, torch.Generator().manual_seed(1))
    step, _ = on_gpu(m, layout)
    store = cache.Cache.empty(layout, step.pages)
    q, k = (torch.empty(0, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    assert cache.append(store, step, k, k, query=q).shape == (0, 4, 64)
    out, lse = cache.attention(store, step, q, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    step.check()


def test_refusals():
    from cozy_runtime_b200 import _lib, cache, rope, ulysses
    import ctypes

    layout = cache.Layout(4, 2, 64, 16)
    m = make([20, 0], [1, 2], 16, torch.Generator().manual_seed(1))
    step, t = on_gpu(m, layout)
    store = cache.Cache.empty(layout, step.pages)
    q, k = (torch.zeros(3, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    bad = [
        lambda: cache.attention(store, step, q.float()),
        lambda: cache.attention(store, step, q[:2]),
        lambda: cache.attention(store, step, q.cpu()),
        lambda: cache.attention(store, step, q.transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: cache.attention(store, step, q, scale=0.0),
        lambda: cache.attention(store, step, q, scale=-1.0),
        lambda: cache.attention(store, step, q, scale=math.inf),
        lambda: cache.attention(store, step, q, out=q),
        lambda: cache.attention(store, step, q, out=q[:1].expand(3, 4, 64)),
        lambda: cache.attention(cache.Cache.empty(layout, step.pages + 1), step, q),
        lambda: cache.attention(cache.Cache.empty(cache.Layout(4, 2, 64, 32), step.pages), step, q),
        lambda: cache.append(store, step, k, q),
        lambda: cache.append(store, step, k, k, out=q),
        lambda: cache.append(store, step, k, k, norm_q=ulysses.Norm()),
        lambda: cache.append(store, step, k, k, query=q, norm_q=ulysses.Norm(torch.ones(32))),
        lambda: cache.append(store, step, k, k, query=q, rope=rope.llama(16, 64).to("cuda")),
        lambda: cache.append(store, step, k, k, query=q, rope=rope.llama(2000, 64)),
        lambda: cache.append(store, step, k, k, query=q, rope=rope.llama(2000, 128).to("cuda")),
        lambda: cache.Cache(store.key, store.value, store.key_exponent[:1], store.value_exponent),
        lambda: cache.Cache(store.key, store.value.bfloat16(), store.key_exponent, store.value_exponent),
        lambda: cache.Cache(store.key, store.value.cpu(), store.key_exponent, store.value_exponent),
        lambda: cache.plan(layout, t["table"], t["lengths"], t["new"], t["free"], t["cursor"].cpu(), tokens=3, longest=2),
        lambda: cache.plan(layout, t["table"].T, t["lengths"], t["new"], t["free"], t["cursor"], tokens=3, longest=2),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    # the C entries' own checks: a workspace too small, a pointer off its boundary
    lib = _lib.load()
    a = _lib.CacheAttend()
    a.query = a.out = q.data_ptr()
    a.query_strides[:] = a.out_strides[:] = (256, 64)
    a.scale, a.workspace, a.workspace_bytes = 1.0, q.data_ptr(), 0
    call = lambda: lib.cozy_cache_attention(ctypes.byref(step._c), ctypes.byref(store._c), ctypes.byref(a), 0)  # noqa: E731
    assert call() == _lib.INVALID_VALUE
    a.query = q.data_ptr() + 2
    assert call() == _lib.INVALID_VALUE
    torch.cuda.synchronize()
