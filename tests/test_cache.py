"""The 8-bit paged cache without a GPU: what is refused before anything is launched, and the oracle's own laws."""

import ctypes
import math

import pytest
import torch

from oracle import cache_oracle as law


def test_layout_refusals():
    from cozy_runtime_b200 import cache

    assert cache.Layout(32, 8, 128).group == 4
    for heads_q, heads_kv, dim, page in ((3, 2, 128, 64), (0, 1, 128, 64), (4, 0, 128, 64), (4, 2, 96, 64),
                                         (4, 2, 128, 48), (129, 1, 64, 64), (258, 2, 64, 16)):
        with pytest.raises(ValueError):
            cache.Layout(heads_q, heads_kv, dim, page)


def test_plan_refusals_before_the_device():
    from cozy_runtime_b200 import cache

    layout = cache.Layout(4, 2, 64, 16)
    good = {"table": torch.zeros(2, 3, dtype=torch.int32), "lengths": torch.zeros(2, dtype=torch.int32),
            "new": torch.ones(2, dtype=torch.int32), "free": torch.zeros(9, dtype=torch.int32),
            "cursor": torch.tensor([0, 9])}
    for change in ({"table": good["table"].long()}, {"table": good["table"][0]}, {"lengths": good["lengths"][:1]},
                   {"new": good["new"].float()}, {"cursor": good["cursor"].int()}, {"cursor": torch.zeros(3, dtype=torch.int64)},
                   {"free": torch.zeros(0, dtype=torch.int32)}, {"free": torch.zeros(9, 1, dtype=torch.int32)},
                   {"table": torch.zeros(2, 0, dtype=torch.int32)}, {"table": torch.zeros(3, 2, dtype=torch.int32).T},
                   {"table": torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)},
                   {"free": torch.zeros(18, dtype=torch.int32)[::2]}, {}):  # as they are: not on a GPU
        with pytest.raises(ValueError):
            cache.plan(layout, **(good | change), tokens=2, longest=1)
    for tokens, longest in ((-1, 1), (2, -1), (2**31, 1), (2, 2**31)):
        with pytest.raises(ValueError):
            cache.plan(layout, **good, tokens=tokens, longest=longest)
    wide = good | {"lengths": torch.zeros(8193, dtype=torch.int32), "new": torch.zeros(8193, dtype=torch.int32),
                   "table": torch.zeros(8193, 1, dtype=torch.int32)}
    with pytest.raises(ValueError, match="requests"):
        cache.plan(layout, **wide, tokens=2, longest=1)


def test_c_entries_refuse_without_a_gpu():
    """Bad structs come back as codes; nothing is launched and nothing throws."""
    from cozy_runtime_b200 import _lib

    lib = _lib.load()
    assert lib.cozy_cache_plan(None, 0) == _lib.INVALID_VALUE
    assert lib.cozy_cache_append(None, None, None, 0) == _lib.INVALID_VALUE
    assert lib.cozy_cache_attention(None, None, None, 0) == _lib.INVALID_VALUE
    assert lib.cozy_cache_workspace(None, None) == 0

    def plan(**change):
        p = _lib.CachePlan()
        fields = dict(requests=2, width=3, table_stride=3, pages=9, page=16, tokens=4, longest=2, group=2, max_blocks=4)
        for name in ("lengths", "added", "table", "free_ring", "cursor", "lengths_after", "starts", "cursor_after",
                     "positions", "slots", "blocks", "units", "status"):
            fields[name] = 1 << 20
        for name, value in (fields | change).items():
            setattr(p, name, value)
        return p

    whole = _lib.CacheStore(1 << 20, 1 << 20, 1 << 20, 1 << 20, 9, 2, 16, 64)
    bad_plan = (("cozy_cache_plan", ()),
                ("cozy_cache_append", (ctypes.byref(whole), ctypes.byref(_lib.CacheAppend()))),
                ("cozy_cache_attention", (ctypes.byref(whole), ctypes.byref(_lib.CacheAttend()))))
    for change, code in (({"requests": 0}, 1), ({"requests": 8193}, 1), ({"width": 0}, 1), ({"pages": 0}, 1),
                         ({"page": 48}, 801), ({"page": 0}, 801), ({"group": 0}, 1), ({"group": 129}, 801),
                         ({"tokens": -1}, 1), ({"longest": -1}, 1), ({"table_stride": 2}, 1), ({"max_blocks": 3}, 1),
                         ({"blocks": (1 << 20) + 8}, 1), ({"status": 0}, 1), ({"slots": 0}, 1),
                         ({"width": 1 << 28}, 1)):
        for entry, more in bad_plan:
            assert getattr(lib, entry)(ctypes.byref(plan(**change)), *more, 0) == code, (entry, change)

    def store(**change):
        s = _lib.CacheStore(1 << 20, 1 << 20, 1 << 20, 1 << 20, 9, 2, 16, 64)
        for name, value in change.items():
            setattr(s, name, value)
        return s

    a, x = _lib.CacheAppend(), _lib.CacheAttend()
    x.query = x.out = x.workspace = 1 << 20
    x.scale, x.workspace_bytes = 1.0, 1 << 40
    for change, code in (({"head_dim": 96}, 801), ({"pages": 8}, 1), ({"page": 32}, 1), ({"heads_kv": 0}, 1),
                         ({"key": (1 << 20) + 64}, 1), ({"value_exponent": 0}, 1)):
        assert lib.cozy_cache_append(ctypes.byref(plan()), ctypes.byref(store(**change)), ctypes.byref(a), 0) == code
        assert lib.cozy_cache_attention(ctypes.byref(plan()), ctypes.byref(store(**change)), ctypes.byref(x), 0) == code
    # more rows than a pool's coordinates reach
    assert lib.cozy_cache_append(ctypes.byref(plan(pages=1 << 27)), ctypes.byref(store(pages=1 << 27)),
                                 ctypes.byref(a), 0) == 1
    assert lib.cozy_cache_append(ctypes.byref(plan()), ctypes.byref(store()), ctypes.byref(a), 0) == 1  # no key
    for change in ({"scale": 0.0}, {"scale": -1.0}, {"scale": math.nan}, {"scale": math.inf}, {"query": 0},
                   {"out": (1 << 20) + 8}, {"workspace": (1 << 20) + 16}, {"workspace": 0}):
        y = _lib.CacheAttend.from_buffer_copy(x)
        for name, value in change.items():
            setattr(y, name, value)
        assert lib.cozy_cache_attention(ctypes.byref(plan()), ctypes.byref(store()), ctypes.byref(y), 0) == 1, change


def plan_struct(**change):
    from cozy_runtime_b200 import _lib

    p = _lib.CachePlan()
    fields = dict(requests=2, width=3, table_stride=3, pages=9, page=16, tokens=4, longest=2, group=2, max_blocks=4)
    for name in ("lengths", "added", "table", "free_ring", "cursor", "lengths_after", "starts", "cursor_after",
                 "positions", "slots", "blocks", "units", "status"):
        fields[name] = 1 << 20
    for name, value in (fields | change).items():
        setattr(p, name, value)
    return p


def test_more_tokens_than_a_grids_indices_reach_are_refused():
    """A thread's index is one of a row and of a row a grid behind: both stay in 31 bits."""
    from cozy_runtime_b200 import _lib, cache

    good = [torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32),
            torch.zeros(9, dtype=torch.int32), torch.tensor([0, 9])]
    for tokens in (2**30 + 1, 2**31 - 8192, 2**31 - 1):
        with pytest.raises(ValueError, match="2\\^30"):
            cache.plan(cache.Layout(4, 2, 64, 16), *good, tokens=tokens, longest=1)
    lib = _lib.load()
    for change in ({"tokens": 2**31 - 1, "max_blocks": 1 << 28}, {"tokens": 2**30 + 1, "max_blocks": 1 << 28},
                   {"max_blocks": 2**31 - 1}):
        assert lib.cozy_cache_plan(ctypes.byref(plan_struct(**change)), 0) == _lib.INVALID_VALUE, change


def test_a_ring_longer_than_any_pool_is_refused():
    """Also one whose length, cut to 32 bits, would be that of a short ring."""
    from cozy_runtime_b200 import _lib, cache

    for pages, page in ((2**27, 16), (2**24, 128), (2**32 + 9, 16), (2**31 + 5, 64)):
        free = torch.empty(pages, dtype=torch.int32, device="meta")  # a shape without memory
        with pytest.raises(ValueError, match="rows"):
            cache.plan(cache.Layout(4, 2, 64, page), torch.zeros(2, 3, dtype=torch.int32),
                       torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), free,
                       torch.tensor([0, 9]), tokens=2, longest=1)
        if pages < 2**31:
            assert _lib.load().cozy_cache_plan(ctypes.byref(plan_struct(pages=pages, page=page)), 0) == _lib.INVALID_VALUE


def test_rows_that_share_memory_are_found():
    """Against the sets of elements themselves, for slices of packed projections and odd strides."""
    import random

    from cozy_runtime_b200 import cache

    r, whole, met = random.Random(3), torch.zeros(6000, dtype=torch.bfloat16), 0
    index = torch.arange(6000)
    cases = []
    for _ in range(3000):
        dim, tokens = 8, r.randint(1, 5)
        token = 8 * r.randint(1, 30)
        shapes = [(tokens, r.randint(1, 4), dim) for _ in "ab"]
        strides = [(token, 8 * r.randint(0, 8), 1) for _ in "ab"]
        cases.append((shapes, strides, [8 * r.randint(0, 40) for _ in "ab"]))
    # q, k and v of a packed row, in its own place and over one another's
    cases += [([(4, 4, 8), (4, 2, 8)], [(64, 8, 1)] * 2, list(at)) for at in ((0, 32), (0, 48), (32, 32), (16, 32), (40, 32), (64, 48))]
    for shapes, strides, starts in cases:
        a, b = (torch.as_strided(whole, s, t, o) for s, t, o in zip(shapes, strides, starts))
        sets = [set(torch.as_strided(index, s, t, o).flatten().tolist()) for s, t, o in zip(shapes, strides, starts)]
        want = bool(sets[0] & sets[1])
        # strides as the calls take them: of one token or one head, any will do
        given = [(s[2] if s[0] <= 1 else t[0], s[2] if s[1] == 1 else t[1]) for s, t in zip(shapes, strides)]
        assert cache._rows_meet(a, given[0], b, given[1]) == want, (shapes, strides, starts)
        met += want
    assert 500 < met < 2500
    a, b = torch.as_strided(whole, (3, 2, 8), (64, 8, 1), 0), torch.as_strided(whole, (3, 2, 8), (80, 8, 1), 16)
    assert cache._rows_meet(a, (64, 8), b, (80, 8))  # not shown to be apart


def test_what_was_reached_is_checked_before_the_device():
    from cozy_runtime_b200 import _lib, cache

    good = [torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32),
            torch.zeros(9, dtype=torch.int32), torch.tensor([0, 9])]
    for reached in (torch.zeros(3, dtype=torch.int32), torch.zeros(2), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="reached"):
            cache.plan(cache.Layout(4, 2, 64, 16), *good, tokens=2, longest=1, reached=reached)
    lib = _lib.load()
    assert lib.cozy_cache_plan_back(ctypes.byref(plan_struct()), None, 0) == _lib.INVALID_VALUE
    assert lib.cozy_cache_plan_back(None, 1 << 20, 0) == _lib.INVALID_VALUE
    assert lib.cozy_cache_plan_back(ctypes.byref(plan_struct(requests=0)), 1 << 20, 0) == _lib.INVALID_VALUE


def test_the_law_keeps_every_page_when_drafts_are_rejected():
    table, free, cursor, reached = [[0, -1, -1]], [0, 1, 2], [1, 3], [15]
    for _ in range(20):
        made = law.plan_step(table, [15], [5], free, cursor, tokens=5, longest=5, page=16, reached=reached)
        assert made["status"] == 0
        table, free, cursor, reached = (made[k] for k in ("table", "free", "cursor", "lengths"))
        assert sorted(table[0][:2] + [free[i % 3] for i in range(*cursor)]) == [0, 1, 2]


def test_oracle_rounds_as_e4m3_does():
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(4000, generator=g) * 2.0 ** torch.randint(-12, 8, (4000,), generator=g),
                   torch.tensor([0.0, 448.0, -448.0, 2**-9, 2**-10, 3 * 2**-10, 17.0, 19.0, 2**-6])])
    x = x.clamp(-448, 448)
    want = x.to(torch.float8_e4m3fn).double()
    assert torch.equal(law.round_e4m3(x.double()), want)


def test_oracle_exponent_is_the_smallest_that_fits():
    for amax, e in ((0.0, -60), (1e-30, -60), (448.0, 0), (448.1, 1), (1.0, -8), (224.0, -1), (law.LARGEST, 40)):
        assert law.exponent(amax) == e
