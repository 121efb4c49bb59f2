"""An 8-bit paged key/value cache and the attention that reads it.

What a causal model needs behind its first pass over a prompt: the keys and values of running
requests, kept as e4m3 codes in pages of a pool, and attention of each step's new tokens over them.
A step is one `plan` for all layers, then for each layer an `append` and an `attention`:

    step = cache.plan(layout, table, lengths, new, free, cursor, tokens=T, longest=L)
    for store, layer in zip(stores, layers):
        query = cache.append(store, step, key, value, query=query, rope=tables, norm_q=..., norm_k=...)
        out = cache.attention(store, step, query)
    lengths, cursor = step.lengths, step.cursor

Where a step's tokens are drafts of which some are rejected, the next step starts from shorter
lengths and says how far the last one went, so that pages behind them come back:

    step = cache.plan(layout, table, step.lengths - rejected, new, free, step.cursor, tokens=T,
                      longest=L, reached=step.lengths)

The step's tokens are packed: request n's rows of `query`, `key` and `value` [tokens, heads,
head_dim] are `step.starts[n]` to `step.starts[n + 1]`. Lengths, page numbers and the plan's answer
stay on the GPU: no call here synchronizes (but an `append` whose norm weights are not on that GPU),
and a step can be captured into a CUDA graph (each replay plans anew from the lengths the tensors
then hold). A plan that cannot be served gives no
pages and its append and attention do nothing; `Plan.check()` says why. As with every torch tensor,
a plan or a cache used on another stream than the one that wrote it is ordered by the caller.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from dataclasses import dataclass

import torch
from torch import Tensor

from cozy_runtime_b200 import _lib
from cozy_runtime_b200.rope import RopeSpec
from cozy_runtime_b200.ulysses import Norm

PAGES = (16, 32, 64, 128)
MAX_REQUESTS = 8192
MAX_GROUP = 128
MAX_TOKENS = 2**30
#: the range of a block's exponent; larger magnitudes than 448 · 2^40 are stored as NaN
EXPONENT_RANGE = (-60, 40)

#: bits of a plan's status word
STATUS_NAMES = {
    1: "too few free pages",
    2: "a request longer than its row of the table",
    4: "more new tokens than `tokens`, or than `longest` in one request",
    8: "a negative length, new < -1, or an impossible ring cursor",
    16: "a page number outside the pool",
    32: "an on-chip wait timed out",
}


@dataclass(frozen=True)
class Layout:
    """The heads of every layer of a model and the tokens of a page."""

    heads_q: int
    heads_kv: int
    head_dim: int
    page: int = 64

    def __post_init__(self) -> None:
        if self.heads_kv < 1 or self.heads_q < 1 or self.heads_q % self.heads_kv:
            raise ValueError(f"{self.heads_q} query heads over {self.heads_kv} key heads")
        if self.group > MAX_GROUP:
            raise ValueError(f"a group of {self.group} query heads is not served ({MAX_GROUP} are)")
        if self.head_dim not in (64, 128):
            raise ValueError(f"head dim {self.head_dim} is not served (64 or 128)")
        if self.page not in PAGES:
            raise ValueError(f"pages of {self.page} tokens are not served ({PAGES})")

    @property
    def group(self) -> int:
        return self.heads_q // self.heads_kv


def _need(t: Tensor, name: str, dtype: torch.dtype, shape: tuple[int, ...]) -> None:
    if t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, not {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")


def _one_device(device: torch.device, index: int, *tensors: Tensor) -> None:
    """All on the CUDA device `index` (-1: not a CUDA device), which is `device`."""
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"operands are on {t.device} and on {device}")
    if index < 0:
        raise ValueError("operands are not on a CUDA device")


_HERE = contextlib.nullcontext()


def _on(index: int):
    """The device's context, entered only where another one is current."""
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


#: the current stream's handle without a Stream object around it: a decode step's calls are short
#: enough for the difference (1.3 us of about 17) to show
_stream = torch._C._cuda_getCurrentRawStream


class Cache:
    """One layer's blocks: `key` and `value` codes [pages, heads_kv, page, head_dim]
    (float8_e4m3fn) and a power of two for each block: `key_exponent`, `value_exponent` [pages,
    heads_kv] int8; a stored value is code · 2^exponent."""

    def __init__(self, key: Tensor, value: Tensor, key_exponent: Tensor, value_exponent: Tensor):
        if key.dim() != 4:
            raise ValueError("key has shape [pages, heads_kv, page, head_dim]")
        pages, heads, page, dim = key.shape
        _need(key, "key", torch.float8_e4m3fn, (pages, heads, page, dim))
        _need(value, "value", torch.float8_e4m3fn, (pages, heads, page, dim))
        _need(key_exponent, "key_exponent", torch.int8, (pages, heads))
        _need(value_exponent, "value_exponent", torch.int8, (pages, heads))
        for name, t in (("key", key), ("value", value), ("key_exponent", key_exponent),
                        ("value_exponent", value_exponent)):
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        self._index = key.get_device()
        _one_device(key.device, self._index, value, key_exponent, value_exponent)
        for name, t in (("key", key), ("value", value)):
            if t.data_ptr() % 128:
                raise ValueError(f"{name} must start on a 128-byte boundary")
        if pages * heads * page > 2**31 - 1:
            raise ValueError("a pool holds at most 2^31 - 1 rows")
        self.key, self.value = key, value
        self._blocks = pages, heads, page, dim
        self.key_exponent, self.value_exponent = key_exponent, value_exponent
        self._c = _lib.CacheStore(
            key.data_ptr(), value.data_ptr(), key_exponent.data_ptr(), value_exponent.data_ptr(),
            pages, heads, page, dim,
        )

    @classmethod
    def empty(cls, layout: Layout, pages: int, device: torch.device | str = "cuda") -> Cache:
        """A pool of `pages` pages (nothing in it has to start at a value)."""
        shape = (pages, layout.heads_kv, layout.page, layout.head_dim)
        key, value = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in "kv")
        exponents = torch.zeros(2, pages, layout.heads_kv, dtype=torch.int8, device=device)
        return cls(key, value, exponents[0], exponents[1])

    def read(self, pages: Tensor) -> tuple[Tensor, Tensor]:
        """What blocks of `pages` (page numbers, any shape) hold, as bf16 [*, heads_kv, page,
        head_dim] keys and values (exact: a code has 4 significant bits)."""
        out = []
        for codes, exponent in ((self.key, self.key_exponent), (self.value, self.value_exponent)):
            x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(torch.bfloat16)
            scale = ((exponent[pages].to(torch.int32) + 127) << 23).view(torch.float32)
            out.append(x * scale.to(torch.bfloat16)[..., None, None])
        return out[0], out[1]


class Plan:
    """A step's plan on the GPU. `lengths` [requests] int32 after the step, `cursor` [2] int64
    after it, `starts` [requests + 1] int32, `positions` [tokens] int32 and `slots` [tokens] int64
    (page number · page + row; both -1 in rows of nobody and of tokens whose page number is outside
    the pool), `status` [1] int32."""

    def __init__(self, layout: Layout, table: Tensor, lengths: Tensor, new: Tensor, free: Tensor,
                 cursor: Tensor, tokens: int, longest: int):
        n, page, device = lengths.shape[0], layout.page, table.device
        blocks = min(tokens, tokens // page + 2 * n)
        # `blocks` entries are 16 bytes and stand first, in front of the status word
        self._cuts = (4 * blocks, 1, n, n + 1, tokens), (2, 2 * n + 2, tokens)
        whole = torch.empty(4 * blocks + 2 * n + 2 + tokens, dtype=torch.int32, device=device)
        wide = torch.empty(2 * n + 4 + tokens, dtype=torch.int64, device=device)
        self._buffers = whole, wide
        self.layout, self.table, self.tokens, self.longest = layout, table, tokens, longest
        self.requests, self.pages = n, free.shape[0]
        self._blocks = self.pages, layout.heads_kv, page, layout.head_dim
        # what the calls of this step read must outlive them
        self._inputs = (lengths, new, free, cursor)
        at, at8 = whole.data_ptr(), wide.data_ptr()
        status = at + 16 * blocks
        self._c = _lib.CachePlan(
            lengths.data_ptr(), new.data_ptr(), table.data_ptr(),
            max(table.stride(0), table.shape[1]), free.data_ptr(), cursor.data_ptr(), n,
            table.shape[1], free.shape[0], page, tokens, longest, layout.group, blocks,
            status + 4, status + 4 + 4 * n, at8, status + 8 + 8 * n, at8 + 8 * (2 * n + 4), at,
            at8 + 16, status,
        )

    @functools.cached_property
    def _whole(self) -> tuple[Tensor, ...]:
        return self._buffers[0].split_with_sizes(self._cuts[0])

    @functools.cached_property
    def _wide(self) -> tuple[Tensor, ...]:
        return self._buffers[1].split_with_sizes(self._cuts[1])

    @property
    def status(self) -> Tensor:
        return self._whole[1]

    @property
    def lengths(self) -> Tensor:
        return self._whole[2]

    @property
    def starts(self) -> Tensor:
        return self._whole[3]

    @property
    def positions(self) -> Tensor:
        return self._whole[4]

    @property
    def cursor(self) -> Tensor:
        return self._wide[0]

    @property
    def slots(self) -> Tensor:
        return self._wide[2]

    def check(self) -> None:
        """Raise if the plan was refused, or if its calls so far met a page number outside the pool
        or a wait that timed out (synchronizes)."""
        word = int(self.status.item())
        if word:
            raise RuntimeError("cache plan: " + "; ".join(
                text for bit, text in STATUS_NAMES.items() if word & bit))


def _check_plan(table, lengths, new, free, cursor) -> tuple[int, int]:
    """(requests, width) of a plan's tensors, whose types and shapes fit each other."""
    if table.dim() != 2:
        raise ValueError(f"table has shape {tuple(table.shape)}, not [requests, width]")
    requests, width = table.shape
    for name, t, shape in (("table", table, None), ("lengths", lengths, (requests,)),
                           ("new", new, (requests,)), ("free", free, None)):
        if t.dtype != torch.int32:
            raise ValueError(f"{name} is {t.dtype}, not torch.int32")
        if shape is not None and t.shape != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")
    if cursor.dtype != torch.int64 or cursor.shape != (2,) or free.dim() != 1:
        raise ValueError("cursor is two int64 counts, free a ring of page numbers")
    stride = table.stride()
    if stride[1] != 1 or (requests > 1 and stride[0] < width):
        raise ValueError("rows of the table must be contiguous and apart")
    if not (lengths.is_contiguous() and new.is_contiguous() and free.is_contiguous()
            and cursor.is_contiguous()):
        raise ValueError("lengths, new, free and cursor must be contiguous")
    return requests, width


def plan(
    layout: Layout,
    table: Tensor,
    lengths: Tensor,
    new: Tensor,
    free: Tensor,
    cursor: Tensor,
    *,
    tokens: int,
    longest: int,
    reached: Tensor | None = None,
) -> Plan:
    """Gives pages to the requests of a step and says where its tokens go, in one launch.

    `table` [requests, width] int32: page numbers of each request, in order. `lengths` [requests]
    int32: tokens a request holds; `new` [requests] int32: tokens it brings (0: none; -1: it is
    finished and releases its pages, its length becomes 0). `free` [pages] int32: a ring of page
    numbers of which entries `cursor` = [head, tail) int64 (counted on, taken modulo pages) are
    free. Pages are given from the head in the requests' order; released ones go behind the tail
    and are given from the next plan on (every page of the row: who lets requests share pages counts
    them, and sets a length to 0 instead of finishing the request). `tokens`: rows of the step's tensors
    (at least the sum of `new`; rows behind it belong to nobody). `longest`: no request brings more
    than that. `reached` [requests] int32: the lengths that the last plan left (`Plan.lengths`),
    where `lengths` may have been set back since: a row holds the pages of the larger of the two,
    and those behind its tokens of this step are released like a finished request's. Without
    `reached` such pages would be lost; with it, a row handed on with a length of 0 needs 0 there
    too, and a step behind a refused one the refused one's `reached`.

    `table` and `free` are written in place, only where they held nothing; the new lengths and
    cursor are the plan's, so planning the same tensors again gives the same plan. A step that
    cannot be served (see `STATUS_NAMES`; a page number outside the pool among those to be released
    is one such) changes nothing: its plan has no rows."""
    requests, width = _check_plan(table, lengths, new, free, cursor)
    if not 1 <= requests <= MAX_REQUESTS:
        raise ValueError(f"{requests} requests are not served (1 to {MAX_REQUESTS})")
    if width < 1 or free.shape[0] < 1:
        raise ValueError("an empty table or pool")
    if free.shape[0] * layout.page >= 2**31:
        raise ValueError(f"a ring of {free.shape[0]} pages: a pool holds at most 2^31 - 1 rows")
    if width * layout.page > 2**30:
        raise ValueError("a request holds at most 2^30 tokens")
    if not 0 <= tokens <= MAX_TOKENS or not 0 <= longest < 2**31:
        raise ValueError("tokens must be a count up to 2^30, longest one below 2^31")
    if reached is not None:
        _need(reached, "reached", torch.int32, (requests,))
        if not reached.is_contiguous():
            raise ValueError("reached must be contiguous")
    index, device = table.get_device(), table.device
    _one_device(device, index, lengths, new, free, cursor)
    if reached is not None:
        _one_device(device, index, reached)
    made = Plan(layout, table, lengths, new, free, cursor, tokens, longest)
    made._inputs += (reached,)
    lib = _lib.load()
    with _on(index):
        if reached is None:
            code = lib.cozy_cache_plan(ctypes.byref(made._c), _stream(index))
        else:
            code = lib.cozy_cache_plan_back(ctypes.byref(made._c), reached.data_ptr(), _stream(index))
    _lib.check("cozy_cache_plan", code)
    return made


def _rows(t: Tensor, name: str, tokens: int, heads: int, dim: int) -> tuple[int, int]:
    """Element strides {token, head} of a step's [tokens, heads, head_dim] rows."""
    if t.dtype != torch.bfloat16 or t.shape != (tokens, heads, dim):
        _need(t, name, torch.bfloat16, (tokens, heads, dim))
    token, head, last = t.stride()
    if tokens <= 1:
        token = dim
    if heads == 1:
        head = dim
    if (last != 1 and tokens > 0) or (token | head) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: the head dimension must be contiguous and rows 16-byte aligned")
    return token, head


def _out(given: Tensor | None, like: Tensor) -> tuple[Tensor, tuple[int, int]]:
    tokens, heads, dim = like.shape
    if given is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format), (heads * dim, dim)
    token, head = _rows(given, "out", tokens, heads, dim)
    apart = head >= dim and token >= (heads - 1) * head + dim
    apart = apart or (token >= dim and head >= (tokens - 1) * token + dim)
    if tokens * heads > 1 and not apart:
        raise ValueError("rows of out overlap")
    return given, (token, head)


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether the spans of memory that two tensors lie in meet."""
    ends = [
        t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
        for t in (a, b)
    ]
    return a.numel() > 0 and a.data_ptr() < ends[1] and b.data_ptr() < ends[0]


def _rows_meet(a: Tensor, at: tuple[int, int], b: Tensor, bt: tuple[int, int]) -> bool:
    """Whether a row of `a` and a row of `b` [tokens, heads, head_dim] share memory; `at`, `bt`:
    their strides {token, head}. Slices of one packed projection lie in each other's span without
    sharing a row. Spans that meet count as sharing where the token strides differ or rows overlap
    their own tensor's."""
    (tokens, heads_a, dim), heads_b, token = a.shape, b.shape[1], at[0]
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    end_a = (tokens - 1) * token + (heads_a - 1) * at[1] + dim
    end_b = apart + (tokens - 1) * bt[0] + (heads_b - 1) * bt[1] + dim
    if tokens == 0 or apart >= end_a or end_b <= 0:
        return False
    if token != bt[0] or token < dim:
        return True
    behind = apart % token
    if behind >= (heads_a - 1) * at[1] + dim and behind + (heads_b - 1) * bt[1] + dim <= token:
        return False  # a token's rows of b between two tokens' of a
    for offset in {apart + j * bt[1] - i * at[1] for i in range(heads_a) for j in range(heads_b)}:
        # two rows that lie `offset` and some tokens apart, of which the nearest are looked at
        near = -offset // token
        for k in (near, near + 1):
            if -tokens < k < tokens and abs(offset + k * token) < dim:
                return True
    return False


def _fits(store: Cache, step: Plan) -> None:
    if store._blocks != step._blocks:
        raise ValueError(f"a cache of {store._blocks} [pages, heads, page, head_dim] "
                         f"and a plan over {step._blocks}")


def append(
    store: Cache,
    step: Plan,
    key: Tensor,
    value: Tensor,
    *,
    query: Tensor | None = None,
    rope: RopeSpec | None = None,
    norm_q: Norm | None = None,
    norm_k: Norm | None = None,
    out: Tensor | None = None,
) -> Tensor | None:
    """Stores a step's keys and values, and readies its queries, in one launch.

    `key`, `value` [tokens, heads_kv, head_dim] and `query` [tokens, heads_q, head_dim] bf16, head
    dimension contiguous. Query and key are normed (`norm_q`, `norm_k`: per-head RMSNorm) and
    rotated (`rope`: row = position in the request; the tables must reach the table's width) in
    fp32 and rounded once to bf16, the laws of `rope.head_norm_rope`. Norm weights are read as they
    are where they are fp32, contiguous and on the cache's GPU. Others are converted in every call,
    one more launch each; those on the host or another GPU are copied, which waits for the copy and
    is refused in a captured step. Returns the ready queries (`out`, or a new tensor; rows of nobody
    are left as they were), None without `query`. `out` is the query itself or shares no memory with
    it, and none with a row of `key` or `value`. A token whose page number is outside the pool (the
    plan's status says so) is not stored, its ready query is zero.

    A block's exponent is the smallest e ≥ -60 with max |x| ≤ 448 · 2^e over the tokens put into it
    so far, those among them that were rejected later. Until a token starts the block anew it only
    grows; the codes the block holds are then rounded to the grown scale, which is exact down to
    e4m3's subnormals. NaN, infinities and magnitudes over 448 · 2^40 are stored as NaN and leave the
    exponent alone. The same step can be appended again: it stores the same.
    A page that requests share must be full: two writers of one block are not ordered."""
    _fits(store, step)
    layout, index, tokens = step.layout, store._index, step.tokens
    device, dim = store.key.device, layout.head_dim
    _one_device(device, index, step.table, key, value)
    a = _lib.CacheAppend()
    a.key, a.value = key.data_ptr(), value.data_ptr()
    a.key_strides[:] = _rows(key, "key", tokens, layout.heads_kv, dim)
    a.value_strides[:] = _rows(value, "value", tokens, layout.heads_kv, dim)
    if query is not None:
        _one_device(device, index, query)
        a.query_strides[:] = _rows(query, "query", tokens, layout.heads_q, dim)
        given, (out, strides) = out, _out(out, query)
        if given is not None:
            _one_device(device, index, out)
            # in place is fine: a thread reads its rows before it writes them
            if _overlap(query, out) and (out.data_ptr() != query.data_ptr() or strides != tuple(a.query_strides)):
                raise ValueError("out overlaps the query and is not the query")
            # other blocks of threads read keys and values while these rows are written
            if _rows_meet(out, strides, key, tuple(a.key_strides)) or _rows_meet(out, strides, value, tuple(a.value_strides)):
                raise ValueError("out shares memory with the key or the value")
        a.query, a.out = query.data_ptr(), out.data_ptr()
        a.out_strides[:] = strides
    elif norm_q is not None or out is not None:
        raise ValueError("norm_q and out are the query's")
    if rope is not None:
        cos, sin, rotary = rope.cos, rope.sin, rope.rotary
        _one_device(device, index, cos, sin)
        if rotary < 0 or rotary > dim or rotary % 2:
            raise ValueError(f"{rotary} rotated channels of {dim}")
        if not rope.interleaved and rotary % 16:
            raise ValueError("split-half rotation serves multiples of 16 channels")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or not (
                cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("rotation tables are contiguous fp32")
        if rope.stride_token < 0 or rope.stride_channel < 0:
            raise ValueError("rotation tables are read forwards")
        columns = rotary // 2 if rope.interleaved else rotary
        last = (step._c.width * layout.page - 1) * rope.stride_token + (columns - 1) * rope.stride_channel
        if columns > 0 and last >= min(cos.numel(), sin.numel()):
            raise ValueError("the rotation tables end before the table's last position")
        a.rope = ctypes.pointer(rope.struct(0))
    weights = []
    for i, norm in enumerate((norm_q, norm_k)):
        if norm is None:
            continue
        a.normalize[i] = 1
        a.norm_offset[i], a.norm_eps[i] = float(norm.offset), float(norm.eps)
        if norm.weight is not None:
            if norm.weight.shape != (layout.head_dim,):
                raise ValueError("a norm's weight has one value for each channel of a head")
            if norm.weight.get_device() != index:
                with _on(index):
                    if torch.cuda.is_current_stream_capturing():
                        raise ValueError(f"a norm's weight on {norm.weight.device} in a captured step on {device}")
            w = norm.weight.to(device=device, dtype=torch.float32).contiguous()
            weights.append(w)
            a.norm_weight[i] = w.data_ptr()
    with _on(index):
        code = _lib.load().cozy_cache_append(
            ctypes.byref(step._c), ctypes.byref(store._c), ctypes.byref(a), _stream(index)
        )
    _lib.check("cozy_cache_append", code)
    return out


def attention(
    store: Cache,
    step: Plan,
    query: Tensor,
    *,
    scale: float | None = None,
    out: Tensor | None = None,
    return_lse: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """Causal attention of a step's queries [tokens, heads_q, head_dim] bf16 over their requests'
    blocks, the step's own tokens among them (`append` comes first): each row sees the keys up to
    its own position. Returns `out` (or a new tensor) of the query's shape, and with `return_lse`
    the natural log of each row's sum of exponentials [tokens, heads_q] fp32, by which outputs
    over parts of the keys can be joined. Rows of nobody are left as they were.

    Arithmetic: fp32 sums and softmax; weights are rounded to f16's 11 bits. A query row alone or
    among few (up to 24 rows a key head) is read exactly from 2^-28 of its largest value on; in a
    longer chunk, as two e4m3 parts, exactly from 2^-9.8 of it on and to 2^-17.8 of it below, so the
    same row may come out a little different there.

    What stands in blocks behind a row's last key, NaN among it, does not reach the row. A query row
    with an infinity or a NaN gives a row of NaN. Keys in a
    page whose number is outside the pool are left out, and the plan's status says so."""
    _fits(store, step)
    layout, index = step.layout, store._index
    _one_device(store.key.device, index, step.table, query)
    scale = 1.0 / math.sqrt(layout.head_dim) if scale is None else float(scale)
    if not 0.0 < scale < 2e38:
        raise ValueError("attention scale must be positive and finite")
    a = _lib.CacheAttend()
    a.query, a.scale = query.data_ptr(), scale
    a.query_strides[:] = _rows(query, "query", step.tokens, layout.heads_q, layout.head_dim)
    given, (out, strides) = out, _out(out, query)
    if given is not None:
        _one_device(store.key.device, index, out)
        if _overlap(query, out):
            raise ValueError("out overlaps the query")
    a.out = out.data_ptr()
    a.out_strides[:] = strides
    lse = None
    if return_lse:
        lse = query.new_empty((step.tokens, layout.heads_q), dtype=torch.float32)
        a.lse = lse.data_ptr()
    lib, plan_c, store_c = _lib.load(), ctypes.byref(step._c), ctypes.byref(store._c)
    with _on(index):
        size = lib.cozy_cache_workspace(plan_c, store_c)
        space = query.new_empty(size, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = space.data_ptr(), size
        code = lib.cozy_cache_attention(plan_c, store_c, ctypes.byref(a), _stream(index))
    _lib.check("cozy_cache_attention", code)
    return out if lse is None else (out, lse)
