"""A KV cache in pages that sequences share, held in 8 bits, and attention over it.

Beside the contiguous 16-bit caches of ``decode``, ``rotary`` and ``tree``: here the cache of
all layers is one pool of pages. A page holds ``page_size`` tokens of every KV head as float8
(e4m3) codes, with a power-of-two scale for each head's keys and values in it; a sequence is a
row of ``tables``, which names its pages, and of ``lengths``. A serving step is

    fork(cache, parents)                     # rows that end, start anew or continue others
    granted = reserve(cache, counts)         # pages for the next tokens, shared ones copied
    append(cache, k, v, layer=i)             # each layer: quantised into the pages
    out = prepared()                         # ``prepare(q, cache, layer=i)``
    cache.lengths += accepted                # what the program keeps of them

``compact`` moves the pages in use to the front of the pool. A page that several rows hold
(``refs`` counts them) is never written: ``reserve`` gives a row its own copy of the one it
goes on writing in. All calls but ``create`` only touch the device and can be captured;
``cache.lengths`` and the tensors given may be changed in place between calls and replays. Calls
on a cache, replays too, run one after the other; only ``prepared()`` ones may overlap.
Inference only: ``requires_grad`` inputs are refused.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

from . import _lib
from . import cache as _cache
from . import ops  # registers torch.ops.sfl

CODES = torch.float8_e4m3fn
PAGE_SIZES = (16, 32, 64, 128)
MAX_PAGES = 1 << 24
MAX_ROWS = 1024
MAX_TOKENS = _cache.MAX_DRAFTS
MAX_SPLITS = 128


@dataclass(eq=False)
class PagedCache:
    """The tensors of a paged cache, contiguous on one device; a program may allocate them itself.

    ``k`` ``[L, P, Hkv, page, D]`` and ``v`` ``[L, P, Hkv, D, page]`` float8_e4m3fn codes of L layers
    and P pages (of 16, 32, 64 or 128 tokens), ``k_scale`` and ``v_scale`` fp32 ``[L, P, Hkv]``:
    a value is its code times its page's scale, a power of two. ``tables`` int32 ``[B, M]``: the
    page of a row's tokens from ``place * page`` on, -1 for none. ``lengths`` int32 ``[B]``:
    committed tokens. ``refs`` int32 ``[P]``: in how many rows a page is, 0 for a free one.
    Up to 1024 rows. The tensors change in place; none is replaced.
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    tables: torch.Tensor
    lengths: torch.Tensor
    refs: torch.Tensor
    # What the calls ask for each time: the device's index, rows, KV heads, head dimension; their workspace.
    _index: int = field(init=False, repr=False)
    _shape: tuple = field(init=False, repr=False)
    _scratch: torch.Tensor = field(init=False, repr=False)
    _spans: tuple = field(init=False, repr=False)  # of memory that calls write: first and last address of each tensor

    def __setattr__(self, name, value):
        # What was checked stays; ``cache.lengths += n`` sets the tensor that it has changed in place.
        if self.__dict__.get(name, value) is not value:
            raise AttributeError(f"{name} of a paged cache is changed in place, not replaced")
        object.__setattr__(self, name, value)

    def __post_init__(self):
        k, tables = self.k, self.tables
        if k.ndim != 5 or 0 in k.shape or tables.ndim != 2 or 0 in tables.shape:
            raise ValueError("k must be [L, P, Hkv, page, D] and tables [B, M], not empty")
        layers, pages, heads, page, dim = k.shape
        if page not in PAGE_SIZES:
            raise ValueError("supported page sizes are 16/32/64/128")
        if dim not in _cache.SUPPORTED_DIMS:
            raise ValueError("supported head dimensions are 16/32/64/128")
        if pages > MAX_PAGES:
            raise ValueError(f"at most {MAX_PAGES} pages are supported")
        if tables.shape[0] > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} rows are supported")
        if tables.shape[1] * page > _cache.MAX_ROWS:
            raise ValueError(f"a row must have at most {_cache.MAX_ROWS} slots")
        index = k.get_device()
        for name, dtype, shape in (("k", CODES, k.shape), ("v", CODES, (layers, pages, heads, dim, page)),
                                   ("k_scale", torch.float32, (layers, pages, heads)),
                                   ("v_scale", torch.float32, (layers, pages, heads)),
                                   ("tables", torch.int32, tables.shape), ("lengths", torch.int32, tables.shape[:1]),
                                   ("refs", torch.int32, (pages,))):
            _cache.check_vector("paged cache", name, getattr(self, name), dtype, shape, index)
        if k.data_ptr() % 16 or self.v.data_ptr() % 16:
            raise ValueError("k and v must be 16-byte aligned")
        held = (k, self.v, self.k_scale, self.v_scale, tables, self.lengths, self.refs)
        self._spans = tuple(sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in held if t.data_ptr()))
        if any(last > start for (_, last), (start, _) in zip(self._spans, self._spans[1:])):
            raise ValueError("the tensors of a cache must not share memory")
        self._index = index
        self._shape = (tables.shape[0], heads, dim)
        self._scratch = torch.empty(4 + 2 * max(pages, tables.shape[0]), dtype=torch.int32, device=k.device)

    def __reduce__(self):  # copies and loaded caches are looked at anew: their tensors are others
        return PagedCache, (self.k, self.v, self.k_scale, self.v_scale, self.tables, self.lengths, self.refs)

    @property
    def layers(self) -> int:
        return self.k.shape[0]

    @property
    def page_size(self) -> int:
        return self.k.shape[3]

    @property
    def capacity(self) -> int:
        """Slots of a row."""
        return self.tables.shape[1] * self.k.shape[3]


def create(batch, capacity, kv_heads, head_dim, pages, *, layers=1, page_size=64, device="cuda") -> PagedCache:
    """A cache of ``batch`` empty rows of up to ``capacity`` tokens over ``pages`` free pages."""
    for name, value in (("batch", batch), ("capacity", capacity), ("kv_heads", kv_heads), ("pages", pages),
                        ("layers", layers)):
        if type(value) is not int or value < 1:
            raise ValueError(f"{name} must be a positive integer")
    if page_size not in PAGE_SIZES:
        raise ValueError("supported page sizes are 16/32/64/128")

    def zeros(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype, device=device)

    codes = (zeros(layers, pages, kv_heads, *rows, dtype=torch.uint8).view(CODES)
             for rows in ((page_size, head_dim), (head_dim, page_size)))
    scales = (zeros(layers, pages, kv_heads, dtype=torch.float32) for _ in range(2))
    return PagedCache(*codes, *scales, zeros(batch, -(-capacity // page_size)) - 1, zeros(batch), zeros(pages))


def _check_cache(operator, cache):
    if not isinstance(cache, PagedCache):
        raise TypeError(f"{operator}: cache must be a PagedCache")
    return cache._index


def _check_apart(cache, name, t):
    """A vector that a call reads while it writes the cache."""
    first = t.data_ptr()
    last = first + 4 * t.numel()
    for start, end in cache._spans:
        if first < end and start < last:
            raise ValueError(f"{name} must not share memory with the cache (its lengths, tables or pages)")


def _check_layer(cache, layer):
    if type(layer) is not int or not 0 <= layer < cache.k.shape[0]:
        raise ValueError("layer must be an integer in [0, layers)")


def fork(cache, parents) -> None:
    """All at once, row b becomes what row ``parents[b]`` was (int32 ``[B]``), in place.

    It leaves its own pages and shares those that the parent's committed tokens are in, with
    the parent's length. ``parents[b] == b``: the row stays; -1: it is freed. (Entries that name
    no row stay, too.) One call reorders, copies and frees any rows.
    """
    index = _check_cache("fork", cache)
    _cache.check_vector("fork", "parents", parents, torch.int32, cache.lengths.shape, index)
    _check_apart(cache, "parents", parents)
    _cache.check_device(index)
    written = (cache.tables, cache.lengths, cache.refs)
    ops.dispatch(torch.ops.sfl.page_fork, (parents, *written), written, cache.k.shape[3], checked=True)


def reserve(cache, counts) -> torch.Tensor:
    """Pages for the next ``counts[b]`` tokens of each row (int32 ``[B]``); returns how many are granted.

    One row after another, place by place: a place that the tokens will be written to and
    that has no page, or one that other rows hold too, gets the lowest free page; where the
    shared one holds committed tokens of the row it is copied, in all layers. (Of several rows
    that go on writing in one page the last keeps it.) ``granted`` int32 ``[B]``, a new tensor:
    the tokens that have a place of their own; less than asked for where the pool or the row
    is full.
    """
    index = _check_cache("reserve", cache)
    _cache.check_vector("reserve", "counts", counts, torch.int32, cache.lengths.shape, index)
    _check_apart(cache, "counts", counts)
    _cache.check_device(index)
    _lib.lib()  # fail here, before allocating, if the library is not built
    granted = torch.empty_like(cache.lengths)
    written = (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.tables, cache.refs, granted, cache._scratch)
    ops.dispatch(torch.ops.sfl.page_reserve, (cache.lengths, counts, *written), written, checked=True)
    return granted


def compact(cache) -> torch.Tensor:
    """Move the pages in use to the front of the pool, in place; returns how many they are (int32 ``[1]``).

    Pages past that number, ascending, go into the free ones below it, ascending, in all
    layers; ``tables`` and ``refs`` follow. Pages in front stay where they are.
    """
    index = _check_cache("compact", cache)
    _cache.check_device(index)
    _lib.lib()
    used = torch.empty(1, dtype=torch.int32, device=cache.k.device)
    written = (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.tables, cache.refs, used, cache._scratch)
    ops.dispatch(torch.ops.sfl.page_compact, written, written, checked=True)
    return used


def append(cache, k, v, *, layer=0, counts=None) -> None:
    """Quantise new tokens ``k``, ``v`` ``[B, Hkv, T, D]`` (fp16, bf16 or fp32 views) into a layer's pages, in place.

    Token t of row b goes to slot ``lengths[b] + t``; those from ``counts[b]`` on (int32 ``[B]``)
    are padding. ``lengths`` is not changed. Tokens whose place has no page, or one that other
    rows hold, are left out: ``reserve`` comes first. For each page and head the scale becomes
    the least power of two (from 2^-100 on) under which the new values fit codes of up to 448;
    where the page holds committed tokens it does not become smaller, and where it grows their
    codes are rounded again under the new one, which stays if the new tokens are rejected. Infinities, NaN and magnitudes from 2^127 on
    become NaN. Tokens and counts must not share memory with the pages and scales of the layer.
    """
    index = _check_cache("append", cache)
    if _cache.check_rows("append", ("k", "v"), (k, v)) != index:
        _cache.check_device(-1)
    _check_layer(cache, layer)
    shape = k.shape
    if v.shape != shape or (shape[0], shape[1], shape[3]) != cache._shape:
        raise ValueError("k, v and the cache must agree in rows, heads and head dimension")
    if counts is not None:
        _cache.check_vector("append", "counts", counts, torch.int32, cache.lengths.shape, index)
    _cache.check_device(index)
    written = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    ops.dispatch(torch.ops.sfl.page_append, (k, v, cache.tables, cache.lengths, counts, cache.refs, *written), written,
                 layer, checked=True)


def auto_splits(batch: int, kv_heads: int, capacity: int, rows: int, dim: int, dtype: torch.dtype,
                window_left: int | None = None) -> int:
    """Workgroups that share a KV head's slots, for ``rows`` query rows over each (new tokens times
    query heads of the KV head).

    A workgroup takes 16 rows, or in bf16 32 of up to 64, or 128 of more than 64 (16-bit heads of
    64 and 128). About as many as run at once, 256; 512 of the last kind, and where sequences
    may differ in length, so that long ones have more of them. About 1024 slots each (to the
    nearest number of splits: 768 at least), at most 64 splits. Measured, us at 1 / 2 / 4 / 8 splits, bf16, 8 KV heads of 128: 32 rows of 8000 slots
    84 / 89 / 92 / -, of 1K to 8K 64 / 56 / 60 / 68; 16 of 4000 29 / 27 / 28 / 31, of 2K to 16K 99 / 64 /
    52 / 56; 8 of 4000 28 / 21 / 17 / 19; 8 of 1000 11.6 / 13.9 / 14.2 / -; 16 heads of 64 with a window
    of 4095 24 / 29 / 33 / 45; 1 of 131072 at 16 / 32 / 64 splits 76 / 52 / 55; 27 tokens of 4 heads
    over 8 of 1K to 8K 206 / 113 / 65 / 50.
    """
    block, blocks, reach = _blocks(batch, kv_heads, capacity, rows, dim, dtype, window_left)
    target = 512 if block == 128 or rows <= 16 and batch > 1 and window_left is None else 256
    return max(1, min(64, round(target / blocks), round(reach / 1024)))


def _blocks(batch, kv_heads, capacity, rows, dim, dtype, window_left):
    """Query rows of a workgroup, such blocks of all sequences, slots that a token may see."""
    tiled = dtype != torch.float32 and dim >= 64
    block = 128 if tiled and rows > 64 else 32 if tiled and dtype == torch.bfloat16 and rows > 32 else 16
    return (block, batch * kv_heads * math.ceil(rows / block),
            capacity if window_left is None else min(capacity, window_left + 1))


def auto_most_splits(splits: int, batch: int, kv_heads: int, capacity: int, rows: int, dim: int, dtype: torch.dtype,
                     window_left: int | None = None) -> int:
    """Those that sequences may have that hold far more than their share of the batch's slots, where
    ``splits`` could leave their workgroups more than 8192 slots each (4096 and 2048 for blocks of 32
    and 128 rows): with 256 more workgroups for the call, of heads and blocks of such sequences.
    """
    block, blocks, reach = _blocks(batch, kv_heads, capacity, rows, dim, dtype, window_left)
    if batch == 1 or reach <= splits * {16: 8192, 32: 4096, 128: 2048}[block]:
        return splits
    return max(splits, min(64, splits + 256 * batch // blocks))


@dataclass
class PreparedPaged:
    q: torch.Tensor
    cache: PagedCache
    counts: torch.Tensor | None
    partial_max: torch.Tensor
    partial_sum: torch.Tensor
    partial_output: torch.Tensor
    output: torch.Tensor
    lse: torch.Tensor
    layer: int
    window_left: int
    splits: int
    most_splits: int
    scale: float

    def __call__(self) -> torch.Tensor:
        """The output ``[B, Hq, T, D]``, overwritten by every call; ``lse`` goes with it."""
        c = self.cache
        written = (self.partial_max, self.partial_sum, self.partial_output, self.output, self.lse)
        ops.dispatch(torch.ops.sfl.page_attention,
                     (self.q, c.k, c.v, c.k_scale, c.v_scale, c.tables, c.lengths, self.counts, *written), written,
                     self.layer, self.window_left, self.splits, self.most_splits, self.scale, checked=True)
        return self.output

    @property
    def scratch_bytes(self) -> int:
        return sum(x.numel() * x.element_size() for x in (self.partial_max, self.partial_sum, self.partial_output))


def prepare(q, cache, *, layer=0, counts=None, window_left=None, splits=None, scale=None) -> PreparedPaged:
    """Validate and allocate, then return a reusable operation: attention of new tokens over a layer's pages.

    ``q`` ``[B, Hq, T, D]`` (fp16, bf16 or fp32, T at most 128) may be a strided view with 16-byte
    aligned rows. New token t of row b is in slot ``lengths[b] + t`` (``append``) and sees the slots
    up to that one that have a page; with ``window_left`` only the last ``window_left`` before it,
    and itself. ``counts`` int32 ``[B]``: tokens in use; the rows of the others are zeros with an
    ``lse`` (fp32 ``[B, Hq, T]``) of -inf, as are those of tokens that see nothing or have no slot. What
    a token does not see has no part in its row, NaN included. Scores and sums are fp32, and
    no code is rounded again: probabilities, of up to 2^8 before the division by their sum, are rounded
    to two bf16 pieces (off by 2^-16) for 16-bit ``q``, to three for fp32. ``splits``: workgroups that
    share a KV head's slots, 1 to 128; by default as many as the sizes ask for, and more for sequences
    far longer than the others. Like ``tree.PreparedTree`` the operation owns its scratch and output
    and holds its inputs by reference; concurrent calls on one race.
    """
    if splits is not None and (type(splits) is not int or not 1 <= splits <= MAX_SPLITS):
        raise ValueError("splits must be an integer in [1, 128]")
    if window_left is not None and (type(window_left) is not int or window_left < 0):
        raise ValueError("window_left must be a non-negative integer or None")
    index = _check_cache("paged attention", cache)
    if _cache.check_rows("paged attention", ("q",), (q,)) != index:
        _cache.check_device(-1)
    _check_layer(cache, layer)
    batch, heads, tokens, dim = q.shape
    rows, kv_heads, width = cache._shape
    if batch != rows or dim != width:
        raise ValueError("q and the cache must agree in rows and head dimension")
    _cache.check_heads(heads, kv_heads)
    if tokens > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} new tokens are supported")
    if counts is not None:
        _cache.check_vector("paged attention", "counts", counts, torch.int32, (batch,), index)
    scale = dim ** -0.5 if scale is None else scale
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    _cache.check_device(index)
    _lib.lib()  # fail here, before allocation, if the library is not built
    most, group_rows = splits, tokens * (heads // kv_heads)
    if splits is None:
        size = batch, kv_heads, cache.capacity, group_rows, dim, q.dtype, window_left
        splits = auto_splits(*size)
        most = auto_most_splits(splits, *size)
    window = -1 if window_left is None else min(window_left, cache.capacity)
    parts = batch * heads * tokens * splits if most > 1 else 0
    if most > splits:
        parts += 256 * (128 if group_rows > 64 else 32) + group_rows
    maximum = torch.empty(parts, device=q.device, dtype=torch.float32)
    numerator = torch.empty((parts, dim), device=q.device, dtype=torch.float32)
    lse = torch.empty((batch, heads, tokens), device=q.device, dtype=torch.float32)
    return PreparedPaged(q, cache, counts, maximum, torch.empty_like(maximum), numerator, torch.empty_like(q), lse,
                         layer, window, splits, most, float(scale))


def attend(q, cache, *, layer=0, counts=None, window_left=None, splits=None, scale=None):
    """``prepare`` and compute once on the current stream: ``(out, lse)``."""
    op = prepare(q, cache, layer=layer, counts=counts, window_left=window_left, splits=splits, scale=scale)
    return op(), op.lse
