"""Attention of drafted tokens over a KV cache, and what verification does with them.

Next to ``decode`` (one query a sequence, all of a row's keys): here a sequence brings
``T`` drafted tokens at once, whose keys and values are in the cache behind its
committed ones, and each draft sees the committed keys and those drafts its mask names.
A token tree (``ancestor_mask``), a chain (no mask) and a single token (``T = 1``) are all
of this form. A step of speculative decoding on a cache is

    q = rotary.rotate_append(...)            # drafts' k, v into slots lengths .. lengths + T - 1
    out = prepared()                         # ``prepare(q, k, v, lengths, mask)``
    ...                                      # the program verifies: path, accepted
    prepared.accumulate(weights, rows)       # where an eviction will ask for weights
    lengths = accept(k, v, lengths, path, accepted, weights=weights)

The prepared operation owns its fp32 scratch, output and ``lse`` and holds its inputs by
reference, like ``decode.PreparedDecode``; ``lengths``, ``counts`` and ``mask`` may be
changed in place between calls and graph replays; concurrent calls on one prepared
operation race on its scratch. Inference only: ``requires_grad`` inputs are refused.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from . import cache
from . import ops  # registers torch.ops.sfl

MAX_DRAFTS = cache.MAX_DRAFTS
MAX_SPLITS = 128


def ancestor_mask(parents: torch.Tensor) -> torch.Tensor:
    """The bool mask ``[..., T, T]`` of token trees: draft t sees itself and its ancestors.

    ``parents`` ``[..., T]`` holds each draft's parent draft, -1 for those that follow the
    committed text; a parent comes before its children. The check of that is read back
    (so the call stays outside graph captures), and the rows are formed one after another
    by elementary operations, some ten a draft.
    """
    if parents.ndim < 1 or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError("parents must be an integer tensor [..., T]")
    tokens = parents.shape[-1]
    order = torch.arange(tokens, device=parents.device)
    if bool(((parents < -1) | (parents >= order)).any()):
        raise ValueError("a draft's parent must be -1 or an earlier draft")
    mask = torch.eye(tokens, dtype=torch.bool, device=parents.device).expand(*parents.shape, tokens).clone()
    for t in range(1, tokens):
        parent = parents[..., t : t + 1, None].long()
        above = mask.gather(-2, parent.clamp(min=0).expand(*parent.shape[:-1], tokens))
        mask[..., t : t + 1, :] |= above & (parent >= 0)
    return mask


def _check(operator, names, rows, lengths, mask, counts):
    """What the calls on drafts ask of rows (q, k and, where it is read, v); returns the mask as [B, T, T] and the device index."""
    index = cache.check_rows(operator, names, rows)
    batch, heads, tokens, dim = rows[0].shape
    kb, kv_heads, _, kd = rows[1].shape
    if kb != batch or kd != dim:
        raise ValueError("q and k must agree in batch and head dimension")
    cache.check_heads(heads, kv_heads)
    if tokens > MAX_DRAFTS:
        raise ValueError(f"at most {MAX_DRAFTS} drafted tokens are supported")
    cache.check_vector(operator, "lengths", lengths, torch.int32, (batch,), index)
    if counts is not None:
        cache.check_vector(operator, "counts", counts, torch.int32, (batch,), index)
    if mask is None:
        mask = torch.ones(tokens, tokens, dtype=torch.bool, device=rows[0].device).tril_()
    shape = mask.shape
    if mask.dtype is not torch.bool or shape != (batch, tokens, tokens) and shape != (tokens, tokens):
        raise ValueError("mask must be a bool tensor [T, T] or [B, T, T]")
    if mask.get_device() != index:
        cache.check_device(-1)
    return mask if len(shape) == 3 else mask.expand(batch, tokens, tokens), index


def _scale(scale, dim):
    scale = dim ** -0.5 if scale is None else scale
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    return float(scale)


def auto_splits(batch: int, kv_heads: int, capacity: int, rows: int, dim: int, dtype: torch.dtype) -> int:
    """Workgroups that share a KV head's keys, for ``rows`` query rows over each (drafts times
    query heads of the KV head).

    A workgroup takes up to 128 rows of 16-bit heads of 64 and 128, 64 of shorter ones, and
    in fp32 32, or 16 of heads of 128. As many workgroups as run at once: 512, but 256 (one
    to a CU, by LDS) for up to 64 rows of the first kind; at most 32 splits, as the merge
    reads them all, of at least 128 keys. Measured, us at 8 / 16 / 32 / 64 splits: B=1 Hkv=4
    N=65536 512 rows 155 / 98 / 94 / 110; B=4 Hkv=4 D=64 N=16384 64 rows 26 / 20 / 22 / 27;
    B=1 Hkv=4 N=8192 32 rows 19 / 16 / 16 / 18; B=8 Hkv=8 N=8191 108 rows 71 / 87 / 112 /
    164; fp32 B=2 Hkv=4 D=128 N=8192 64 rows 39 / 37 / 43 / 56. A few rows over one long cache
    (us at 16 / 32 / 64 / 128, 8 rows): Hkv=4 N=65536 40 / 29 / 32 / 38, N=131072 70 / 50 / 51 / 56;
    Hkv=1 N=65536 40 / 27 / 22 / 22, N=131072 69 / 41 / 29 / 27, so with one or two KV heads
    ``splits=64`` is the better choice there.
    """
    tiled = dtype != torch.float32 and dim >= 64
    block = 128 if tiled else 64 if dtype != torch.float32 else 16 if dim == 128 else 32
    blocks = batch * kv_heads * math.ceil(rows / block)
    target = 256 if tiled and rows <= 64 else 512
    return max(1, min(32, round(target / blocks), math.ceil(capacity / 128)))


@dataclass
class PreparedTree:
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    lengths: torch.Tensor
    mask: torch.Tensor
    counts: torch.Tensor | None
    partial_max: torch.Tensor
    partial_sum: torch.Tensor
    partial_output: torch.Tensor
    output: torch.Tensor
    lse: torch.Tensor
    splits: int
    scale: float

    def __call__(self) -> torch.Tensor:
        """The output ``[B, Hq, T, D]``, overwritten by every call; ``lse`` goes with it."""
        written = (self.partial_max, self.partial_sum, self.partial_output, self.output, self.lse)
        ops.dispatch(torch.ops.sfl.tree_attention,
                     (self.q, self.k, self.v, self.lengths, self.mask, self.counts, *written), written, self.splits,
                     self.scale, checked=True)
        return self.output

    def accumulate(self, weights: torch.Tensor, rows: torch.Tensor | None = None) -> torch.Tensor:
        """``accumulate`` with the operands and ``lse`` of the last call."""
        return accumulate(self.q, self.k, self.lse, weights, self.lengths, self.mask, counts=self.counts, rows=rows,
                          scale=self.scale)

    @property
    def scratch_bytes(self) -> int:
        return sum(x.numel() * x.element_size() for x in (self.partial_max, self.partial_sum, self.partial_output))


def prepare(q, k, v, lengths, mask=None, *, counts=None, splits=None, scale=None) -> PreparedTree:
    """Validate and allocate outside capture, then return a reusable operation.

    ``q`` ``[B, Hq, T, D]`` (T at most 128) and ``k``, ``v`` ``[B, Hkv, N, D]`` may be strided
    views with 16-byte aligned rows. ``lengths`` int32 ``[B]`` counts the *committed* keys;
    draft j of sequence b has its key and value in slot ``lengths[b] + j``. ``mask`` bool
    ``[T, T]`` or ``[B, T, T]``: whether draft t sees draft j, itself included (default: all
    up to itself). ``counts`` int32 ``[B]``: drafts in use; the rows of the others are zeros
    with an ``lse`` of -inf, as are those of drafts that see nothing. What a draft does not
    see has no part in its row, NaN included; an infinite value that it sees with a weight too
    small for the products (in fp16 below 2^-36 of the row's largest) can give NaN.
    ``splits``: workgroups that share a KV head's keys, 1 to 128 (default by size).
    """
    if splits is not None and (type(splits) is not int or not 1 <= splits <= MAX_SPLITS):
        raise ValueError("splits must be an integer in [1, 128]")
    mask, index = _check("tree attention", ("q", "k", "v"), (q, k, v), lengths, mask, counts)
    batch, heads, tokens, dim = q.shape
    kv_heads, capacity = k.shape[1:3]
    if v.shape != k.shape:
        raise ValueError("k and v must have the same [B, Hkv, N, D] shape")
    scale = _scale(scale, dim)
    cache.check_device(index)
    used = tokens if counts is None else counts
    if counts is not None and not bool(((counts >= 0) & (counts <= tokens)).all()):
        raise ValueError("each count must be in [0, T]")
    if not bool(((lengths >= 0) & (lengths <= capacity - used)).all()):
        raise ValueError("each length must be in [0, cache capacity - drafts]")
    _lib.lib()  # fail here, before allocation, if the library is not built
    if splits is None:
        splits = auto_splits(batch, kv_heads, capacity, tokens * (heads // kv_heads), dim, q.dtype)
    maximum = torch.empty((batch, heads, tokens, splits if splits > 1 else 0), device=q.device, dtype=torch.float32)
    numerator = torch.empty((*maximum.shape, dim), device=q.device, dtype=torch.float32)
    lse = torch.empty((batch, heads, tokens), device=q.device, dtype=torch.float32)
    return PreparedTree(q, k, v, lengths, mask, counts, maximum, torch.empty_like(maximum), numerator,
                        torch.empty_like(q), lse, splits, scale)


def attend(q, k, v, lengths, mask=None, *, counts=None, splits=None, scale=None):
    """``prepare`` and compute once on the current stream, outside captures: ``(out, lse)``."""
    op = prepare(q, k, v, lengths, mask, counts=counts, splits=splits, scale=scale)
    return op(), op.lse


def accumulate(q, k, lse, weights, lengths, mask=None, *, counts=None, rows=None, scale=None):
    """Add the drafts' attention weights up by slot, in place: ``weights`` fp32 ``[B, Hkv, N]``.

    Every slot gains ``exp(scale * q . k - lse)`` of each draft that sees it, over the query
    heads of its KV head; ``lse`` fp32 ``[B, Hq, T]`` is that of the attention call. ``rows``
    bool ``[B, T]``: the drafts that count (default: all in use). Without a ``mask`` one is
    built by every call. Call it before ``accept``, which moves the slots.
    """
    mask, index = _check("accumulate", ("q", "k"), (q, k), lengths, mask, counts)
    batch, heads, tokens, dim = q.shape
    cache.check_vector("accumulate", "lse", lse, torch.float32, (batch, heads, tokens), index)
    cache.check_vector("accumulate", "weights", weights, torch.float32, k.shape[:3], index)
    if rows is not None:
        cache.check_vector("accumulate", "rows", rows, torch.bool, (batch, tokens), index)
    scale = _scale(scale, dim)
    cache.check_device(index)
    ops.dispatch(torch.ops.sfl.tree_weights, (q, k, lse, lengths, mask, counts, rows, weights), (weights,), scale,
                 checked=True)
    return weights


def accept(k, v, lengths, path, accepted, *, weights=None, positions=None):
    """Commit an accepted path in place and return the new lengths (a new tensor).

    Slot ``lengths[b] + j`` takes the rows that slot ``lengths[b] + path[b, j]`` held, for the
    first ``accepted[b]`` entries of ``path`` (int32 ``[B, T]`` for the T drafts of the step, at
    most 128, drafts by index; one may stand in several entries).
    ``weights`` (fp32) and ``positions`` (int32), ``[B, Hkv, N]``, move with them, and the
    weights of the rejected drafts' slots become 0, as ``accumulate`` adds to them next time.
    The positions of the drafts' slots are the program's to write before the call.
    Entries outside ``[0, T)`` or the cache move nothing.
    """
    index = cache.check_rows("accept", ("k", "v"), (k, v))
    cache.check_cache(k, v)
    batch = k.shape[0]
    if path.ndim != 2 or not 1 <= path.shape[1] <= MAX_DRAFTS:
        raise ValueError(f"path must be [B, T] with T in [1, {MAX_DRAFTS}]")
    cache.check_vector("accept", "lengths", lengths, torch.int32, (batch,), index)
    cache.check_vector("accept", "path", path, torch.int32, (batch, path.shape[1]), index)
    cache.check_vector("accept", "accepted", accepted, torch.int32, (batch,), index)
    if weights is not None:
        cache.check_vector("accept", "weights", weights, torch.float32, k.shape[:3], index)
    if positions is not None:
        cache.check_vector("accept", "positions", positions, torch.int32, k.shape[:3], index)
    cache.check_device(index)
    _lib.lib()
    new_lengths = torch.empty_like(lengths)
    written = (k, v, weights, positions, new_lengths)
    ops.dispatch(torch.ops.sfl.accept_path, (lengths, path, accepted, *written), written, checked=True)
    return new_lengths
