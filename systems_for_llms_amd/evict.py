"""Eviction from a KV cache: the slots with the most accumulated attention weight stay.

``select`` chooses, for every KV head on its own, the ``keep`` slots that stay: the
``recent`` newest and of the others those with the largest weight (what
``tree.accumulate`` added up). ``compact`` then moves their rows so that they lie in
slots ``[0, keep)``. A slot that stays and lies there already does not move: the rows
that stay above ``keep`` fill the holes below it, so an eviction moves no more rows than
it must (attention does not care for the order of its keys, whose rotation is in them).
Slots are then no longer in the order of their tokens; ``positions`` keeps track of that
for the next ``select``: the program writes a token's position into its slot, for every KV
head, when it appends it, and ``tree.accept`` and ``compact`` move it with the row. Both
calls only touch the device and can be captured.
"""

from __future__ import annotations

import torch

from . import _lib
from . import cache
from . import ops  # registers torch.ops.sfl

MAX_SLOTS = 262144


def select(weights, lengths, keep, *, recent=0, positions=None):
    """``(kept, new_lengths)``: which slot's rows belong into each of the first ``keep`` slots.

    ``weights`` fp32 ``[B, Hkv, N]`` (N at most 262144), ``lengths`` int32 ``[B]``: slots in use.
    ``kept`` int32 ``[B, Hkv, keep]`` holds i where slot i < keep stays in place; the other
    places, in ascending order, take the slots from ``keep`` on that stay, in ascending
    order. A sequence of at most ``keep`` slots keeps them all, followed by -1.
    ``recent``: a slot stays before all others when its position is above its head's largest
    minus ``recent``; ``positions`` int32 ``[B, Hkv, N]``, written by the program for each
    token it appends (default: a slot's index, the age until slots have moved). Equal
    weights stay from the lowest slot on, as do recent slots that share positions and are
    more than ``keep``; NaN counts below every number.
    ``new_lengths`` is ``min(lengths, keep)``.
    """
    if weights.ndim != 3 or 0 in weights.shape:
        raise ValueError("weights must be [B, Hkv, N] and not empty")
    batch, heads, capacity = shape = weights.shape
    index = weights.get_device()
    cache.check_vector("select", "weights", weights, torch.float32, shape, index)
    if capacity > MAX_SLOTS:
        raise ValueError(f"at most {MAX_SLOTS} slots are supported")
    if type(keep) is not int or type(recent) is not int:
        raise TypeError("keep and recent must be integers")
    if not 1 <= keep <= capacity:
        raise ValueError("keep must be in [1, cache capacity]")
    if not 0 <= recent <= keep:
        raise ValueError("recent must be in [0, keep]")
    cache.check_vector("select", "lengths", lengths, torch.int32, (batch,), index)
    if positions is not None:
        cache.check_vector("select", "positions", positions, torch.int32, shape, index)
    cache.check_device(index)
    _lib.lib()  # fail here, before allocating, if the library is not built
    kept = torch.empty((batch, heads, keep), dtype=torch.int32, device=weights.device)
    new_lengths = torch.empty_like(lengths)
    ops.dispatch(torch.ops.sfl.select_slots, (weights, lengths, positions, kept, new_lengths), (kept, new_lengths),
                 recent, checked=True)
    return kept, new_lengths


def compact(kept, k, v, *, weights=None, positions=None):
    """Move the rows of ``k`` and ``v`` (``[B, Hkv, N, D]``) as ``kept`` (from ``select``) says, in place.

    ``weights`` (fp32) and ``positions`` (int32), ``[B, Hkv, N]``, move with them, and the
    weights of the slots from ``keep`` on become 0.
    """
    index = cache.check_rows("compact", ("k", "v"), (k, v))
    cache.check_cache(k, v)
    batch, heads, capacity, _ = k.shape
    if kept.ndim != 3 or not 1 <= kept.shape[2] <= capacity:
        raise ValueError("kept must be [B, Hkv, keep] with keep in [1, cache capacity]")
    cache.check_vector("compact", "kept", kept, torch.int32, (batch, heads, kept.shape[2]), index)
    if weights is not None:
        cache.check_vector("compact", "weights", weights, torch.float32, (batch, heads, capacity), index)
    if positions is not None:
        cache.check_vector("compact", "positions", positions, torch.int32, (batch, heads, capacity), index)
    cache.check_device(index)
    written = (k, v, weights, positions)
    ops.dispatch(torch.ops.sfl.compact_slots, (kept, *written), written, checked=True)


def evict(k, v, weights, lengths, keep, *, recent=0, positions=None):
    """``select`` and ``compact`` with everything moved: returns ``(kept, new_lengths)``."""
    index = cache.check_rows("evict", ("k", "v"), (k, v))
    cache.check_cache(k, v)
    cache.check_vector("evict", "weights", weights, torch.float32, k.shape[:3], index)
    kept, new_lengths = select(weights, lengths, keep, recent=recent, positions=positions)
    compact(kept, k, v, weights=weights, positions=positions)
    return kept, new_lengths
