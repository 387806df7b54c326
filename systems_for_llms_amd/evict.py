"""Eviction from a KV cache: the slots with the most accumulated attention weight stay.

``select`` chooses, for every KV head on its own, the ``keep`` slots that stay: the
``recent`` newest and of the others those with the largest weight (what
``tree.accumulate`` added up). ``compact`` then moves their rows so that they lie in
slots ``[0, keep)``. A slot that stays and lies there already does not move: the rows
that stay above ``keep`` fill the holes below it, so an eviction moves no more rows than
it must (attention does not care for the order of its keys, whose rotation is in them).
Slots are then no longer in the order of their tokens; ``positions`` keeps track of that
for the next ``select``. Both calls only touch the device and can be captured.
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
    minus ``recent``; ``positions`` int32 ``[B, Hkv, N]`` (default: a slot's index). Equal
    weights stay from the lowest slot on, as do recent slots that share positions and are
    more than ``keep``; NaN counts below every number.
    ``new_lengths`` is ``min(lengths, keep)``.
    """
    if weights.ndim != 3 or weights.dtype != torch.float32 or not weights.is_contiguous() or min(weights.shape) < 1:
        raise ValueError("weights must be a contiguous float32 tensor [B, Hkv, N]")
    if weights.requires_grad:
        raise RuntimeError("select is forward-only; requires_grad inputs are unsupported")
    batch, heads, capacity = weights.shape
    if capacity > MAX_SLOTS:
        raise ValueError(f"at most {MAX_SLOTS} slots are supported")
    for name, value in (("keep", keep), ("recent", recent)):
        if type(value) is not int:
            raise TypeError(f"{name} must be an integer")
    if not 1 <= keep <= capacity:
        raise ValueError("keep must be in [1, cache capacity]")
    if not 0 <= recent <= keep:
        raise ValueError("recent must be in [0, keep]")
    cache.check_vector("lengths", lengths, torch.int32, (batch,))
    cache.check_vector("positions", positions, torch.int32, tuple(weights.shape))
    cache.check_device(weights.device, {"lengths": lengths, "positions": positions})
    _lib.lib()  # fail here, before allocating, if the library is not built
    kept = torch.empty((batch, heads, keep), dtype=torch.int32, device=weights.device)
    new_lengths = torch.empty_like(lengths)
    ops.dispatch(torch.ops.sfl.select_slots, (weights, lengths, positions, kept, new_lengths), (kept, new_lengths),
                 recent)
    return kept, new_lengths


def compact(kept, k, v, *, weights=None, positions=None):
    """Move the rows of ``k`` and ``v`` (``[B, Hkv, N, D]``) as ``kept`` (from ``select``) says, in place.

    ``weights`` (fp32) and ``positions`` (int32), ``[B, Hkv, N]``, move with them, and the
    weights of the slots from ``keep`` on become 0.
    """
    cache.check_rows("compact", {"k": k, "v": v})
    cache.check_cache(k, v)
    batch, heads, capacity, _ = k.shape
    if kept.ndim != 3 or not 1 <= kept.shape[2] <= capacity:
        raise ValueError("kept must be [B, Hkv, keep] with keep in [1, cache capacity]")
    cache.check_vector("kept", kept, torch.int32, (batch, heads, kept.shape[2]))
    cache.check_vector("weights", weights, torch.float32, (batch, heads, capacity))
    cache.check_vector("positions", positions, torch.int32, (batch, heads, capacity))
    cache.check_device(k.device, {"kept": kept, "weights": weights, "positions": positions})
    if weights is not None and weights.requires_grad:
        raise RuntimeError("compact is forward-only; requires_grad inputs are unsupported")
    written = (k, v, weights, positions)
    ops.dispatch(torch.ops.sfl.compact_slots, (kept, *written), written)


def evict(k, v, weights, lengths, keep, *, recent=0, positions=None):
    """``select`` and ``compact`` with everything moved: returns ``(kept, new_lengths)``."""
    cache.check_rows("evict", {"k": k, "v": v})
    cache.check_cache(k, v)
    if tuple(weights.shape) != tuple(k.shape[:3]):
        raise ValueError("weights must be [B, Hkv, N] for caches [B, Hkv, N, D]")
    cache.check_device(k.device, {"weights": weights})
    kept, new_lengths = select(weights, lengths, keep, recent=recent, positions=positions)
    compact(kept, k, v, weights=weights, positions=positions)
    return kept, new_lengths
