"""Plain float64 forms of the KV-cache operators (test infrastructure; not imported by the product).

Each follows its definition row by row: only what a row sees is indexed, so values in
places it does not see cannot reach it. Next to the results come the magnitudes that
the tests' error bounds are made of.
"""

from __future__ import annotations

import math

import torch


def rotate(x, positions, cos, sin, layout, gain=None, eps=1e-5):
    """(y, size): the turned rows of x [B, H, T, D] and, by element, the length of the pair turned (or the value)."""
    y = x.double().clone()
    if gain is not None:
        y = y / ((y * y).mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    half, table = cos.shape[1], cos.shape[0]
    known = ((positions >= 0) & (positions < table))[..., None]  # [B, T, 1]
    at = positions.clamp(0, table - 1).long()
    c, sn = (torch.where(known, x[at].double(), math.nan)[:, None] for x in (cos, sin))
    first = torch.arange(half) if layout == "half" else 2 * torch.arange(half)
    second = first + half if layout == "half" else first + 1
    u, w = y[..., first], y[..., second]
    out, size = y.clone(), y.abs()
    out[..., first], out[..., second] = u * c - w * sn, w * c + u * sn
    size[..., first] = size[..., second] = torch.hypot(u, w)
    return out, size


def seen_slots(b, t, lengths, mask, counts, capacity):
    """Slots that draft t of sequence b sees."""
    n = min(max(int(lengths[b]), 0), capacity)
    count = mask.shape[-1] if counts is None else int(counts[b])
    row = mask[b, t] if mask.ndim == 3 else mask[t]
    if t >= count:
        return []
    return list(range(n)) + [n + j for j in range(count) if bool(row[j]) and n + j < capacity]


def tree_attention(q, k, v, lengths, mask, counts=None, scale=None):
    """out, lse and the bounds' magnitudes: sum of weights times |v|, and the largest sum of |q k| by row."""
    batch, heads, tokens, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    spread, size = torch.zeros_like(out), torch.zeros(q.shape[:3], dtype=torch.float64)
    for b in range(batch):
        for t in range(tokens):
            slots = seen_slots(b, t, lengths, mask, counts, k.shape[2])
            if not slots:
                continue
            keys, values = (x[b, :, slots].double().repeat_interleave(group, 0) for x in (k, v))  # [Hq, n, D]
            row = q[b, :, t].double()[..., None]
            scores = (keys @ row)[..., 0] * scale
            lse[b, :, t] = torch.logsumexp(scores, -1)
            p = torch.softmax(scores, -1)[:, None]
            out[b, :, t] = (p @ values)[:, 0]
            spread[b, :, t] = (p @ values.abs())[:, 0]
            size[b, :, t] = (keys.abs() @ row.abs())[..., 0].amax(-1) * scale
    return out, lse, spread, size


def tree_weights(q, k, lse, weights, lengths, mask, counts=None, rows=None, scale=None):
    """weights plus exp(s - lse) by slot; by slot also the largest sum of |q k|."""
    batch, heads, tokens, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    total, size = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    for b in range(batch):
        for t in range(tokens):
            slots = seen_slots(b, t, lengths, mask, counts, k.shape[2])
            if not slots or (rows is not None and not bool(rows[b, t])):
                continue
            keys = k[b, :, slots].double().repeat_interleave(group, 0)
            row = q[b, :, t].double()[..., None]
            base = lse[b, :, t].double()[:, None]
            p = torch.where(base == -math.inf, 0.0, torch.exp((keys @ row)[..., 0] * scale - base))
            total[b, :, slots] += p.unflatten(0, (-1, group)).sum(1)
            reach = (keys.abs() @ row.abs())[..., 0].unflatten(0, (-1, group)).amax(1) * scale
            size[b, :, slots] = torch.maximum(size[b, :, slots], reach)
    return total, size


def accept(tensors, lengths, path, accepted, weights=None):
    """The caches after an accepted path, and the new lengths; ``weights`` (one of the tensors) loses the rejected."""
    done = [x.clone() for x in tensors]
    tokens = path.shape[1]
    for b in range(path.shape[0]):
        n, capacity = int(lengths[b]), tensors[0].shape[2]
        for x, y in zip(tensors, done):
            for j in range(tokens):
                at = n + j
                if at >= capacity:
                    break
                if j < int(accepted[b]):
                    y[b, :, at] = x[b, :, n + int(path[b, j])]
                elif x is weights:
                    y[b, :, at] = 0
    return done, lengths + accepted


def select(weights, lengths, keep, recent=0, positions=None):
    """kept and the new lengths, by sorting: recent slots by index, then the others by weight and index."""
    batch, heads, _ = weights.shape
    kept = torch.full((batch, heads, keep), -1, dtype=torch.int32)
    for b in range(batch):
        n = int(lengths[b])
        for h in range(heads):
            w = weights[b, h, :n].tolist()
            age = list(range(n)) if positions is None else positions[b, h, :n].tolist()
            since = max(age, default=0) - recent

            def place(i):
                if age[i] > since:
                    return (0, 0.0, i)
                return (2, 0.0, i) if math.isnan(w[i]) else (1, -w[i], i)

            rank = sorted(range(n), key=place)
            stay = set(rank[:keep])
            movers = iter(sorted(i for i in stay if i >= keep))
            row = [i if i in stay else next(movers) for i in range(min(n, keep))]
            kept[b, h, : len(row)] = torch.tensor(row, dtype=torch.int32)
    return kept, lengths.clamp(max=keep)


def compact(tensors, kept, weights=None):
    """Slot i of every tensor as kept says; ``weights`` (one of the tensors) is cleared from keep on."""
    done = [x.clone() for x in tensors]
    keep = kept.shape[2]
    for b in range(kept.shape[0]):
        for h in range(kept.shape[1]):
            for i, source in enumerate(kept[b, h].tolist()):
                for x, y in zip(tensors, done):
                    if source >= keep:
                        y[b, h, i] = x[b, h, source]
    for x, y in zip(tensors, done):
        if x is weights:
            y[:, :, keep:] = 0
    return done
