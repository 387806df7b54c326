"""Plain float64 and list forms of the paged 8-bit cache's operators (test infrastructure; not imported by the product).

A cache is a dict of CPU tensors by the names of ``PagedCache``'s fields. Rows, places and
tokens are gone through one after another, as the definitions say.
"""

from __future__ import annotations

import math

import torch

F8 = torch.float8_e4m3fn
LEAST = -100


def nearest_code(x):
    """float64 values as the nearest e4m3 numbers (4 bits from 2^-6 on, steps of 2^-9 below), ties to even."""
    exponent = torch.frexp(x)[1].double() - 1
    step = torch.exp2(exponent.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def least_exponent(amax):
    """The least e >= -100 with amax <= 448 * 2^e."""
    e = LEAST
    while amax > 448 * 2.0 ** e:
        e += 1
    return e


def append(cache, k, v, counts=None, layer=0):
    """The cache with new tokens in its pages, a new dict."""
    done = {n: x.clone() for n, x in cache.items()}
    page, pages = cache["k"].shape[3], cache["k"].shape[1]
    places = cache["tables"].shape[1]
    for b in range(k.shape[0]):
        n = int(cache["lengths"][b])
        count = k.shape[2] if counts is None else min(max(int(counts[b]), 0), k.shape[2])
        for place in range(n // page, places):
            lo, hi = max(n - place * page, 0), min(n + count - place * page, page)
            at = int(cache["tables"][b, place])
            if lo >= hi or not 0 <= at < pages or int(cache["refs"][at]) != 1:
                continue
            for name, new in (("k", k), ("v", v)):
                for h in range(k.shape[1]):
                    x = new[b, h, place * page + lo - n: place * page + hi - n].double()
                    x = torch.where(x.abs() < 2.0 ** 127, x, math.nan)
                    e = least_exponent(float(x.abs().nan_to_num(0.0).max()))
                    codes = done[name][layer, at, h].double()
                    if name == "v":
                        codes = codes.T
                    scale = done[name + "_scale"][layer, at, h]
                    if lo:
                        before = max(int(torch.frexp(scale)[1]) - 1, LEAST) if scale else LEAST
                        if e > before:
                            codes[:lo] = nearest_code(codes[:lo] * 2.0 ** (before - e))
                        e = max(e, before)
                    codes[lo:hi] = nearest_code(x / 2.0 ** e)
                    done[name][layer, at, h] = (codes if name == "k" else codes.T).float().to(F8)
                    done[name + "_scale"][layer, at, h] = 2.0 ** e
    return done


def rows_of(cache, b, slots, layer=0):
    """Keys and values [Hkv, n, D] of a row's slots, in float64."""
    page = cache["k"].shape[3]
    at = [int(cache["tables"][b, s // page]) for s in slots]
    off = [s % page for s in slots]
    k = cache["k"][layer].double()[at, :, off] * cache["k_scale"][layer].double()[at][..., None]
    v = cache["v"][layer].double()[at, :, :, off] * cache["v_scale"][layer].double()[at][..., None]
    return k.transpose(0, 1), v.transpose(0, 1)


def seen_slots(cache, b, t, tokens, counts=None, window=None):
    page, pages = cache["k"].shape[3], cache["k"].shape[1]
    row = cache["tables"][b].tolist()
    n = min(max(int(cache["lengths"][b]), 0), len(row) * page)
    count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
    if t >= count or n + t >= len(row) * page:
        return []
    first = 0 if window is None else max(0, n + t - window)
    return [s for s in range(first, n + t + 1) if 0 <= row[s // page] < pages]


def attention(q, cache, layer=0, counts=None, window=None, scale=None):
    """out, lse and the bounds' magnitudes: sum of weights times |v|, and the largest sum of |q k| by row."""
    batch, heads, tokens, dim = q.shape
    kv_heads = cache["k"].shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    spread, size = torch.zeros_like(out), torch.zeros(q.shape[:3], dtype=torch.float64)
    for b in range(batch):
        for t in range(tokens):
            slots = seen_slots(cache, b, t, tokens, counts, window)
            if not slots:
                continue
            keys, values = (x.repeat_interleave(heads // kv_heads, 0) for x in rows_of(cache, b, slots, layer))
            row = q[b, :, t].double()[..., None]
            scores = (keys @ row)[..., 0] * scale
            lse[b, :, t] = torch.logsumexp(scores, -1)
            p = torch.softmax(scores, -1)[:, None]
            out[b, :, t] = (p @ values)[:, 0]
            spread[b, :, t] = (p @ values.abs())[:, 0]
            size[b, :, t] = (keys.abs() @ row.abs())[..., 0].amax(-1) * scale
    return out, lse, spread, size


def _copied(cache, moves):
    done = {n: x.clone() for n, x in cache.items()}
    for source, target in moves:
        for name in ("k", "v", "k_scale", "v_scale"):
            done[name][:, target] = cache[name][:, source]
    return done


def _with_books(cache, tables, lengths, refs):
    for name, x in (("tables", tables), ("lengths", lengths), ("refs", refs)):
        cache[name] = torch.tensor(x, dtype=torch.int32).reshape(cache[name].shape)
    return cache


def fork(cache, parents):
    page = cache["k"].shape[3]
    old, lengths, refs = cache["tables"].tolist(), cache["lengths"].tolist(), cache["refs"].tolist()
    tables, new = [list(r) for r in old], list(lengths)
    for b, p in enumerate(parents.tolist()):
        if p == b or not -1 <= p < len(old):
            continue
        new[b] = lengths[p] if p >= 0 else 0
        filled = -(-new[b] // page)
        for x in old[b]:
            if x >= 0:
                refs[x] -= 1
        tables[b] = [old[p][j] if j < filled else -1 for j in range(len(old[b]))]
        for x in tables[b]:
            if x >= 0:
                refs[x] += 1
    return _with_books({n: x.clone() for n, x in cache.items()}, tables, new, refs)


def reserve(cache, counts):
    """(granted, cache): each row after the one before, each place after the one before."""
    page = cache["k"].shape[3]
    tables, lengths, refs = cache["tables"].tolist(), cache["lengths"].tolist(), cache["refs"].tolist()
    granted, moves = [], []
    for b, row in enumerate(tables):
        n = lengths[b]
        end = n + min(max(int(counts[b]), 0), len(row) * page - n)
        reach = end
        for place in range(n // page, -(-end // page) if end > n else 0):
            held = row[place]
            if held >= 0 and refs[held] == 1:
                continue
            if 0 not in refs:
                reach = min(reach, max(n, place * page))
                continue
            now = refs.index(0)
            if held >= 0:
                refs[held] -= 1
                if place * page < n:
                    moves.append((held, now))
            refs[now], row[place] = 1, now
        granted.append(reach - n)
    return torch.tensor(granted, dtype=torch.int32), _with_books(_copied(cache, moves), tables, lengths, refs)


def compact(cache):
    """(used, cache)"""
    refs = cache["refs"].tolist()
    used = sum(r > 0 for r in refs)
    movers = [p for p in range(used, len(refs)) if refs[p] > 0]
    holes = [p for p in range(used) if refs[p] <= 0]
    to = dict(zip(movers, holes))
    done = _copied(cache, to.items())
    for source, target in to.items():
        refs[target], refs[source] = refs[source], 0
    tables = [[to.get(x, x) for x in row] for row in cache["tables"].tolist()]
    return used, _with_books(done, tables, cache["lengths"].tolist(), refs)
