"""Workloads of the operators that keep a bounded KV cache and verify drafted tokens over it.

Each case is one call (or the two calls of an eviction) that a serving program makes:

* ``rotate``      ``rotary.rotate_append``: per-head RMSNorm and rotation of q and k, k and v
  written into the cache; q, k and v are the slices of one projection's output;
* ``tree``        ``tree.prepare`` kept and called: attention of a tree of drafted tokens over
  the cached keys and over those drafts that are their ancestors;
* ``accumulate``  ``tree.accumulate``: the attention weights of the counted drafts added up by slot;
* ``accept``      ``tree.accept``: the accepted path's rows moved behind the committed ones;
* ``evict``       ``evict.select`` and ``evict.compact``: the heaviest and the newest slots stay.

With ``own`` false ``run`` computes the same in elementary torch operations in 32 bits;
``exact`` computes it in 64 bits from the definitions.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
TABLE = 131072  # positions of the rotary tables


def listed():
    return [
        # One token each of a serving batch: normed heads, half layout, far positions.
        {"name": "rotate_decode_b32", "kind": "rotate", "dtype": "bf16", "batch": 32, "drafts": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "norm": True, "keys": 600, "ragged": False},
        # A batch of padded prompts, interleaved pairs on half of each head.
        {"name": "rotate_prompt_b4", "kind": "rotate", "dtype": "fp16", "batch": 4, "drafts": 4001, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 64, "layout": "interleaved", "norm": True, "keys": 4100,
         "ragged": True},
        # One interactive sequence, no drafts: the latency of the operator itself.
        {"name": "tree_one_token", "kind": "tree", "dtype": "bf16", "batch": 1, "drafts": 1, "heads": 32,
         "kv_heads": 4, "dim": 128, "keys": 1024, "ragged": False},
        # The parity model's heads (16 of 32) in float32 with a few drafts.
        {"name": "tree_fp32_b4", "kind": "tree", "dtype": "fp32", "batch": 4, "drafts": 7, "heads": 16,
         "kv_heads": 16, "dim": 32, "keys": 1001, "ragged": True},
        # A serving batch that verifies trees of 27 drafts, rows of different lengths.
        {"name": "tree_b8_t27", "kind": "tree", "dtype": "bf16", "batch": 8, "drafts": 27, "heads": 32,
         "kv_heads": 8, "dim": 128, "keys": 8191, "ragged": True},
        # A wide tree over one long context: 512 query rows for each cached head.
        {"name": "tree_long_t64", "kind": "tree", "dtype": "fp16", "batch": 1, "drafts": 64, "heads": 32,
         "kv_heads": 4, "dim": 128, "keys": 65536, "ragged": False},
        # The weights of single tokens of a short batch.
        {"name": "accumulate_one_token", "kind": "accumulate", "dtype": "bf16", "batch": 4, "drafts": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "keys": 2048, "ragged": True},
        # The weights of the accepted rows of drafted trees over long caches, heads of 64.
        {"name": "accumulate_b16_t16", "kind": "accumulate", "dtype": "bf16", "batch": 16, "drafts": 16,
         "heads": 16, "kv_heads": 16, "dim": 64, "keys": 8192, "ragged": True},
        # Accepted paths of a small and of a large batch.
        {"name": "accept_b2_t16", "kind": "accept", "dtype": "fp16", "batch": 2, "drafts": 16, "kv_heads": 16,
         "dim": 64, "keys": 500},
        {"name": "accept_b64_t64", "kind": "accept", "dtype": "bf16", "batch": 64, "drafts": 64, "kv_heads": 8,
         "dim": 128, "keys": 700},
        # A long prompt cut down to a budget, once.
        {"name": "evict_prompt", "kind": "evict", "dtype": "bf16", "batch": 4, "kv_heads": 8, "dim": 128,
         "keys": 20011, "keep": 4096, "recent": 512, "positions": False, "short": False},
        # The same budget kept up while decoding: a few new slots each time, rows that need nothing among them.
        {"name": "evict_steady", "kind": "evict", "dtype": "fp16", "batch": 16, "kv_heads": 8, "dim": 64,
         "keys": 4160, "keep": 4096, "recent": 256, "positions": True, "short": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= limit:
            return case


def _draw(rng):
    kind = rng.choice(["rotate", "tree", "tree", "accumulate", "accept", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv_heads = rng.choice([4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 128, 128])
    if kind == "rotate":
        drafts = _log_int(rng, 1, 4096)
        return {"kind": kind, "dtype": dtype, "batch": max(1, min(64, _log_int(rng, 1, 16384) // drafts)),
                "drafts": drafts, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
                "norm": rng.random() < 0.5, "keys": drafts + _log_int(rng, 16, 600), "ragged": rng.random() < 0.5}
    if kind in ("tree", "accumulate"):
        drafts = _log_int(rng, 1, 64)
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, 32), "drafts": drafts, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "keys": drafts + _log_int(rng, 100, 32768),
                "ragged": rng.random() < 0.6}
    if kind == "accept":
        drafts = _log_int(rng, 2, 64)
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, 64), "drafts": drafts, "kv_heads": kv_heads,
                "dim": dim, "keys": drafts + _log_int(rng, 16, 700)}
    keys = _log_int(rng, 500, 24000)
    keep = _log_int(rng, keys // 8, keys - 1)
    return {"kind": kind, "dtype": dtype, "batch": min(_log_int(rng, 1, 16), max(1, 100000 // keys)),
            "kv_heads": kv_heads, "dim": dim, "keys": keys, "keep": keep, "recent": _log_int(rng, 16, keep // 2), "positions": rng.random() < 0.5,
            "short": rng.random() < 0.3}


def _shared_lengths(case):
    """Committed lengths as Python ints, the same for every seed, so that ``work`` can count them."""
    b, room = case["batch"], case["keys"] - case.get("drafts", 0)
    if not case.get("ragged"):
        return [room] * b
    return [max(0, room - (room * 7 * i) // (8 * b)) for i in range(b)]


def _counts(case):
    """Drafts in use in each row."""
    t, b = case["drafts"], case["batch"]
    return [t - (t * i) // (3 * b) for i in range(b)] if case.get("ragged") else [t] * b


def _rotate_counts(case):
    """Tokens in use in each row of a rotation (the rest is padding)."""
    return _counts(case)


def _counted_rows(case):
    """How many of a row's drafts count in an accumulation: one of three, and the root always."""
    return [max(1, -(-c // 3)) for c in _counts(case)]


def _evict_lengths(case):
    keys, keep, b = case["keys"], case["keep"], case["batch"]
    lengths = [keys - (keys - keep) * i // (2 * b) for i in range(b)]
    if case["short"]:
        lengths[-1] = keep // 2 + 1
    return lengths


def work(case):
    es, kind = SIZE[case["dtype"]], case["kind"]
    b, dim, kv = case["batch"], case["dim"], case["kv_heads"]
    if kind == "rotate":
        tokens, heads = sum(_rotate_counts(case)), case["heads"]
        elements = tokens * (heads + 2 * kv) * dim
        return {"bytes": 2 * elements * es + tokens * case["rotary"] * 4, "flops": 8 * elements}
    if kind == "tree":
        pairs = list(zip(_shared_lengths(case), _counts(case)))
        seen = sum(n + c for n, c in pairs)
        rows = sum((n + c) * c for n, c in pairs)
        io = 2 * b * case["drafts"] * case["heads"] * dim * es
        return {"bytes": 2 * seen * kv * dim * es + io, "flops": 4 * rows * case["heads"] * dim}
    if kind == "accumulate":
        trio = list(zip(_shared_lengths(case), _counts(case), _counted_rows(case)))
        seen = sum(n + c for n, c, _ in trio)
        rows = sum((n + c) * r for n, c, r in trio)
        return {"bytes": seen * kv * (dim * es + 8) + sum(r for _, _, r in trio) * case["heads"] * dim * es,
                "flops": 2 * rows * case["heads"] * dim}
    if kind == "accept":
        moved = sum(_accepted(case))
        return {"bytes": 4 * moved * kv * dim * es + 16 * moved * kv, "flops": 0}
    # About keep * (n - keep) / n slots change places where weights do not go by age.
    lengths = _evict_lengths(case)
    moved = sum(case["keep"] * (n - case["keep"]) // n for n in lengths if n > case["keep"])
    slots = sum(lengths) * (8 if case["positions"] else 4)
    return {"bytes": kv * (slots + 4 * b * case["keep"] + 4 * moved * dim * es), "flops": 2 * sum(lengths) * kv}


def _accepted(case):
    t = case["drafts"]
    return [1 + (t * (i % 5)) // 8 if i % 5 else 0 for i in range(1, case["batch"] + 1)]


def _tree_mask(case, g):
    """Ancestor masks [B, T, T] of random trees: draft t hangs on an earlier draft or on the committed text."""
    b, t = case["batch"], case["drafts"]
    mask = torch.zeros(b, t, t, dtype=torch.bool)
    for i in range(t):
        if i:
            parents = torch.randint(-1, i, (b,), generator=g)
            mask[:, i] = mask[torch.arange(b), parents.clamp(min=0)] & (parents >= 0)[:, None]
        mask[:, i, i] = True
    return mask


def _tables(rotary):
    """Angles of TABLE positions in 64 bits, frequencies lowered by a ramp for a context 8 times longer."""
    inverse = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    turns = TABLE / 8 * inverse / (2 * math.pi)
    ramp = ((turns - 1) / 31).clamp(0, 1)
    inverse = inverse * ramp + inverse / 8 * (1 - ramp)
    angles = torch.arange(TABLE, dtype=torch.float64, device="cuda")[:, None] * inverse
    return angles.cos().float(), angles.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    b, dim, kv, keys = case["batch"], case["dim"], case["kv_heads"], case["keys"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32).cuda()

    state = {"case": case, "k": normal(b, kv, keys, dim), "v": normal(b, kv, keys, dim)}
    if kind == "rotate":
        t, heads = case["drafts"], case["heads"]
        qkv = normal(b, t, heads + 2 * kv, dim).transpose(1, 2)
        state["q"], state["k_new"], state["v_new"] = qkv.split([heads, kv, kv], 1)
        state["cos"], state["sin"] = _tables(case["rotary"])
        first = torch.randint(0, TABLE - t, (b, 1), generator=g, device="cuda")
        state["positions"] = (first + torch.arange(t, device="cuda")).to(torch.int32)
        state["lengths"] = ints([(keys - t) * (i + 1) // b for i in range(b)])
        state["counts"] = ints(_rotate_counts(case)) if case["ragged"] else None
        for name in ("q_norm", "k_norm"):
            state[name] = 1 + 0.1 * normal(dim) if case["norm"] else None
        return state
    if kind in ("tree", "accumulate"):
        t, heads = case["drafts"], case["heads"]
        # q as a projection leaves it ([B, T, H, D]); sharper than normal, so that some keys stand out.
        state["q"] = (2 * torch.randn(b, t, heads, dim, generator=g, device="cuda")).to(dtype).transpose(1, 2)
        state["lengths"] = ints(_shared_lengths(case))
        state["counts"] = ints(_counts(case)) if case["ragged"] else None
        state["mask"] = _tree_mask(case, host).cuda()
        if kind == "accumulate":
            counted = torch.zeros(b, t, dtype=torch.bool)
            for i, n in enumerate(_counted_rows(case)):
                counted[i, 0] = True
                counted[i, 1 + torch.randperm(_counts(case)[i] - 1, generator=host)[: n - 1]] = True
            state["rows"] = counted.cuda()
            state["lse"] = torch.logsumexp(_scores(state, torch.float32), -1).reshape(b, heads, t)
            state["weights"] = torch.rand(b, kv, keys, generator=g, device="cuda") * 3
        elif own:
            from systems_for_llms_amd import tree

            state["op"] = tree.prepare(state["q"], state["k"], state["v"], state["lengths"], state["mask"],
                                       counts=state["counts"])
        return state
    if kind == "accept":
        t = case["drafts"]
        state["lengths"] = ints([(keys - t) * (i + 1) // b for i in range(b)])
        state["path"] = torch.stack([torch.cat([torch.randperm(t, generator=host)[:n].sort().values,
                                                torch.zeros(t - n, dtype=torch.int64)])
                                     for n in _accepted(case)]).to(torch.int32).cuda()
        state["accepted"] = ints(_accepted(case))
        state["weights"] = torch.rand(b, kv, keys, generator=g, device="cuda")
        state["positions"] = torch.randint(0, TABLE, (b, kv, keys), generator=g, device="cuda", dtype=torch.int32)
        return state
    # Accumulated weights are heavy-tailed, and many slots have none at all: ties.
    u = torch.rand(b, kv, keys, generator=g, device="cuda")
    state["weights"] = torch.where(u < 0.2, torch.zeros_like(u), u.pow(8) * 100)
    state["lengths"] = ints(_evict_lengths(case))
    state["positions"] = None
    if case["positions"]:
        state["positions"] = torch.rand(b, kv, keys, generator=g, device="cuda").argsort(-1).to(torch.int32)
    return state


def run(state):
    case = state["case"]
    return {"rotate": _run_rotate, "tree": _run_tree, "accumulate": _run_accumulate, "accept": _run_accept,
            "evict": _run_evict}[case["kind"]](case, state)


def _rotated(x, gain, cos, sin, layout):
    """x [B, H, T, D] in the type of cos, normed where there is a gain, its first dims rotated by [B, 1, T, rd/2]."""
    if gain is not None:
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain
    half = cos.shape[-1]
    head, rest = x[..., : 2 * half], x[..., 2 * half:]
    if layout == "half":
        a, b = head[..., :half], head[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _run_rotate(case, s):
    if own:
        from systems_for_llms_amd import rotary

        q = rotary.rotate_append(s["q"], s["k_new"], s["v_new"], s["positions"], s["cos"], s["sin"], s["k"], s["v"],
                                 s["lengths"], counts=s["counts"], layout=case["layout"], q_norm=s["q_norm"],
                                 k_norm=s["k_norm"], eps=EPS)
        return {"q": q, "k": s["k"], "v": s["v"]}
    dtype, t = s["q"].dtype, s["q"].shape[2]
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    gains = [None if s[n] is None else s[n].float() for n in ("q_norm", "k_norm")]
    q = _rotated(s["q"].float(), gains[0], cos, sin, case["layout"]).to(dtype)
    k = _rotated(s["k_new"].float(), gains[1], cos, sin, case["layout"]).to(dtype)
    slots = s["lengths"].long()[:, None] + torch.arange(t, device=q.device)
    rows = torch.arange(q.shape[0], device=q.device)[:, None].expand_as(slots)
    v = s["v_new"]
    if s["counts"] is not None:
        used = torch.arange(t, device=q.device) < s["counts"][:, None]
        q = torch.where(used[:, None, :, None], q, 0)
        s["k"][rows[used], :, slots[used]] = k.transpose(1, 2)[used]
        s["v"][rows[used], :, slots[used]] = v.transpose(1, 2)[used]
    else:
        s["k"][rows, :, slots] = k.transpose(1, 2)
        s["v"][rows, :, slots] = v.transpose(1, 2)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _visible(s):
    """[B, T, N]: which slots each draft attends to (none for drafts that are not in use)."""
    t, n = s["q"].shape[2], s["k"].shape[2]
    slot = torch.arange(n, device=s["k"].device)
    offset = slot - s["lengths"].long()[:, None]  # [B, N]: which draft a slot holds
    tree = s["mask"].gather(2, offset.clamp(0, t - 1)[:, None].expand(-1, t, -1))
    inside = (offset >= 0) & (offset < t)
    if s["counts"] is not None:
        inside = inside & (offset < s["counts"][:, None])
    seen = (offset < 0)[:, None] | (tree & inside[:, None])
    if s["counts"] is not None:
        seen = seen & (torch.arange(t, device=slot.device) < s["counts"][:, None])[:, :, None]
    return seen


def _scores(s, kind):
    """Scaled scores [B, Hkv, G*T, N] in the given type, -inf where a draft does not look."""
    b, heads, t, dim = s["q"].shape
    kv = s["k"].shape[1]
    q = s["q"].to(kind).reshape(b, kv, heads // kv * t, dim)
    x = torch.matmul(q, s["k"].to(kind).transpose(-1, -2)) * dim ** -0.5
    seen = _visible(s)[:, None, None].expand(-1, kv, heads // kv, -1, -1).reshape(x.shape)
    return x.masked_fill(~seen, -math.inf)


def _run_tree(case, s):
    if own:
        return {"out": s["op"](), "lse": s["op"].lse}
    b, heads, t, dim = s["q"].shape
    x = _scores(s, torch.float32)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = (x - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, s["v"].float()) / torch.where(total == 0, 1, total)
    return {"out": out.reshape(b, heads, t, dim).to(s["q"].dtype), "lse": (top + total.log()).reshape(b, heads, t)}


def _run_accumulate(case, s):
    if own:
        from systems_for_llms_amd import tree

        return tree.accumulate(s["q"], s["k"], s["lse"], s["weights"], s["lengths"], s["mask"], counts=s["counts"],
                               rows=s["rows"])
    b, heads, t, _ = s["q"].shape
    kv = s["k"].shape[1]
    lse = s["lse"].reshape(b, kv, -1, 1)
    p = torch.where(lse == -math.inf, 0, (_scores(s, torch.float32) - lse).exp())
    counted = s["rows"][:, None, None].expand(-1, kv, heads // kv, -1).reshape(b, kv, -1, 1)
    s["weights"] += torch.where(counted, p, 0).sum(2)
    return s["weights"]


def _run_accept(case, s):
    if own:
        from systems_for_llms_amd import tree

        lengths = tree.accept(s["k"], s["v"], s["lengths"], s["path"], s["accepted"], weights=s["weights"],
                              positions=s["positions"])
        return {"lengths": lengths, "k": s["k"], "v": s["v"], "weights": s["weights"], "positions": s["positions"]}
    t = s["path"].shape[1]
    start = s["lengths"].long()[:, None]
    j = torch.arange(t, device=start.device)
    source = start + torch.where(j < s["accepted"][:, None], s["path"].long(), j)
    rows = torch.arange(start.shape[0], device=start.device)[:, None]
    for name in ("k", "v", "weights", "positions"):
        s[name][rows, :, start + j] = s[name][rows, :, source]
    kept = (j < s["accepted"][:, None])[..., None]
    s["weights"][rows, :, start + j] = torch.where(kept, s["weights"][rows, :, start + j], 0)
    return {"lengths": s["lengths"] + s["accepted"], "k": s["k"], "v": s["v"], "weights": s["weights"],
            "positions": s["positions"]}


def _run_evict(case, s):
    keep = case["keep"]
    if own:
        from systems_for_llms_amd import evict

        kept, lengths = evict.select(s["weights"], s["lengths"], keep, recent=case["recent"],
                                     positions=s["positions"])
        evict.compact(kept, s["k"], s["v"])
        return {"kept": kept, "lengths": lengths, "k": s["k"], "v": s["v"]}
    n = s["lengths"].long()[:, None, None]
    slot = torch.arange(s["k"].shape[2], device=n.device)
    used = slot < n
    age = torch.where(used, slot if s["positions"] is None else s["positions"].long(), -1)
    newest = age.amax(-1, keepdim=True)
    weight = torch.where(age > newest - case["recent"], math.inf, s["weights"])
    weight = torch.where(used, weight, -math.inf)
    order = weight.sort(dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros(weight.shape, dtype=torch.bool, device=n.device)
    chosen.scatter_(-1, order[..., :keep], True)
    chosen &= used
    movers = slot.masked_fill(~(chosen & (slot >= keep)), slot.numel()).sort(-1).values
    rank = (~chosen[..., :keep]).cumsum(-1) - 1
    kept = torch.where(chosen[..., :keep], slot[:keep], movers.gather(-1, rank.clamp(min=0)))
    kept = torch.where(slot[:keep] < n, kept, -1)
    source = torch.where(kept < 0, slot[:keep], kept)[..., None]
    for name in ("k", "v"):
        s[name][:, :, :keep] = s[name].gather(2, source.expand(-1, -1, -1, s[name].shape[-1]))
    return {"kept": kept.to(torch.int32), "lengths": s["lengths"].clamp(max=keep), "k": s["k"], "v": s["v"]}


def exact(case, seed):
    s = prepare({**case}, seed)
    s.pop("op", None)
    return {"rotate": _exact_rotate, "tree": _exact_tree, "accumulate": _exact_accumulate, "accept": _exact_accept,
            "evict": _exact_evict}[case["kind"]](case, s)


def _exact_rotate(case, s):
    # The rotation as a product with a complex unit, one sequence at a time.
    half = case["rotary"] // 2

    def turned(x, gain, at):
        x = x.double()  # [H, T, D]
        if gain is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * gain.double()
        unit = torch.complex(s["cos"][at].double(), s["sin"][at].double())
        front = x[..., : 2 * half]
        pairs = front.unflatten(-1, (2, half)).transpose(-1, -2) if case["layout"] == "half" else \
            front.unflatten(-1, (half, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
        z = z.transpose(-1, -2) if case["layout"] == "half" else z
        return torch.cat([z.flatten(-2), x[..., 2 * half:]], -1)

    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    k, v = s["k"].double(), s["v"].double()
    for b, used in enumerate(_rotate_counts(case)):
        at, n = s["positions"][b, :used].long(), int(s["lengths"][b])
        q[b, :, :used] = turned(s["q"][b, :, :used], s["q_norm"], at)
        k[b, :, n:n + used] = turned(s["k_new"][b, :, :used], s["k_norm"], at)
        v[b, :, n:n + used] = s["v_new"][b, :, :used].double()
    return {"q": q, "k": k, "v": v}


def _exact_rows(case, s):
    """For each sequence: its slots in sight, as scores [Hkv, G, T, n] in 64 bits with -inf where nothing is seen."""
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    for b, (n, c) in enumerate(zip(_shared_lengths(case), _counts(case))):
        q = s["q"][b, :, :c].double().unflatten(0, (kv, group))
        k = s["k"][b, :, : n + c].double()
        x = torch.matmul(q.reshape(kv, group * c, -1), k.mT.contiguous()).reshape(kv, group, c, n + c)
        x /= math.sqrt(case["dim"])
        x[..., n:].masked_fill_(~s["mask"][b, :c, :c], -math.inf)
        yield b, n, c, x


def _exact_tree(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    for b, n, c, x in _exact_rows(case, s):
        lse[b, :, :c] = x.logsumexp(-1).flatten(0, 1)
        p = x.softmax(-1).flatten(1, 2)
        o = torch.matmul(p, s["v"][b, :, : n + c].double())
        out[b, :, :c] = o.unflatten(1, x.shape[1:3]).flatten(0, 1)
    return {"out": out, "lse": lse}


def _exact_accumulate(case, s):
    weights = s["weights"].double()
    for b, n, c, x in _exact_rows(case, s):
        lse = s["lse"][b, :, :c].double().unflatten(0, x.shape[:2])[..., None]
        weights[b, :, : n + c] += ((x - lse).exp() * s["rows"][b, :c, None]).sum((1, 2))
    return weights


def _exact_accept(case, s):
    result = {name: s[name].clone() for name in ("k", "v", "weights", "positions")}
    t = case["drafts"]
    for b, n in enumerate(_accepted(case)):
        at = int(s["lengths"][b])
        for name in result:
            result[name][b, :, at:at + n] = s[name][b, :, at + s["path"][b, :n].long()]
        result["weights"][b, :, at + n:at + t] = 0
    result = {name: x.double() if x.is_floating_point() else x for name, x in result.items()}
    return {"lengths": s["lengths"] + s["accepted"], **result}


def _exact_evict(case, s):
    keep, shape = case["keep"], s["weights"].shape
    weights = s["weights"].cpu().tolist()
    ages = None if s["positions"] is None else s["positions"].cpu().tolist()
    kept = torch.full((*shape[:2], keep), -1, dtype=torch.int32)
    for b, n in enumerate(_evict_lengths(case)):
        for h in range(shape[1]):
            age = range(n) if ages is None else ages[b][h][:n]
            since, w = max(age) - case["recent"], weights[b][h]
            ranked = sorted(range(n), key=lambda i: (age[i] <= since, -w[i], i))
            chosen = set(ranked[:keep])
            movers = iter(sorted(i for i in chosen if i >= keep))
            row = [i if i in chosen else next(movers) for i in range(min(n, keep))]
            kept[b, h, : len(row)] = torch.tensor(row, dtype=torch.int32)
    kept = kept.cuda()
    source = torch.where(kept < 0, torch.arange(keep, device="cuda"), kept.long())
    k, v = s["k"].double(), s["v"].double()
    at = torch.meshgrid(*(torch.arange(x, device="cuda") for x in shape[:2]), indexing="ij")
    moved = (x.clone() for x in (k[at[0][..., None], at[1][..., None], source],
                                 v[at[0][..., None], at[1][..., None], source]))
    k[:, :, :keep], v[:, :, :keep] = moved
    return {"kept": kept, "lengths": s["lengths"].clamp(max=keep), "k": k, "v": v}
