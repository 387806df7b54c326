"""Host side of the KV-cache operators (no GPU): tables, masks, refusals, schemas, C argument checks."""

import ctypes
import math

import pytest
import torch

from systems_for_llms_amd import _lib, evict, rotary, tree


def test_tables_hold_the_angle_of_far_positions():
    cos, sin = rotary.rotary_tables(64, 131072)
    for p, i in ((0, 0), (131071, 0), (131071, 3), (100003, 31)):
        angle = p * 10000.0 ** (-2 * i / 64)
        assert abs(float(cos[p, i]) - math.cos(angle)) < 1e-7 and abs(float(sin[p, i]) - math.sin(angle)) < 1e-7


def test_unscaled_tables_agree_with_the_models():
    from systems_for_llms_amd.model import rope_tables

    cos, sin = rotary.rotary_tables(32, 300)
    want = rope_tables(10000.0, 32, 300)  # angles in fp32: off by 300 * 2^-24
    assert (cos - want[0]).abs().max() < 3e-5 and (sin - want[1]).abs().max() < 3e-5


def _angles(table):
    """Angles of position 1 from the tables (below pi)."""
    return torch.atan2(table[1][1].double(), table[0][1].double())


def test_scalings_change_the_frequencies_they_say():
    plain = _angles(rotary.rotary_tables(32, 2))
    linear = _angles(rotary.rotary_tables(32, 2, scaling="linear", factor=4.0))
    assert torch.allclose(linear, plain / 4, rtol=1e-6)
    base = _angles(rotary.rotary_tables(32, 2, scaling="base", factor=4.0))
    assert torch.allclose(base[0], plain[0], rtol=1e-6) and torch.allclose(base[-1], plain[-1] / 4, rtol=1e-5)
    ramp = _angles(rotary.rotary_tables(32, 2, scaling="ramp", factor=4.0, original_positions=2048))
    turns = 2048 * plain / (2 * math.pi)
    assert torch.allclose(ramp[turns >= 32], plain[turns >= 32], rtol=1e-6)
    assert torch.allclose(ramp[turns <= 1], plain[turns <= 1] / 4, rtol=1e-5)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((ramp < plain) & (ramp > plain / 4))[between].all()
    cos, _ = rotary.rotary_tables(32, 2, magnitude=1.5)
    assert float(cos[0, 0]) == 1.5


@pytest.mark.parametrize("arguments, message", [
    (dict(rotary_dim=7, positions=4), "even"), (dict(rotary_dim=0, positions=4), "positive"),
    (dict(rotary_dim=8, positions=4, theta=0.0), "theta"), (dict(rotary_dim=8, positions=4, scaling="other"), "scaling"),
    (dict(rotary_dim=8, positions=4, scaling="ramp"), "original_positions"),
    (dict(rotary_dim=8, positions=4, scaling="ramp", original_positions=9, low=5.0, high=5.0), "low < high"),
    (dict(rotary_dim=2, positions=4, scaling="base", factor=2.0), "above 2"),
    (dict(rotary_dim=8, positions=4, factor=math.inf), "factor")])
def test_tables_refuse(arguments, message):
    with pytest.raises(ValueError, match=message):
        rotary.rotary_tables(**arguments)


def test_ancestor_mask():
    parents = torch.tensor([[-1, 0, 0, 2, -1], [-1, -1, 1, 2, 3]])
    want = torch.zeros(2, 5, 5, dtype=torch.bool)
    for b in range(2):
        for t in range(5):
            at = t
            while at >= 0:
                want[b, t, at] = True
                at = int(parents[b, at])
    assert torch.equal(tree.ancestor_mask(parents), want)
    assert torch.equal(tree.ancestor_mask(parents[1]), want[1])
    for bad in (torch.tensor([0]), torch.tensor([-2]), torch.tensor([-1, 1])):
        with pytest.raises(ValueError, match="parent"):
            tree.ancestor_mask(bad)
    with pytest.raises(ValueError, match="integer"):
        tree.ancestor_mask(torch.tensor([-1.0]))


def _tree(batch=2, heads=8, kv_heads=2, tokens=3, keys=40, dim=64, dtype=torch.float16):
    q = torch.zeros(batch, heads, tokens, dim, dtype=dtype)
    k = torch.zeros(batch, kv_heads, keys, dim, dtype=dtype)
    return dict(q=q, k=k, v=k.clone(), lengths=torch.zeros(batch, dtype=torch.int32))


@pytest.mark.parametrize("change, error, message", [
    (dict(), ValueError, "same CUDA"), (dict(splits=0), ValueError, "splits"), (dict(splits=True), ValueError, "splits"),
    (dict(q=torch.zeros(2, 8, 64)), ValueError, r"\[B, H, rows, D\]"),
    (dict(q=torch.zeros(2, 8, 3, 64)), TypeError, "same FP16"),
    (dict(q=torch.zeros(2, 8, 3, 64, dtype=torch.float64)), TypeError, "same FP16"),
    (dict(q=torch.zeros(2, 8, 3, 64, dtype=torch.float16, requires_grad=True)), RuntimeError, "forward-only")])
def test_tree_refusals_before_any_launch(change, error, message):
    with pytest.raises(error, match=message):
        tree.prepare(**{**_tree(), **change})


def test_cpu_tensors_are_refused_everywhere():
    t = _tree()
    q, k, lengths = t["q"], t["k"], t["lengths"]
    cos, sin = rotary.rotary_tables(64, 16)
    positions = torch.zeros(2, 3, dtype=torch.int32)
    new = torch.zeros(2, 2, 3, 64, dtype=torch.float16)
    weights = torch.zeros(2, 2, 40)
    path = torch.zeros(2, 3, dtype=torch.int32)
    calls = (lambda: rotary.rotate(q, new, positions, cos, sin),
             lambda: rotary.rotate_append(q, new, new, positions, cos, sin, k, k.clone(), lengths),
             lambda: tree.attend(q, k, k, lengths), lambda: tree.accept(k, k.clone(), lengths, path, lengths),
             lambda: tree.accumulate(q, k, torch.zeros(2, 8, 3), weights, lengths),
             lambda: evict.select(weights, lengths, 8), lambda: evict.evict(k, k.clone(), weights, lengths, 8),
             lambda: evict.compact(torch.zeros(2, 2, 8, dtype=torch.int32), k, k.clone()))
    for call in calls:
        with pytest.raises(ValueError, match="same CUDA"):
            call()


def test_rotary_refusals():
    t = _tree()
    new = torch.zeros(2, 2, 3, 64, dtype=torch.float16)
    cos, sin = rotary.rotary_tables(64, 16)
    good = dict(q=t["q"], k=new, positions=torch.zeros(2, 3, dtype=torch.int32), cos=cos, sin=sin)
    gain = torch.ones(64, dtype=torch.float16)
    for change, error, message in (
            (dict(layout="other"), ValueError, "layout"), (dict(eps=-1.0), ValueError, "eps"),
            (dict(positions=good["positions"].long()), ValueError, "positions"),
            (dict(cos=cos.half()), ValueError, "cos"), (dict(cos=torch.ones(16, 33), sin=torch.ones(16, 33)), ValueError, "rotary_dim"),
            (dict(k=new[:1]), ValueError, "agree"), (dict(k=new.float()), TypeError, "same FP16"),
            (dict(q_norm=gain[:32]), ValueError, "gains"), (dict(q_norm=gain.bfloat16()), ValueError, "gains"),
            (dict(q_norm=gain, k_norm=gain.float()), ValueError, "same dtype"),
            (dict(q_norm=gain.float().requires_grad_()), RuntimeError, "forward-only"),
            (dict(counts=torch.zeros(2)), ValueError, "counts"),
            (dict(q=t["q"][..., ::2], k=new[..., ::2]), ValueError, "contiguous last"),
            (dict(q=t["q"][..., :48], k=new[..., :48]), ValueError, "head dimensions")):
        with pytest.raises(error, match=message):
            rotary.rotate(**{**good, **change})


def test_select_refusals():
    weights, lengths = torch.zeros(1, 2, 40), torch.zeros(1, dtype=torch.int32)
    for arguments, error, message in (
            ((weights, lengths, 0), ValueError, "keep"), ((weights, lengths, 41), ValueError, "keep"),
            ((weights, lengths, True), TypeError, "keep"), ((weights, lengths, 8.0), TypeError, "keep"),
            ((weights.half(), lengths, 8), ValueError, "float32"), ((weights, lengths.long(), 8), ValueError, "lengths"),
            ((weights.clone().requires_grad_(), lengths, 8), RuntimeError, "forward-only")):
        with pytest.raises(error, match=message):
            evict.select(*arguments)
    with pytest.raises(ValueError, match="recent"):
        evict.select(weights, lengths, 8, recent=9)
    with pytest.raises(ValueError, match="at most"):
        evict.select(torch.zeros(1, 1, evict.MAX_SLOTS + 1), lengths, 8)


def test_auto_splits_bounds():
    bf16, fp32 = torch.bfloat16, torch.float32
    assert tree.auto_splits(1, 4, 1024, 8, 128, bf16) == 8      # 128 keys to a split
    assert tree.auto_splits(1, 4, 65536, 512, 128, bf16) == 32  # 4 row blocks of 4 heads, 512 workgroups
    assert tree.auto_splits(8, 8, 8191, 108, 128, bf16) == 8
    assert tree.auto_splits(64, 16, 16384, 16, 64, bf16) == 1
    assert tree.auto_splits(2, 4, 8192, 64, 128, fp32) == 16    # four row blocks in fp32
    assert tree.auto_splits(14, 4, 2735, 352, 64, bf16) == 3    # 168 row blocks: three rounds fit at once
    for args in ((1, 1, 1, 1), (1, 4, 65536, 512), (128, 16, 100, 1024), (1, 1, 1 << 20, 1)):
        for dim, dtype in ((16, bf16), (128, bf16), (128, fp32)):
            assert 1 <= tree.auto_splits(*args, dim, dtype) <= 32


def test_schemas_and_meta_dispatch():
    for name, written in (("rotate", ("q_out", "k_out")), ("tree_attention", ("out", "lse", "partial_max")),
                          ("tree_weights", ("weights",)), ("accept_path", ("k", "v", "new_lengths")),
                          ("select_slots", ("kept", "new_lengths")), ("compact_slots", ("k", "v"))):
        schema = str(getattr(torch.ops.sfl, name).default._schema)
        for w in written:
            assert f"!) {w}" in schema, (name, w)
    q = torch.empty(1, 4, 2, 64, device="meta", dtype=torch.bfloat16)
    k = torch.empty(1, 2, 16, 64, device="meta", dtype=torch.bfloat16)
    n = torch.empty(1, device="meta", dtype=torch.int32)
    f = torch.empty(1, 4, 2, 1, device="meta")
    mask = torch.empty(1, 2, 2, device="meta", dtype=torch.bool)
    torch.ops.sfl.tree_attention(q, k, k, n, mask, None, f, f.clone(), torch.empty(1, 4, 2, 1, 64, device="meta"),
                                 torch.empty_like(q), torch.empty(1, 4, 2, device="meta"), 1, 0.125)
    w = torch.empty(1, 2, 16, device="meta")
    torch.ops.sfl.select_slots(w, n, None, torch.empty(1, 2, 8, device="meta", dtype=torch.int32), n.clone(), 2)


def test_float64_forms_agree_with_the_older_oracles():
    """One draft that sees itself is decode attention over one key more; weights of a row add up to one."""
    from oracle import cache as oc
    from oracle.attention import decode_reference

    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 8, 1, 16, generator=g)
    k, v = torch.randn(2, 3, 2, 20, 16, generator=g)
    lengths = torch.tensor([0, 7, 19], dtype=torch.int32)
    mask = torch.ones(1, 1, dtype=torch.bool)
    out, lse, _, _ = oc.tree_attention(q, k, v, lengths, mask)
    want = decode_reference(q[:, :, 0], k, v, lengths + 1)
    assert (out[:, :, 0] - want).abs().max() < 1e-5  # the older one works in float32
    weights, _ = oc.tree_weights(q, k, lse, torch.zeros(3, 2, 20), lengths, mask)
    assert (weights.sum(-1) - 4).abs().max() < 1e-12
    kept, _ = oc.select(torch.tensor([[[3.0, 1.0, 2.0, 2.0, 5.0]]]), torch.tensor([5]), 3, 1)
    assert kept.tolist() == [[[0, 4, 2]]]


INVALID, UNSUPPORTED = -1, -2


def _status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def test_entry_points_refuse_before_any_launch():
    """Argument errors, not the failed launch that a call without a GPU ends with."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libsfl.so not built")

    def strides(n, change=None):
        values = [64] * n
        if change is not None:
            values[change[0]] = change[1]
        return (ctypes.c_long * n)(*values)

    p, f = 64, 1
    tree_tail = (1, 4, 2, 16, 3, 64, 1, 0.125, f, None)

    def attention(change=None, value=None, st=None):
        args = [p] * 11 + [st or strides(15), *tree_tail]
        if change is not None:
            args[change] = value
        return _status("sfl_tree_attention", *args)

    for change, value, code in ((0, None, INVALID), (1, None, INVALID), (2, None, INVALID), (3, None, INVALID),
                                (4, None, INVALID), (9, None, INVALID), (10, None, INVALID), (0, 72, INVALID),
                                (2, 72, INVALID), (12, 0, INVALID), (13, 3, INVALID), (13, 6, UNSUPPORTED),
                                (15, 0, INVALID), (16, 129, UNSUPPORTED), (17, 48, UNSUPPORTED), (18, 0, INVALID),
                                (18, 1025, INVALID), (19, 0.0, INVALID), (19, math.nan, INVALID), (20, 3, UNSUPPORTED)):
        assert attention(change, value) == code, (change, value)
    assert attention(st=strides(15, (5, 63))) == INVALID
    args = [p] * 6 + [None] * 3 + [p] * 2 + [strides(15), 1, 4, 2, 16, 3, 64, 2, 0.125, f, None]
    assert _status("sfl_tree_attention", *args) == INVALID  # splits without scratch

    weights = [p] * 8 + [strides(15), 1, 4, 2, 16, 3, 64, 0.125, f, None]
    for change, value, code in ((3, None, INVALID), (13, 200, UNSUPPORTED), (16, 7, UNSUPPORTED)):
        assert _status("sfl_tree_weights", *[value if i == change else x for i, x in enumerate(weights)]) == code

    rotate = [p] * 13 + [strides(18), 1, 3, 4, 2, 64, 64, 16, 16, 0, f, 1e-5, f, None]
    for change, value, code in ((0, None, INVALID), (3, None, INVALID), (12, None, INVALID), (15, 0, INVALID),
                                (18, 80, UNSUPPORTED), (19, 66, INVALID), (19, 3, INVALID), (23, 2, UNSUPPORTED),
                                (24, -1.0, INVALID), (25, 9, UNSUPPORTED)):
        assert _status("sfl_rotate", *[value if i == change else x for i, x in enumerate(rotate)]) == code, change

    accept = [p] * 8 + [strides(6), 1, 2, 16, 3, 64, f, None]
    for change, value, code in ((0, None, INVALID), (7, None, INVALID), (1, 72, INVALID), (12, 129, UNSUPPORTED),
                                (12, 0, UNSUPPORTED), (13, 8, UNSUPPORTED)):
        assert _status("sfl_accept_path", *[value if i == change else x for i, x in enumerate(accept)]) == code, change
    assert _status("sfl_accept_path", *accept[:8], strides(6, (2, 60)), *accept[9:]) == INVALID

    select = [p] * 5 + [1, 2, 16, 4, 1, None]
    for change, value, code in ((0, None, INVALID), (3, None, INVALID), (7, evict.MAX_SLOTS + 1, UNSUPPORTED),
                                (8, 0, INVALID), (8, 17, INVALID), (9, 5, INVALID), (9, -1, INVALID)):
        assert _status("sfl_select_slots", *[value if i == change else x for i, x in enumerate(select)]) == code, change

    compact = [p] * 5 + [strides(6), 1, 2, 16, 4, 64, f, None]
    for change, value, code in ((4, None, INVALID), (9, 17, INVALID), (10, 24, UNSUPPORTED), (11, 5, UNSUPPORTED)):
        assert _status("sfl_compact_slots", *[value if i == change else x for i, x in enumerate(compact)]) == code, change


def test_caches_of_more_slots_than_the_kernels_count_are_refused():
    """2^30 rows: an expanded view has that many without holding them."""
    from systems_for_llms_amd.cache import MAX_ROWS

    t = _tree()
    lengths, path = t["lengths"], torch.zeros(2, 3, dtype=torch.int32)
    new = torch.zeros(2, 2, 3, 64, dtype=torch.float16)
    cos, sin = rotary.rotary_tables(64, 16)
    for rows in (MAX_ROWS + 1, 2 ** 31 - 1, 2 ** 32 + 40):
        k = torch.zeros(1, 1, 1, 64, dtype=torch.float16).expand(2, 2, rows, 64)
        for call in (lambda: tree.prepare(t["q"], k, k, lengths),
                     lambda: tree.accumulate(t["q"], k, torch.zeros(2, 8, 3), torch.zeros(2, 2, 40), lengths),
                     lambda: tree.accept(k, k, lengths, path, lengths),
                     lambda: evict.compact(torch.zeros(2, 2, 8, dtype=torch.int32), k, k),
                     lambda: rotary.rotate_append(t["q"], new, new, path, cos, sin, k, k, lengths)):
            with pytest.raises(ValueError, match="rows"):
                call()
    if not _lib.LIB_PATH.exists():
        pytest.skip("libsfl.so not built")
    many, p, f = MAX_ROWS + 1, 64, 1
    strides = (ctypes.c_long * 18)(*[64] * 18)
    assert _status("sfl_tree_attention", *[p] * 11, strides, 1, 4, 2, many, 3, 64, 1, 0.125, f, None) == UNSUPPORTED
    assert _status("sfl_tree_weights", *[p] * 8, strides, 1, 4, 2, many, 3, 64, 0.125, f, None) == UNSUPPORTED
    assert _status("sfl_accept_path", *[p] * 8, strides, 1, 2, many, 3, 64, f, None) == UNSUPPORTED
    assert _status("sfl_compact_slots", *[p] * 5, strides, 1, 2, many, 4, 64, f, None) == UNSUPPORTED
    assert _status("sfl_rotate", *[p] * 13, strides, 1, 3, 4, 2, 64, 64, 16, many, 0, f, 1e-5, f, None) == UNSUPPORTED


def test_append_of_k_and_v_to_the_same_rows_is_refused():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libsfl.so not built")
    p, f = 64, 1
    strides = (ctypes.c_long * 18)(*[64] * 18)
    tail = (strides, 1, 3, 4, 2, 64, 64, 16, 16, 0, f, 1e-5, f, None)
    assert _status("sfl_rotate", *[p] * 11, 4096, 4096, *tail) == INVALID
