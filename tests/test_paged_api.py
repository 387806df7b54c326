"""Host side of the paged 8-bit cache (no GPU): refusals, schemas, C argument checks, the plain forms against each other."""

import copy
import ctypes
import io
import math

import pytest
import torch

from oracle import paged as op_
from systems_for_llms_amd import _lib, paged

INVALID, UNSUPPORTED = -1, -2


def small(**change):
    """A cache of 2 rows on the CPU, fields replaced as asked."""
    cache = paged.create(2, 48, 2, 64, 7, layers=3, page_size=16, device="cpu")
    fields = {n: getattr(cache, n) for n in ("k", "v", "k_scale", "v_scale", "tables", "lengths", "refs")}
    return paged.PagedCache(**{**fields, **change})


def test_create():
    cache = paged.create(3, 100, 2, 32, 9, layers=4, page_size=32, device="cpu")
    assert cache.k.shape == (4, 9, 2, 32, 32) and cache.k.dtype == torch.float8_e4m3fn
    assert cache.tables.tolist() == [[-1] * 4] * 3 and cache.capacity == 128 and cache.layers == 4 and cache.page_size == 32
    assert not cache.lengths.any() and not cache.refs.any()
    for arguments in (dict(batch=0), dict(capacity=True), dict(kv_heads=2.0), dict(pages=-1), dict(layers=0)):
        with pytest.raises(ValueError, match="positive"):
            paged.create(**{**dict(batch=1, capacity=9, kv_heads=1, head_dim=16, pages=1, device="cpu"), **arguments})
    with pytest.raises(ValueError, match="page sizes"):
        paged.create(1, 9, 1, 16, 1, page_size=8, device="cpu")
    with pytest.raises(ValueError, match="head dimensions"):
        paged.create(1, 9, 1, 48, 1, device="cpu")
    with pytest.raises(ValueError, match="at most 1024 rows"):
        paged.create(1025, 16, 1, 16, 1, page_size=16, device="cpu")


@pytest.mark.parametrize("change, message", [
    (dict(k=torch.zeros(3, 7, 2, 16, 64)), "k must be a contiguous float8_e4m3fn"),
    (dict(v=torch.zeros(3, 7, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)), "v must be"),
    (dict(k_scale=torch.zeros(3, 7, 2, dtype=torch.float64)), "k_scale"), (dict(v_scale=torch.zeros(3, 7, 3)), "v_scale"),
    (dict(tables=torch.zeros(2, 3, dtype=torch.int64)), "tables"), (dict(tables=torch.zeros(6, dtype=torch.int32)), "tables"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"), (dict(refs=torch.zeros(8, dtype=torch.int32)), "refs"),
    (dict(tables=torch.zeros(3, 2, dtype=torch.int32).T), "tables must be a contiguous"),
    (dict(tables=torch.zeros(1, 1, dtype=torch.int32).expand(2, (1 << 26) + 1)), "slots")])
def test_caches_that_are_refused(change, message):
    with pytest.raises(ValueError, match=message):
        small(**change)


def test_cpu_tensors_are_refused_everywhere():
    cache = small()
    new, q = torch.zeros(2, 2, 3, 64), torch.zeros(2, 4, 3, 64)
    counts = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: paged.fork(cache, counts), lambda: paged.reserve(cache, counts), lambda: paged.compact(cache),
                 lambda: paged.append(cache, new, new), lambda: paged.attend(q, cache), lambda: paged.prepare(q, cache)):
        with pytest.raises(ValueError, match="same CUDA"):
            call()


def test_refusals_before_any_launch():
    cache = small()
    counts = torch.zeros(2, dtype=torch.int32)
    new, q = torch.zeros(2, 2, 3, 64), torch.zeros(2, 4, 3, 64)
    for call, error, message in (
            (lambda: paged.fork("cache", counts), TypeError, "PagedCache"),
            (lambda: paged.fork(cache, counts.long()), ValueError, "parents"),
            (lambda: paged.fork(cache, counts[:1]), ValueError, "parents"),
            (lambda: paged.fork(cache, cache.lengths), ValueError, "lengths"),
            (lambda: paged.reserve(cache, counts.float()), ValueError, "counts"),
            (lambda: paged.append(cache, new.double(), new.double()), TypeError, "same FP16"),
            (lambda: paged.append(cache, new, new.half()), TypeError, "same FP16"),
            (lambda: paged.append(cache, new, new[:, :1]), ValueError, "agree"),
            (lambda: paged.append(cache, new[:1], new[:1]), ValueError, "agree"),
            (lambda: paged.append(cache, new[..., :32], new[..., :32]), ValueError, "agree"),
            (lambda: paged.append(cache, new.expand(2, 2, 3, 64).transpose(1, 3), new), ValueError, "head dimensions"),
            (lambda: paged.append(cache, torch.zeros(2, 2, 3, 65)[..., 1:], new), ValueError, "16-byte"),
            (lambda: paged.append(cache, new, new, layer=3), ValueError, "layer"),
            (lambda: paged.append(cache, new, new, layer=True), ValueError, "layer"),
            (lambda: paged.append(cache, new, new, counts=torch.zeros(2)), ValueError, "counts"),
            (lambda: paged.append(cache, new.clone().requires_grad_(), new), RuntimeError, "forward-only"),
            (lambda: paged.append(cache, new[:, :, :0], new[:, :, :0]), ValueError, "empty"),
            (lambda: paged.prepare(q, cache, splits=0), ValueError, "splits"),
            (lambda: paged.prepare(q, cache, splits=129), ValueError, "splits"),
            (lambda: paged.prepare(q, cache, splits=True), ValueError, "splits"),
            (lambda: paged.prepare(q, cache, window_left=-1), ValueError, "window_left"),
            (lambda: paged.prepare(q, cache, window_left=1.5), ValueError, "window_left"),
            (lambda: paged.prepare(q, cache, scale=0.0), ValueError, "scale"),
            (lambda: paged.prepare(q, cache, scale=math.nan), ValueError, "scale"),
            (lambda: paged.prepare(q, cache, layer=-1), ValueError, "layer"),
            (lambda: paged.prepare(q[:, :3], cache), ValueError, "divisible"),
            (lambda: paged.prepare(torch.zeros(2, 6, 3, 64), cache), ValueError, "ratios"),
            (lambda: paged.prepare(torch.zeros(2, 4, 129, 64), cache), ValueError, "at most 128"),
            (lambda: paged.prepare(torch.zeros(1, 4, 3, 64), cache), ValueError, "agree"),
            (lambda: paged.prepare(torch.zeros(2, 4, 3, 32), cache), ValueError, "agree"),
            (lambda: paged.prepare(q[..., ::2], cache), ValueError, "contiguous last"),
            (lambda: paged.prepare(q.long(), cache), TypeError, "same FP16"),
            (lambda: paged.prepare(q, cache, counts=torch.zeros(3, dtype=torch.int32)), ValueError, "counts"),
            (lambda: paged.prepare(q.clone().requires_grad_(), cache), RuntimeError, "forward-only")):
        with pytest.raises(error, match=message):
            call()


def test_auto_splits_bounds():
    bf16, fp16, fp32 = torch.bfloat16, torch.float16, torch.float32
    assert paged.auto_splits(1, 4, 1024, 8, 128, bf16) == 1        # 1024 slots to a split
    assert paged.auto_splits(32, 8, 8192, 4, 128, bf16) == 2       # rows may differ in length
    assert paged.auto_splits(16, 16, 20000, 5, 64, fp16, 4095) == 1  # a window: they do not matter
    assert paged.auto_splits(1, 8, 131072, 4, 128, fp16) == 32
    assert paged.auto_splits(8, 8, 8192, 108, 128, bf16) == 8
    assert paged.auto_splits(8, 8, 8192, 64, 128, bf16) == 2       # two blocks of 32 rows
    assert paged.auto_splits(8, 8, 8192, 64, 128, fp32) == 1       # four of 16
    for args in ((1, 1, 16, 1), (1, 1, 1 << 30, 1024), (1024, 16, 1 << 20, 1024), (1, 1, 1 << 30, 1)):
        for dim, dtype, window in ((16, bf16, None), (128, fp16, 0), (128, fp32, 100)):
            assert 1 <= paged.auto_splits(*args, dim, dtype, window) <= 64


def test_schemas_and_meta_dispatch():
    for name, written in (("page_append", ("k_codes", "v_codes", "k_scale", "v_scale")),
                          ("page_attention", ("partial_max", "partial_output", "out", "lse")),
                          ("page_fork", ("tables", "lengths", "refs")),
                          ("page_reserve", ("k_codes", "tables", "refs", "granted", "scratch")),
                          ("page_compact", ("v_codes", "tables", "refs", "used", "scratch"))):
        schema = str(getattr(torch.ops.sfl, name).default._schema)
        for w in written:
            assert f"!) {w}" in schema, (name, w)
    m = paged.create(2, 48, 2, 64, 7, page_size=16, device="meta")
    new = torch.empty(2, 2, 3, 64, device="meta", dtype=torch.bfloat16)
    q = torch.empty(2, 4, 3, 64, device="meta", dtype=torch.bfloat16)
    n, f = torch.empty(2, device="meta", dtype=torch.int32), torch.empty(2, 4, 3, 2, device="meta")
    torch.ops.sfl.page_append(new, new, m.tables, m.lengths, None, m.refs, m.k, m.v, m.k_scale, m.v_scale, 0)
    torch.ops.sfl.page_attention(q, m.k, m.v, m.k_scale, m.v_scale, m.tables, m.lengths, n, f, f.clone(),
                                 torch.empty(2, 4, 3, 2, 64, device="meta"), torch.empty_like(q),
                                 torch.empty(2, 4, 3, device="meta"), 0, -1, 2, 2, 0.125)
    torch.ops.sfl.page_fork(n, m.tables, m.lengths, m.refs, 16)


def _status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def test_entry_points_refuse_before_any_launch():
    """Argument errors, not the failed launch that a call without a GPU ends with."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libsfl.so not built")

    def strides(change=None):
        values = [64] * 6
        if change is not None:
            values[change[0]] = change[1]
        return (ctypes.c_long * 6)(*values)

    def refused(name, good, cases):
        for change, value, code in cases:
            args = [value if i == change else x for i, x in enumerate(good)]
            assert _status(name, *args) == code, (name, change, value)

    p, f = 64, 1
    append = [p] * 10 + [strides(), 1, 2, 3, 4, 9, 16, 64, f, None]  # batch heads tokens places pages page dim dtype
    refused("sfl_page_append", append, (
        *((i, None, INVALID) for i in (0, 1, 2, 3, 4, 5, 6, 7, 9, 10)), (0, 72, INVALID), (3, 72, INVALID), (11, 0, INVALID),
        (12, 0, INVALID), (13, 0, INVALID), (14, 0, INVALID), (15, -1, INVALID), (16, 24, UNSUPPORTED), (16, 256, UNSUPPORTED),
        (17, 48, UNSUPPORTED), (18, 3, UNSUPPORTED), (14, (1 << 26) + 1, UNSUPPORTED), (15, (1 << 24) + 1, UNSUPPORTED),
        (10, strides((2, 60)), INVALID)))
    assert _status("sfl_page_append", *append[:11], 1 << 20, 1 << 12, *append[13:]) == UNSUPPORTED  # workgroups

    attention = [p] * 13 + [strides(), 1, 4, 2, 3, 4, 9, 16, 64, -1, 1, 1, 0.125, f, None]
    refused("sfl_page_attention", attention, (
        *((i, None, INVALID) for i in (0, 1, 2, 3, 4, 5, 6, 11, 12, 13)), (0, 72, INVALID), (2, 72, INVALID), (11, 72, INVALID),
        (14, 0, INVALID), (15, 3, INVALID), (15, 6, UNSUPPORTED), (17, 129, UNSUPPORTED), (17, 0, INVALID), (18, 0, INVALID),
        (20, 8, UNSUPPORTED), (21, 80, UNSUPPORTED), (23, 0, INVALID), (23, 2, INVALID), (24, 1025, INVALID), (25, -1.0, INVALID),
        (25, math.inf, INVALID), (26, 7, UNSUPPORTED), (13, strides((4, 63)), INVALID)))
    assert _status("sfl_page_attention", *[p] * 8, None, p, p, *attention[11:23], 1, 2, 0.125, f, None) == INVALID  # no scratch

    fork = [p] * 4 + [2, 4, 9, 16, None]
    refused("sfl_page_fork", fork, (*((i, None, INVALID) for i in range(4)), (4, 1025, UNSUPPORTED), (5, 0, INVALID),
                                    (7, 12, UNSUPPORTED)))
    reserve = [p] * 10 + [2, 4, 9, 1, 2, 16, 64, None]
    refused("sfl_page_reserve", reserve, (*((i, None, INVALID) for i in range(10)), (0, 72, INVALID), (10, 1025, UNSUPPORTED),
                                          (13, 0, INVALID), (14, 0, INVALID), (16, 24, UNSUPPORTED)))
    assert _status("sfl_page_reserve", *[p] * 10, 1024, 1 << 26, 1 << 24, 1, 2, 16, 64, None) == UNSUPPORTED  # places
    compact = [p] * 8 + [2, 4, 9, 1, 2, 16, 64, None]
    refused("sfl_page_compact", compact, (*((i, None, INVALID) for i in range(8)), (1, 72, INVALID), (9, 0, INVALID),
                                          (11, 0, INVALID), (14, 8, UNSUPPORTED)))


def test_float64_forms_agree_with_torch_and_the_older_oracle():
    """Rounding is torch's; attention over codes that hold their values exactly is that over a contiguous cache."""
    from oracle import cache as oc

    x = torch.cat([torch.linspace(-448, 448, 40001), torch.linspace(-0.03, 0.03, 20001)]).double()
    assert torch.equal(op_.nearest_code(x), x.float().to(torch.float8_e4m3fn).double())
    for amax, e in ((448.0, 0), (448.5, 1), (224.0, -1), (0.0, -100), (1.0, -8), (1.75, -8), (1.76, -7)):
        assert op_.least_exponent(amax) == e
    g = torch.Generator().manual_seed(1)
    cache = {n: getattr(paged.create(2, 48, 2, 16, 7, page_size=16, device="cpu"), n)
             for n in ("k", "v", "k_scale", "v_scale", "tables", "lengths", "refs")}
    granted, cache = op_.reserve(cache, torch.tensor([40, 20]))
    assert granted.tolist() == [40, 20] and cache["tables"].tolist() == [[0, 1, 2], [3, 4, -1]]
    k, v = (torch.randint(-15, 16, (2, 2, 40, 16), generator=g).float() for _ in range(2))
    cache = op_.append(cache, k, v, granted)
    q = torch.randn(2, 4, 3, 16, generator=g)
    cache["lengths"] = torch.tensor([37, 17], dtype=torch.int32)
    out, lse, _, _ = op_.attention(q, cache)
    want, want_lse, _, _ = oc.tree_attention(q, k, v, cache["lengths"], torch.ones(3, 3, dtype=torch.bool).tril())
    assert (out - want).abs().max() < 1e-12 and (lse - want_lse).abs().max() < 1e-12
    forked = op_.fork(cache, torch.tensor([1, 0]))
    assert forked["tables"].tolist() == [[3, 4, -1], [0, 1, 2]] and forked["refs"].tolist() == [1] * 5 + [0] * 2
    both = op_.fork(cache, torch.tensor([0, 0]))
    granted, both = op_.reserve(both, torch.tensor([1, 1]))
    assert both["tables"].tolist() == [[0, 1, 3], [0, 1, 2]] and both["refs"].tolist() == [2, 2, 1, 1, 0, 0, 0]
    freed = op_.fork(both, torch.tensor([-1, 1]))
    used, packed = op_.compact(op_.fork(freed, torch.tensor([0, 1])))
    assert used == 3 and packed["tables"].tolist() == [[-1] * 3, [0, 1, 2]]


def test_lengths_move_in_place_and_nothing_is_replaced():
    cache = small()
    lengths = cache.lengths
    cache.lengths += torch.tensor([3, 1], dtype=torch.int32)
    assert cache.lengths is lengths and lengths.tolist() == [3, 1]
    for name in ("k", "lengths", "_scratch"):
        with pytest.raises(AttributeError, match="in place"):
            setattr(cache, name, getattr(cache, name).clone())


def test_copies_are_caches_of_their_own():
    cache = small()
    cache.lengths += 5
    file = io.BytesIO()
    torch.save(cache, file)
    file.seek(0)
    for other in (copy.deepcopy(cache), torch.load(file, weights_only=False)):
        assert other.lengths.tolist() == [5, 5] and other.k.shape == cache.k.shape and other._spans != cache._spans
        other.lengths += 1
        assert cache.lengths.tolist() == [5, 5]
        with pytest.raises(ValueError, match="must not share"):
            paged.fork(other, other.lengths)
        with pytest.raises(ValueError, match="same CUDA"):
            paged.fork(other, cache.lengths)


def test_shared_memory_is_refused():
    cache = small()
    books = torch.zeros(20, dtype=torch.int32)
    small(tables=books[:6].view(2, 3), lengths=books[6:8], refs=books[8:15])
    for lengths, refs in ((books[4:6], books[8:15]), (books[6:8], books[7:14]), (books[:2], books[8:15])):
        with pytest.raises(ValueError, match="share memory"):
            small(tables=books[:6].view(2, 3), lengths=lengths, refs=refs)
    with pytest.raises(ValueError, match="share memory"):
        small(v_scale=cache.k_scale, k_scale=cache.k_scale)
    for vector in (cache.lengths, cache.refs[3:5], cache.tables.view(-1)[1:3], cache.k_scale.view(-1).view(torch.int32)[7:9]):
        with pytest.raises(ValueError, match="parents must not share"):
            paged.fork(cache, vector)
        with pytest.raises(ValueError, match="counts must not share"):
            paged.reserve(cache, vector)


def test_most_splits_bounds():
    bf16, fp16, fp32 = torch.bfloat16, torch.float16, torch.float32
    for size, most in (((32, 8, 8192, 4, 128, bf16), 2),         # rows of up to 8192 slots: nothing to win
                       ((32, 8, 131072, 4, 128, bf16), 34),      # 256 more workgroups of 8 heads
                       ((1, 8, 131072, 4, 128, bf16), 32),       # a sequence alone has all of them
                       ((8, 8, 8192, 108, 128, fp16), 8), ((8, 8, 32768, 108, 128, fp16), 40),
                       ((32, 8, 131072, 4, 128, bf16, 4095), 1), ((600, 1, 9024, 1, 128, fp16), 64)):
        splits = paged.auto_splits(*size)
        assert paged.auto_most_splits(splits, *size) == most
    for batch in (2, 64, 1024):
        for rows in (1, 40, 100, 1024):
            for dtype in (bf16, fp32):
                size = (batch, 8, 1 << 20, rows, 128, dtype)
                splits = paged.auto_splits(*size)
                most = paged.auto_most_splits(splits, *size)
                # No sequence can need more: the further workgroups are 256, a block of a head's rows each.
                assert splits <= most <= 64


def test_attention_of_more_threads_than_a_launch_holds_is_refused():
    """2^23 workgroups of 512 threads, and as many of the kernels of 256 threads as reach 2^32."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libsfl.so not built")

    def status(batch, heads, kv_heads, tokens, dim, splits, dtype):
        strides = (ctypes.c_long * 6)(*[64] * 6)
        return _status("sfl_page_attention", *[64] * 13, strides, batch, heads, kv_heads, tokens, 4, 9, 16, dim, -1, splits,
                       splits, 0.125, dtype, None)

    fp32, bf16, fp16 = 0, 1, 2
    assert status(1024, 64, 64, 1, 64, 128, bf16) == UNSUPPORTED      # 2^23 of 8 waves
    assert status(1024, 64, 64, 1, 64, 128, fp32) == UNSUPPORTED
    assert status(512, 128, 16, 128, 64, 16, fp32) == UNSUPPORTED     # 64 blocks of rows
    assert status(1024, 128, 64, 20, 128, 128, bf16) == UNSUPPORTED   # 2^24 of 4 waves, blocks of 32 rows
    assert status(1024, 64, 64, 128, 128, 256, fp16) == UNSUPPORTED   # 2^24 of 4 waves, blocks of 128 rows


def test_append_from_the_memory_that_it_writes_is_refused():
    """Tokens or counts that overlap the layer's pages or scales; those beside them are not."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libsfl.so not built")
    if torch.cuda.is_available():
        pytest.skip("calls that are not refused here must not reach a GPU: their addresses are none")
    page, heads, dim, pages, batch, tokens = 16, 2, 64, 9, 3, 5
    pool, scales, row, lane = pages * heads * page * dim, 4 * pages * heads, 2 * dim, 2 * dim * heads
    base = 1 << 20
    at = dict(k_codes=base, v_codes=2 * base, k_scale=3 * base, v_scale=4 * base, k=5 * base, v=6 * base, counts=7 * base)
    size = 2 * ((batch * tokens * heads - 1) * dim + dim)  # tokens as a projection leaves them: [B, T, H, D]

    def refused(**moved):
        x = {**at, **moved}
        strides = (ctypes.c_long * 6)(*[lane // 2 * tokens, dim, lane // 2] * 2)
        status = _status("sfl_page_append", x["k"], x["v"], x["k_codes"], x["v_codes"], x["k_scale"], x["v_scale"], 64, 64,
                         x["counts"], 64, strides, batch, heads, tokens, 4, pages, page, dim, 1, None)
        return status == INVALID and b"share memory" in _lib.lib().sfl_last_error()

    for name, extent in (("k_codes", pool), ("v_codes", pool), ("k_scale", scales), ("v_scale", scales)):
        for new in ("k", "v"):
            assert refused(**{new: at[name]}) and refused(**{new: at[name] + (extent - 1) // 16 * 16})
            assert refused(**{new: at[name] - size + 16})
        assert refused(counts=at[name]) and refused(counts=at[name] + extent - 4) and refused(counts=at[name] - 4 * batch + 4)
    for name, extent in (("k_codes", pool), ("v_scale", scales)):  # these end with the launch that fails without a GPU
        assert not refused(k=at[name] + -(-extent // 16) * 16) and not refused(v=at[name] - size)
        assert not refused(counts=at[name] + extent) and not refused(counts=at[name] - 4 * batch)
    assert not refused() and not refused(counts=None)


def test_a_page_that_was_never_written_holds_no_scale():
    """Behind committed tokens of a page whose scale is still 0 the new tokens alone choose it."""
    cache = paged.create(1, 48, 1, 16, 3, page_size=16, device="cpu")
    state = {n: getattr(cache, n) for n in ("k", "v", "k_scale", "v_scale", "tables", "lengths", "refs")}
    _, state = op_.reserve(state, torch.tensor([20]))
    state["lengths"] = torch.tensor([5], dtype=torch.int32)
    new = torch.full((1, 1, 3, 16), 2.0 ** -20)
    done = op_.append(state, new, 4 * new)
    assert done["k_scale"][0, 0, 0] == 2.0 ** -28 and done["v_scale"][0, 0, 0] == 2.0 ** -26
    assert torch.equal(done["k"][0, 0, 0, 5:8].float(), torch.full((3, 16), 256.0)) and not done["k"][0, 0, 0, :5].float().any()


def test_what_codes_hold_of_the_values_that_were_appended():
    """Off by 2^-4 of the value or 2^-10 of the scale under the scale they were appended with; where it grew afterwards,
    by 2^-4 of the value and less than 2^-9 of the scale: each rounding of a small code adds 2^-10 of a scale at most half the next."""
    g = torch.Generator().manual_seed(3)
    worst = 0.0
    for trial in range(60):
        cache = paged.create(1, 32, 1, 32, 1, page_size=32, device="cpu")
        state = {n: getattr(cache, n) for n in ("k", "v", "k_scale", "v_scale", "tables", "lengths", "refs")}
        _, state = op_.reserve(state, torch.tensor([32]))
        given = []
        size = 1.0
        for _ in range(8):
            x = torch.randn(1, 1, 4, 32, generator=g) * torch.exp2(-torch.randint(0, 18, (1, 1, 4, 32), generator=g).float()) * size
            state = op_.append(state, x, x)
            given.append(x)
            state["lengths"] = state["lengths"] + 4
            want, unit = torch.cat(given, 2)[0].double(), float(state["k_scale"][0, 0, 0])
            held = op_.rows_of(state, 0, range(want.shape[1]))
            assert torch.equal(held[0], held[1])
            off = (held[0] - want).abs()
            assert bool((off[:, -4:] <= torch.maximum(2.0 ** -4 * want.abs(), torch.tensor(2.0 ** -10 * unit))[:, -4:]).all())
            assert bool((off <= 2.0 ** -4 * want.abs() + 2.0 ** -9 * unit).all())
            worst = max(worst, float((off / torch.maximum(2.0 ** -4 * want.abs(), torch.tensor(2.0 ** -10 * unit))).max()))
            size *= float(torch.randint(1, 4, (), generator=g))
    assert worst > 1.3  # once rounded again, values are further off than one rounding says


def test_auto_splits_leave_768_slots_each():
    """Capacities between the multiples of 1024: the number of splits is the nearest one."""
    for reach, splits in ((1, 1), (1535, 1), (1537, 2), (2559, 2), (2561, 3), (3583, 3), (3585, 4), (66000, 64)):
        assert paged.auto_splits(1, 1, reach, 1, 128, torch.bfloat16) == splits
        assert paged.auto_splits(1, 1, 1 << 20, 1, 128, torch.bfloat16, reach - 1) == splits
    for reach in range(1, 9000):
        splits = paged.auto_splits(1, 1, reach, 1, 128, torch.bfloat16)
        assert splits == 1 or reach // splits >= 768
