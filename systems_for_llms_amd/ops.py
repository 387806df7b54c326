"""The library's operators as ``torch.library`` custom ops (namespace ``sfl``).

The drop-in operator APIs (``decode.prepare/decode``, ``attention.attention``)
validate their arguments with the reference's messages and then launch
through these ops, so the launches are visible to PyTorch (dispatcher,
``torch.compile`` graphs, fake-tensor tracing) as ops that write into
caller-owned outputs, like the reference's JIT extension
(``attention_lab/cuda_decode/decode.cu:213-256``). Each op is a thin ctypes
call into ``libsfl.so`` on the caller's current stream; there is no CPU
implementation, and a missing library raises.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib


# Leaves out the dispatch keys of autograd and version counting for a ``with`` block; None where torch lacks it.
_below_autograd = getattr(torch._C, "_AutoDispatchBelowADInplaceOrView", None)


def dispatch(op, tensors: tuple, written: tuple, *rest, checked: bool = False) -> None:
    """``op(*tensors, *rest)``, below the custom op's autograd layers where they would do nothing.

    The op goes through the dispatcher either way, so whatever watches or
    transforms it (dispatch and function modes, tracing, functorch transforms,
    the profiler and its observers, lazily negated tensors) takes part. Its
    autograd and version-counting layers are Python, 10 of the 19 us of a call:
    where no tensor requires grad they only count the versions of the
    ``written`` tensors, which is done here. ``checked``: the caller has refused tensors
    that require grad.
    """
    if _below_autograd is None or torch.compiler.is_compiling() or not checked and _any_requires_grad(tensors):
        op(*tensors, *rest)
        return
    with _below_autograd():
        op(*tensors, *rest)
    mark_written(*written)


def _any_requires_grad(tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def mark_written(*tensors: torch.Tensor | None) -> None:
    """Bump the version counters of tensors an op wrote, as its own layers do (inference tensors have none)."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])


def _strides(t: torch.Tensor):
    return (ctypes.c_long * 3)(t.stride(0), t.stride(1), t.stride(2))


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def launch_decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor,
                            partial_max: torch.Tensor, partial_sum: torch.Tensor, partial_output: torch.Tensor,
                            out: torch.Tensor, splits: int, scale: float) -> None:
    """Split-KV decode attention into ``out`` [B, Hq, D] (``sfl_decode_attention``).

    ``partial_*`` are the fp32 split scratch ([B, Hq, splits] and
    [B, Hq, splits, D]); ``out`` has q's dtype.
    """
    batch, heads, dim = q.shape
    kv_heads, capacity = k.shape[1], k.shape[2]
    code = _lib.dtype_code(q.dtype)
    _lib.call("sfl_decode_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths.data_ptr(),
              partial_max.data_ptr(), partial_sum.data_ptr(), partial_output.data_ptr(), out.data_ptr(),
              batch, heads, kv_heads, capacity, dim, splits, scale, code, code, code,
              _lib.stream_handle(q.device))


decode_attention = torch.library.custom_op(
    "sfl::decode_attention", mutates_args=("partial_max", "partial_sum", "partial_output", "out"))(
        launch_decode_attention)


@decode_attention.register_fake
def _decode_attention_fake(q, k, v, lengths, partial_max, partial_sum, partial_output, out, splits, scale):
    return None


def launch_masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                            lse: torch.Tensor | None, scale: float, causal: bool, window_left: int,
                            window_right: int, global_prefix: int, document_ids: torch.Tensor | None,
                            row_ptr: torch.Tensor | None, col_idx: torch.Tensor | None,
                            full_blocks: torch.Tensor | None, use_full_blocks: bool) -> None:
    """Masked attention of [B, H, N, D] q/k/v into ``out`` (and natural-log ``lse``).

    Windows are ``-1`` when unbounded. With ``row_ptr`` the kernel walks that
    64 x 64 CSR schedule; without it, the interval schedule of the mask.
    """
    batch, heads, length, dim = q.shape
    mode = 1 if row_ptr is not None else 0
    _lib.call("sfl_masked_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse),
              batch, heads, length, dim, _strides(q), _strides(k), _strides(v), _strides(out), scale,
              int(causal), window_left, window_right, global_prefix, _ptr(document_ids), mode,
              _ptr(row_ptr), _ptr(col_idx), _ptr(full_blocks), int(use_full_blocks),
              _lib.dtype_code(q.dtype), _lib.stream_handle(q.device))


masked_attention = torch.library.custom_op("sfl::masked_attention", mutates_args=("out", "lse"))(
    launch_masked_attention)


@masked_attention.register_fake
def _masked_attention_fake(q, k, v, out, lse, scale, causal, window_left, window_right, global_prefix,
                           document_ids, row_ptr, col_idx, full_blocks, use_full_blocks):
    return None


_NO_STRIDES = (0, 0, 0)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without building a Stream object
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(device: torch.device, name: str, *args) -> None:
    """The entry point on ``device``'s current stream, with that device current."""
    index = device.index
    if index != _current_device():
        with torch.cuda.device(device):
            _lib.call(name, *args, _lib.stream_handle(device))
        return
    _lib.call(name, *args, _lib.stream_handle(device) if _raw_stream is None else _raw_stream(index))


# Strides of several tensors {batch, head, row} as the array of longs the entry points take.
_strides_2, _strides_5, _strides_6 = (struct.Struct(f"{3 * n}l").pack for n in (2, 5, 6))


def launch_rotate(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, positions: torch.Tensor,
                  cos: torch.Tensor, sin: torch.Tensor, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None,
                  start: torch.Tensor | None, counts: torch.Tensor | None, q_out: torch.Tensor, k_out: torch.Tensor,
                  v_out: torch.Tensor | None, half_layout: bool, eps: float) -> None:
    """Norm and rotation of q and k rows; k and v into a cache where ``start`` says so (``sfl_rotate``)."""
    batch, heads, tokens, dim = q.shape
    strides = _strides_6(*q.stride()[:3], *k.stride()[:3], *(_NO_STRIDES if v is None else v.stride()[:3]),
                         *q_out.stride()[:3], *k_out.stride()[:3], *(_NO_STRIDES if v is None else v_out.stride()[:3]))
    gain = q.dtype if q_norm is None and k_norm is None else (k_norm if q_norm is None else q_norm).dtype
    _call(q.device, "sfl_rotate", q.data_ptr(), k.data_ptr(), _ptr(v), positions.data_ptr(), cos.data_ptr(),
          sin.data_ptr(), _ptr(q_norm), _ptr(k_norm), _ptr(start), _ptr(counts), q_out.data_ptr(), k_out.data_ptr(),
          _ptr(v_out), strides, batch, tokens, heads, k.shape[1], dim,
          2 * cos.shape[1], cos.shape[0], k_out.shape[2], int(half_layout), _lib.dtype_code(gain), eps,
          _lib.dtype_code(q.dtype))


def launch_tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor,
                          mask: torch.Tensor, counts: torch.Tensor | None, partial_max: torch.Tensor,
                          partial_sum: torch.Tensor, partial_output: torch.Tensor, out: torch.Tensor,
                          lse: torch.Tensor, splits: int, scale: float) -> None:
    """Attention of drafted tokens over a cache into ``out`` and ``lse`` (``sfl_tree_attention``).

    ``mask`` is [B, T, T] (an expanded [T, T] has a batch stride of 0).
    """
    batch, heads, tokens, dim = q.shape
    _call(q.device, "sfl_tree_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths.data_ptr(),
          mask.data_ptr(), _ptr(counts), partial_max.data_ptr(), partial_sum.data_ptr(), partial_output.data_ptr(),
          out.data_ptr(), lse.data_ptr(),
          _strides_5(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *mask.stride()), batch, heads, k.shape[1], k.shape[2],
          tokens, dim, splits, scale, _lib.dtype_code(q.dtype))


def launch_tree_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, lengths: torch.Tensor,
                        mask: torch.Tensor, counts: torch.Tensor | None, rows: torch.Tensor | None,
                        weights: torch.Tensor, scale: float) -> None:
    """Attention weights of the counted drafts added to ``weights`` by slot (``sfl_tree_weights``)."""
    batch, heads, tokens, dim = q.shape
    _call(q.device, "sfl_tree_weights", q.data_ptr(), k.data_ptr(), lse.data_ptr(), weights.data_ptr(),
          lengths.data_ptr(), mask.data_ptr(), _ptr(counts), _ptr(rows),
          _strides_5(*q.stride()[:3], *k.stride()[:3], *_NO_STRIDES, *_NO_STRIDES, *mask.stride()), batch, heads, k.shape[1], k.shape[2], tokens, dim, scale, _lib.dtype_code(q.dtype))


def launch_accept_path(lengths: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor, k: torch.Tensor,
                       v: torch.Tensor, weights: torch.Tensor | None, positions: torch.Tensor | None,
                       new_lengths: torch.Tensor) -> None:
    """The accepted path's rows moved behind the committed ones (``sfl_accept_path``)."""
    batch, heads, capacity, dim = k.shape
    _call(k.device, "sfl_accept_path", k.data_ptr(), v.data_ptr(), _ptr(weights), _ptr(positions),
          lengths.data_ptr(), path.data_ptr(), accepted.data_ptr(), new_lengths.data_ptr(),
          _strides_2(*k.stride()[:3], *v.stride()[:3]), batch, heads, capacity, path.shape[1], dim, _lib.dtype_code(k.dtype))


def launch_select_slots(weights: torch.Tensor, lengths: torch.Tensor, positions: torch.Tensor | None,
                        kept: torch.Tensor, new_lengths: torch.Tensor, recent: int) -> None:
    """The slots that stay, into ``kept`` (``sfl_select_slots``)."""
    batch, heads, capacity = weights.shape
    _call(weights.device, "sfl_select_slots", weights.data_ptr(), lengths.data_ptr(), _ptr(positions),
          kept.data_ptr(), new_lengths.data_ptr(), batch, heads, capacity, kept.shape[2], recent)


def launch_compact_slots(kept: torch.Tensor, k: torch.Tensor, v: torch.Tensor, weights: torch.Tensor | None,
                         positions: torch.Tensor | None) -> None:
    """Kept rows moved into the free places below them (``sfl_compact_slots``)."""
    batch, heads, capacity, dim = k.shape
    _call(k.device, "sfl_compact_slots", k.data_ptr(), v.data_ptr(), _ptr(weights), _ptr(positions), kept.data_ptr(),
          _strides_2(*k.stride()[:3], *v.stride()[:3]), batch, heads, capacity, kept.shape[2], dim, _lib.dtype_code(k.dtype))


def launch_page_append(k: torch.Tensor, v: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                       counts: torch.Tensor | None, refs: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                       k_scale: torch.Tensor, v_scale: torch.Tensor, layer: int) -> None:
    """New tokens quantised into one layer's pages (``sfl_page_append``)."""
    batch, heads, tokens, dim = k.shape
    pages, _, page_size = k_codes.shape[1:4]
    codes, scales = layer * k_codes.stride(0), 4 * layer * k_scale.stride(0)
    _call(k.device, "sfl_page_append", k.data_ptr(), v.data_ptr(), k_codes.data_ptr() + codes,
          v_codes.data_ptr() + codes, k_scale.data_ptr() + scales, v_scale.data_ptr() + scales, tables.data_ptr(),
          lengths.data_ptr(), _ptr(counts), refs.data_ptr(), _strides_2(*k.stride()[:3], *v.stride()[:3]), batch, heads,
          tokens, tables.shape[1], pages, page_size, dim, _lib.dtype_code(k.dtype))


def launch_page_attention(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
                          v_scale: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                          counts: torch.Tensor | None, partial_max: torch.Tensor, partial_sum: torch.Tensor,
                          partial_output: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, layer: int,
                          window_left: int, splits: int, most_splits: int, scale: float) -> None:
    """Attention of new tokens over one layer's pages into ``out`` and ``lse`` (``sfl_page_attention``)."""
    batch, heads, tokens, dim = q.shape
    pages, kv_heads, page_size = k_codes.shape[1:4]
    codes, scales = layer * k_codes.stride(0), 4 * layer * k_scale.stride(0)
    _call(q.device, "sfl_page_attention", q.data_ptr(), k_codes.data_ptr() + codes, v_codes.data_ptr() + codes,
          k_scale.data_ptr() + scales, v_scale.data_ptr() + scales, tables.data_ptr(), lengths.data_ptr(), _ptr(counts),
          partial_max.data_ptr(), partial_sum.data_ptr(), partial_output.data_ptr(), out.data_ptr(), lse.data_ptr(),
          _strides_2(*q.stride()[:3], *out.stride()[:3]), batch, heads, kv_heads, tokens, tables.shape[1], pages,
          page_size, dim, window_left, splits, most_splits, scale, _lib.dtype_code(q.dtype))


def launch_page_fork(parents: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
                     page_size: int) -> None:
    """Every row of the tables becomes its parent's (``sfl_page_fork``)."""
    batch, places = tables.shape
    _call(tables.device, "sfl_page_fork", tables.data_ptr(), lengths.data_ptr(), refs.data_ptr(), parents.data_ptr(),
          batch, places, refs.shape[0], page_size)


def _pools(k_codes, v_codes, k_scale, v_scale):
    return k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()


def launch_page_reserve(lengths: torch.Tensor, counts: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                        k_scale: torch.Tensor, v_scale: torch.Tensor, tables: torch.Tensor, refs: torch.Tensor,
                        granted: torch.Tensor, scratch: torch.Tensor) -> None:
    """Pages for the next tokens, shared ones copied (``sfl_page_reserve``)."""
    batch, places = tables.shape
    layers, pages, heads, page_size, dim = k_codes.shape
    _call(tables.device, "sfl_page_reserve", *_pools(k_codes, v_codes, k_scale, v_scale), tables.data_ptr(),
          lengths.data_ptr(), refs.data_ptr(), counts.data_ptr(), granted.data_ptr(), scratch.data_ptr(), batch, places,
          pages, layers, heads, page_size, dim)


def launch_page_compact(k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                        tables: torch.Tensor, refs: torch.Tensor, used: torch.Tensor, scratch: torch.Tensor) -> None:
    """The pages in use moved to the front of the pool (``sfl_page_compact``)."""
    batch, places = tables.shape
    layers, pages, heads, page_size, dim = k_codes.shape
    _call(tables.device, "sfl_page_compact", *_pools(k_codes, v_codes, k_scale, v_scale), tables.data_ptr(),
          refs.data_ptr(), used.data_ptr(), scratch.data_ptr(), batch, places, pages, layers, heads, page_size, dim)


def _nothing(*args):
    return None


_CACHE_OPS = {
    "rotate": (launch_rotate, ("q_out", "k_out", "v_out")),
    "tree_attention": (launch_tree_attention, ("partial_max", "partial_sum", "partial_output", "out", "lse")),
    "tree_weights": (launch_tree_weights, ("weights",)),
    "accept_path": (launch_accept_path, ("k", "v", "weights", "positions", "new_lengths")),
    "select_slots": (launch_select_slots, ("kept", "new_lengths")),
    "compact_slots": (launch_compact_slots, ("k", "v", "weights", "positions")),
    "page_append": (launch_page_append, ("k_codes", "v_codes", "k_scale", "v_scale")),
    "page_attention": (launch_page_attention, ("partial_max", "partial_sum", "partial_output", "out", "lse")),
    "page_fork": (launch_page_fork, ("tables", "lengths", "refs")),
    "page_reserve": (launch_page_reserve, ("k_codes", "v_codes", "k_scale", "v_scale", "tables", "refs", "granted",
                                           "scratch")),
    "page_compact": (launch_page_compact, ("k_codes", "v_codes", "k_scale", "v_scale", "tables", "refs", "used",
                                           "scratch")),
}
for _name, (_launch, _written) in _CACHE_OPS.items():
    torch.library.custom_op(f"sfl::{_name}", mutates_args=_written)(_launch).register_fake(_nothing)


# The same launches as kernels of the GPU's dispatch key: the wrapper a custom op
# puts around its function for every device is another 3.6 us of a call.
_gpu_kernels = torch.library.Library("sfl", "FRAGMENT")
_gpu_kernels.impl("decode_attention", launch_decode_attention, "CUDA")
_gpu_kernels.impl("masked_attention", launch_masked_attention, "CUDA")
for _name, (_launch, _) in _CACHE_OPS.items():
    _gpu_kernels.impl(_name, _launch, "CUDA")
