"""Argument checks that the KV-cache operators (``rotary``, ``tree``, ``evict``) share.

Nothing here reads a tensor's values: lengths, counts and positions live on the
device and are looked at by the kernels, which clamp them or leave rows out. The
calls are short (a few us of kernel for a small batch), so each tensor is looked at
once: one condition for all that has to hold, and its parts only where it does not.
"""

from __future__ import annotations

import torch

from . import _lib
from .decode import SUPPORTED_DIMS, SUPPORTED_GROUPS

MAX_DRAFTS = 128
MAX_ROWS = 1 << 30  # of a tensor's [B, H, rows, D]: the kernels count slots in 32 bits, a step or two past the last
_STEPS = {dtype: 16 // dtype.itemsize for dtype in _lib.DTYPE_CODES}  # elements of 16 bytes


def check_rows(operator: str, names: tuple, tensors: tuple, aligned: bool = True) -> int:
    """``[B, H, rows, D]`` tensors of one device and dtype; returns the device's index (-1: CPU).

    ``aligned``: the kernels read their rows 16 bytes at a time.
    """
    dtype, index = tensors[0].dtype, tensors[0].get_device()
    step = _STEPS.get(dtype)
    for name, t in zip(names, tensors):
        if t.requires_grad:
            _refuse_grad(operator)
        if t.ndim != 4:
            raise ValueError(f"{name} must be [B, H, rows, D]")
        if step is None or t.dtype is not dtype:
            raise TypeError(f"{operator}: all rows must have the same FP16, BF16 or FP32 dtype")
        shape = t.shape
        if 0 in shape:
            raise ValueError(f"{name} must not be empty")
        if shape[3] not in SUPPORTED_DIMS:
            raise ValueError("supported head dimensions are 16/32/64/128")
        if shape[2] > MAX_ROWS:
            raise ValueError(f"{name} must have at most {MAX_ROWS} rows")
        sb, sh, sr, sd = t.stride()
        if sd != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
        if aligned and (sb % step or sh % step or sr % step or t.data_ptr() % 16):
            raise ValueError(f"{name} must have 16-byte aligned rows")
        if t.get_device() != index:
            _refuse_device()
    return index


def check_vector(operator: str, name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, index: int) -> None:
    """A contiguous tensor of this dtype and shape on the device of this index."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        kind = str(dtype).removeprefix("torch.")
        raise ValueError(f"{name} must be a contiguous {kind} tensor of shape {list(shape)}")
    if t.get_device() != index:
        _refuse_device()
    if t.requires_grad:
        _refuse_grad(operator)


def check_device(index: int) -> None:
    """After all other checks: tensors on the CPU are refused."""
    if index < 0:
        _refuse_device()


def _refuse_device():
    raise ValueError("all tensors must be on the same CUDA device")


def _refuse_grad(operator):
    raise RuntimeError(f"{operator} is forward-only; requires_grad inputs are unsupported")


def check_cache(k: torch.Tensor, v: torch.Tensor) -> None:
    """A cache that is written to: k and v of one shape, no row in two places."""
    shape = k.shape
    if v.shape != shape:
        raise ValueError("k and v caches must have the same [B, Hkv, N, D] shape")
    if 0 in k.stride() or 0 in v.stride():
        for t in (k, v):
            if any(stride == 0 and size > 1 for stride, size in zip(t.stride(), shape)):
                raise ValueError("a cache that is written to must not be expanded")


def check_heads(query_heads: int, kv_heads: int) -> None:
    if query_heads % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if query_heads // kv_heads not in SUPPORTED_GROUPS:
        raise ValueError("supported GQA ratios are 1/2/4/8")
