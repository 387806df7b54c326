"""Argument checks that the KV-cache operators (``rotary``, ``tree``, ``evict``) share.

Nothing here reads a tensor's values: lengths, counts and positions live on the
device and are looked at by the kernels, which clamp them or leave rows out.
"""

from __future__ import annotations

import torch

from . import _lib
from .decode import SUPPORTED_DIMS, SUPPORTED_GROUPS

MAX_DRAFTS = 128


def check_rows(operator: str, named: dict[str, torch.Tensor]) -> None:
    """``[B, H, rows, D]`` tensors of one device and dtype that the kernels read 16 bytes at a time."""
    first = next(iter(named.values()))
    device, dtype = first.device, first.dtype
    for name, t in named.items():
        if t.ndim != 4:
            raise ValueError(f"{name} must be [B, H, rows, D]")
        if t.requires_grad:
            raise RuntimeError(f"{operator} is forward-only; requires_grad inputs are unsupported")
        if t.dtype != dtype:
            raise TypeError(f"{operator}: all rows must have the same FP16, BF16 or FP32 dtype")
    if dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"{operator}: all rows must have the same FP16, BF16 or FP32 dtype")
    check_device(device, named)
    step = 16 // first.element_size()
    for name, t in named.items():
        if min(t.shape) < 1:
            raise ValueError(f"{name} must not be empty")
        if t.shape[-1] not in SUPPORTED_DIMS:
            raise ValueError("supported head dimensions are 16/32/64/128")
        sb, sh, sr, sd = t.stride()
        if sd != 1 or t.data_ptr() % 16 or sb % step or sh % step or sr % step:
            raise ValueError(f"{name} must have a contiguous last dimension and 16-byte aligned rows")


def check_device(device: torch.device, named: dict[str, torch.Tensor | None]) -> None:
    if device.type != "cuda" or any(t is not None and t.device != device for t in named.values()):
        raise ValueError("all tensors must be on the same CUDA device")


def check_cache(k: torch.Tensor, v: torch.Tensor) -> None:
    """A cache that is written to: k and v of one shape, no row in two places."""
    if v.shape != k.shape:
        raise ValueError("k and v caches must have the same [B, Hkv, N, D] shape")
    for t in (k, v):
        if any(stride == 0 and size > 1 for stride, size in zip(t.stride(), t.shape)):
            raise ValueError("a cache that is written to must not be expanded")


def check_heads(query_heads: int, kv_heads: int) -> None:
    if query_heads % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if query_heads // kv_heads not in SUPPORTED_GROUPS:
        raise ValueError("supported GQA ratios are 1/2/4/8")


def check_vector(name: str, t: torch.Tensor | None, dtype: torch.dtype, shape: tuple) -> None:
    """A contiguous tensor of this dtype and shape, or None."""
    if t is not None and (t.dtype != dtype or t.shape != shape or not t.is_contiguous()):
        kind = str(dtype).removeprefix("torch.")
        raise ValueError(f"{name} must be a contiguous {kind} tensor of shape {list(shape)}")
