"""Rotary positions of queries and keys, with a norm for each head and the cache append.

``rotate`` turns q and k; ``rotate_append`` also writes k and v of new tokens into a
KV cache. Both can normalise each head first (RMSNorm over the head dimension, a gain
for all heads of q and one for all of k) and do everything in one pass over the rows,
in fp32, rounded once. The model's own layers have this fused into their projections
(``sfl_rmsnorm_qkv_rope_append``, ``sfl_gemm_qkv_rope``) for interleaved pairs over the
whole head; these operators take other layouts, parts of a head and grouped heads.

The angles come from host-built tables (``rotary_tables``): they are formed in float64,
so far positions keep their angle to fp32's last bits, and the kernels evaluate no sine.
Inference only, as the framework's attention: ``requires_grad`` inputs are refused.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from . import cache
from . import ops  # registers torch.ops.sfl

LAYOUTS = ("interleaved", "half")
SCALINGS = ("linear", "base", "ramp")


def rotary_tables(rotary_dim, positions, theta=10000.0, *, scaling=None, factor=1.0, original_positions=None,
                  low=1.0, high=32.0, magnitude=1.0, device=None):
    """fp32 ``(cos, sin)`` of ``[positions, rotary_dim / 2]`` for frequencies ``theta^(-2i / rotary_dim)``.

    ``scaling`` fits a context ``factor`` times as long as the one trained on:

    * ``"linear"``: every angle divided by ``factor``;
    * ``"base"``: theta raised to ``theta * factor^(rotary_dim / (rotary_dim - 2))``, which
      divides the lowest frequency by ``factor`` and leaves the highest;
    * ``"ramp"``: frequencies that turn at most ``low`` times within ``original_positions``
      are divided by ``factor``, those that turn at least ``high`` times stay, and the
      ones between are blended linearly in the number of turns.

    ``magnitude`` multiplies both tables (a scale of the scores of ``magnitude`` squared).
    """
    for name, value in (("rotary_dim", rotary_dim), ("positions", positions)):
        if type(value) is not int or value < 1:
            raise ValueError(f"{name} must be a positive integer")
    if rotary_dim % 2:
        raise ValueError("rotary_dim must be even because pairs of dimensions are rotated")
    for name, value in (("theta", theta), ("factor", factor), ("magnitude", magnitude)):
        if not math.isfinite(value) or value <= 0:
            raise ValueError(f"{name} must be finite and positive")
    if scaling is not None and scaling not in SCALINGS:
        raise ValueError("scaling must be None, 'linear', 'base' or 'ramp'")
    exponents = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("'base' scaling needs a rotary_dim above 2")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inverse = theta ** -exponents
    if scaling == "linear":
        inverse = inverse / factor
    elif scaling == "ramp":
        if type(original_positions) is not int or original_positions < 1:
            raise ValueError("'ramp' scaling needs original_positions, a positive integer")
        if not 0 <= low < high:
            raise ValueError("'ramp' scaling needs 0 <= low < high")
        turns = original_positions * inverse / (2 * math.pi)
        stay = ((turns - low) / (high - low)).clamp(0, 1)
        inverse = inverse * stay + inverse / factor * (1 - stay)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * inverse
    cos, sin = (magnitude * angles.cos()).float(), (magnitude * angles.sin()).float()
    return cos.to(device), sin.to(device)


def _check(operator, names, rows, positions, cos, sin, counts, layout, q_norm, k_norm, eps):
    """What both calls ask of their arguments; rows are q, k and what else has the same dtype. Returns the device index."""
    if layout not in LAYOUTS:
        raise ValueError("layout must be 'interleaved' or 'half'")
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be finite and not negative")
    index = cache.check_rows(operator, names, rows, aligned=False)
    q = rows[0]
    batch, _, tokens, dim = q.shape
    kb, _, kt, kd = rows[1].shape
    if kb != batch or kt != tokens or kd != dim:
        raise ValueError("q and k must agree in batch, tokens and head dimension")
    table = cos.shape
    if len(table) != 2 or not 1 <= table[1] <= dim // 2 or table[0] < 1:
        raise ValueError("cos and sin must be [positions, rotary_dim / 2] with rotary_dim at most the head dimension")
    cache.check_vector(operator, "cos", cos, torch.float32, table, index)
    cache.check_vector(operator, "sin", sin, torch.float32, table, index)
    cache.check_vector(operator, "positions", positions, torch.int32, (batch, tokens), index)
    if counts is not None:
        cache.check_vector(operator, "counts", counts, torch.int32, (batch,), index)
    for gain in (q_norm, k_norm):
        if gain is None:
            continue
        if gain.dtype not in (q.dtype, torch.float32):
            raise ValueError("q_norm and k_norm must be contiguous [D] gains in the dtype of q or float32")
        cache.check_vector(operator, "gains (q_norm and k_norm)", gain, gain.dtype, (dim,), index)
    if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
        raise ValueError("q_norm and k_norm must have the same dtype")
    return index


def rotate(q, k, positions, cos, sin, *, counts=None, layout="interleaved", q_norm=None, k_norm=None, eps=1e-5):
    """q ``[B, Hq, T, D]`` and k ``[B, Hkv, T, D]`` (strided views) normed and rotated, as new tensors.

    ``positions`` int32 ``[B, T]`` index the tables; one outside them gives NaN. The first
    ``2 * cos.shape[1]`` dimensions turn, in pairs ``(2i, 2i + 1)`` (``"interleaved"``) or
    ``(i, i + rotary_dim / 2)`` (``"half"``); the others keep their (normed) values.
    ``counts`` int32 ``[B]``: tokens in use; the rows of the others are zeros.
    """
    cache.check_device(_check("rotate", ("q", "k"), (q, k), positions, cos, sin, counts, layout, q_norm, k_norm, eps))
    _lib.lib()  # fail here, before allocating, if the library is not built
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    _launch((q, k, None, positions, cos, sin, q_norm, k_norm, None, counts, q_out, k_out, None), layout, eps)
    return q_out, k_out


def rotate_append(q, k, v, positions, cos, sin, k_cache, v_cache, lengths, *, counts=None, layout="interleaved",
                  q_norm=None, k_norm=None, eps=1e-5):
    """``rotate`` with k and v written into a cache: returns the turned q.

    Token t of sequence b goes to slot ``lengths[b] + t`` of ``k_cache`` and ``v_cache``
    (``[B, Hkv, N, D]`` views; slots they do not have are left out), v unchanged.
    ``positions`` are independent of the slots: drafts of a tree share positions, and
    after an eviction a slot is not a position. Tokens from ``counts[b]`` on are padding:
    zero rows of q, and the cache stays as it was. ``lengths`` is not changed. The caches
    are two tensors and share no memory with q, k and v.
    """
    index = _check("rotate_append", ("q", "k", "v", "k_cache", "v_cache"), (q, k, v, k_cache, v_cache), positions, cos,
                   sin, counts, layout, q_norm, k_norm, eps)
    batch, heads, _, dim = shape = k.shape
    cb, ch, _, cd = k_cache.shape
    if v.shape != shape or cb != batch or ch != heads or cd != dim:
        raise ValueError("k, v and the caches must agree in batch, heads and head dimension")
    cache.check_cache(k_cache, v_cache)
    cache.check_vector("rotate_append", "lengths", lengths, torch.int32, (batch,), index)
    cache.check_device(index)
    _lib.lib()
    q_out = torch.empty_like(q)
    _launch((q, k, v, positions, cos, sin, q_norm, k_norm, lengths, counts, q_out, k_cache, v_cache), layout, eps)
    return q_out


def _launch(tensors, layout, eps):
    ops.dispatch(torch.ops.sfl.rotate, tensors, tensors[-3:], layout == "half", float(eps), checked=True)
