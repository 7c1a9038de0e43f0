"""Rotary positions of queries and keys, with an optional RMS norm per head in the same pass.

    y = x * rsqrt(mean(x^2) + eps) * weight        (where a weight is given)
    (a, b) -> (a cos - b sin, b cos + a sin)       for the pairs of the first rotary dims of y

One kernel reads queries and keys once and writes them once; sums and products are in fp32 and a result is rounded once.
``rotary_embedding`` is differentiable in queries, keys and norm weights; ``paged.rotary_append`` is the form for new tokens
of a key / value cache.  (No counterpart in the reference, whose attention takes queries and keys as they are.)
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _cabi, attention

SCALINGS = (None, "linear", "ntk", "by_parts")


def native():
    """The native host path, which these calls go through."""
    if attention._status_word is None:
        if not torch.cuda.is_available():
            raise RuntimeError("flaxattention_b200 needs a CUDA device (B200, sm_100a); there is no CPU path")
        attention._status()
    return _cabi.host()


def rotary_table(length: int, rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: Optional[int] = None, low: float = 1.0, high: float = 32.0, magnitude: float = 1.0,
                 device=None) -> torch.Tensor:
    """cos and sin of the angles ``position * frequency`` for positions ``0 .. length - 1``: float32 ``[length, rotary_dim]``,
    the cosines of the ``rotary_dim / 2`` pairs in front of the sines.  Worked out in 64 bits, so that far positions keep
    their angles.  The frequencies are ``base ** (-2 i / rotary_dim)``; for contexts ``factor`` times as long as a model
    was trained on, ``scaling`` changes them:

    ``"linear"``    all divided by ``factor`` (positions interpolated)
    ``"ntk"``       ``base * factor ** (rotary_dim / (rotary_dim - 2))`` instead of ``base``: the slowest frequency is divided by
                    ``factor``, the fastest stays
    ``"by_parts"``  frequencies that turn at least ``high`` times over ``original_length`` stay, those that turn at most ``low``
                    times are divided by ``factor``, with a linear passage in between

    ``magnitude`` multiplies the table (a factor of ``m`` for queries and keys makes one of ``m * m`` for the scores).
    """
    if length < 0 or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"length must not be negative and rotary_dim must be even, got {length} and {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("scaling 'ntk' needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-pair / max(rotary_dim, 1))
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "by_parts":
        if original_length is None or original_length <= 0 or not low < high:
            raise ValueError("scaling 'by_parts' needs original_length and low < high")
        stay = ((original_length * freq / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * stay + freq / factor * (1.0 - stay)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], 1) * magnitude).float()


def rotary_embedding(query, key, table, positions=None, *, query_weight=None, key_weight=None, eps: float = 1e-6,
                     interleaved: bool = False, bhln: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with their rotary positions, ``(query, key)`` of the same shapes and dtype.

    ``query`` ``[B, Hq, S, D]`` and ``key`` ``[B, Hkv, S, D]`` (``bhln=False``: ``[B, S, H, D]``), float16, bfloat16 or
    float32, with any strides but a contiguous head dimension.  ``table`` is that of ``rotary_table``; its columns, an even number up to
    ``D``, are the part of the head that is rotated, the rest is passed on (``None``: nothing is rotated).  ``positions`` ``[B, S]`` or ``[S]``
    (int32 or int64, ``None``: 0 to S - 1) are its rows; a position beyond it makes the rotated part 0 and the next call raise
    ``FlaxAttnError`` (``check_status``).  ``interleaved``: neighbouring values make a pair, instead of ``i`` and ``i + rotary_dim / 2``.
    ``query_weight`` / ``key_weight`` ``[D]`` (the tensors' dtype or float32): an RMS norm over the head dimension in front.

    Gradients of the weights are sums over all rows in a fixed order.  What would look on (a tracer, a dispatch mode, a functorch transform, a
    tensor class with a ``__torch_function__`` of its own) is refused with ``NotImplementedError``.
    """
    return native().rotary(query, key, table, positions, query_weight, key_weight, eps, interleaved, not bhln)
