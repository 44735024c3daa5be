"""Rotary positions of query and key heads: any position, half or interleaved
pairs, part of the head, frequencies scaled for long contexts.

``kernels.buffers.RotaryQKV`` rotates the pooled attention's packed projection by
a table that starts at step 0; this operator takes q and k heads as they lie (views
of a projection row included) and a position for every token, so a stream can go on
where it stopped. Angles are formed in 64 bits, the rotation in FP32 with one
rounding to the tensors' type.
"""

from __future__ import annotations

import math

import torch

from . import _lib

_LAYOUTS = ("half", "interleaved")


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, trained_length=None,
                       turns=(1.0, 32.0), device="cuda"):
    """``(inv_freq, amplitude)`` for :func:`apply_rotary`: FP64 ``[rotary_dim / 2]`` inverse
    frequencies ``base^(-2 i / rotary_dim)`` on ``device`` and the factor on the rotated values.

    ``scaling`` stretches them for contexts ``factor`` times the trained one:

    * ``None``: as they are;
    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: the base raised to ``base * factor^(R / (R - 2))``, which keeps the highest
      frequency and divides the lowest by ``factor``;
    * ``"parts"``: frequencies that make fewer than ``turns[0]`` turns within
      ``trained_length`` positions are divided by ``factor``, those with more than
      ``turns[1]`` kept, the ones between blended linearly; amplitude ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim must be even and positive")
    if not base > 0 or not factor > 0:
        raise ValueError("rotary_frequencies: base and factor must be positive")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    amplitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        low, high = turns
        if trained_length is None or not 0 <= low < high:
            raise ValueError("rotary_frequencies: scaling by parts needs trained_length and turns (low, high)")
        keep = ((trained_length * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freq.to(device), amplitude


def apply_rotary(q, k, positions, inv_freq, *, layout="half", amplitude=1.0, inplace=False):
    """Rotate ``q`` ([B, T, H, D]) and ``k`` ([B, T, Hk, D], or None) by ``positions * inv_freq``.

    ``positions`` is int64 [B, T] or [T], any values; ``inv_freq`` FP64 [R/2] with
    ``R <= D``: elements R.. of each head are copied. Pairs are ``(i, i + R/2)`` (``layout
    "half"``) or ``(2 i, 2 i + 1)`` (``"interleaved"``); a pair becomes ``amplitude * (x1 cos -
    x2 sin, x2 cos + x1 sin)``. q and k are FP32 or BF16 with any strides, the last one 1.
    Returns new contiguous tensors, or the arguments themselves when ``inplace``.
    """
    if layout not in _LAYOUTS:
        raise ValueError(f"apply_rotary: layout must be 'half' or 'interleaved', got {layout!r}")
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError("apply_rotary: q must be [B,T,H,D] and k [B,T,Hk,D]")
    if k is not None and k.dtype != q.dtype:
        raise TypeError("apply_rotary: q and k must have one dtype")
    dtype = _lib.dtype_code(q, "apply_rotary")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not 2 <= 2 * inv_freq.shape[0] <= q.shape[3]:
        raise ValueError("apply_rotary: inv_freq must be float64 [R/2] with 2 <= R <= D")
    b, t, h, d = q.shape
    if positions.dtype != torch.int64 or tuple(positions.shape) not in ((b, t), (t,)):
        raise ValueError("apply_rotary: positions must be int64 [B,T] or [T]")
    _lib.no_gradient("apply_rotary", q, k)
    dev = _lib.require_cuda("apply_rotary", q, q if k is None else k, positions, inv_freq)
    if inplace:
        if q.stride(3) != 1 or (k is not None and k.stride(3) != 1):
            raise ValueError("apply_rotary: in place needs a unit stride in the last dimension")
        qo, ko = q, k
    else:
        q = q if q.stride(3) == 1 else q.contiguous()
        qo = torch.empty((b, t, h, d), dtype=q.dtype, device=dev)
        if k is not None:
            k = k if k.stride(3) == 1 else k.contiguous()
            ko = torch.empty(k.shape, dtype=k.dtype, device=dev)
        else:
            ko = None
    inv_freq = inv_freq.contiguous()
    none = (0, 0, 0)
    strides = _lib.int64_array((*q.stride()[:3], *(none if k is None else k.stride()[:3]), *qo.stride()[:3],
                                *(none if k is None else ko.stride()[:3]),
                                *(positions.stride() if positions.dim() == 2 else (0, positions.stride(0)))))
    _lib.launch("tf_rotary_positions_fwd", dev, q.data_ptr(), None if k is None else k.data_ptr(), qo.data_ptr(),
                None if k is None else ko.data_ptr(), dtype, positions.data_ptr(), inv_freq.data_ptr(),
                float(amplitude), 1 if layout == "interleaved" else 0, strides, b, t, h,
                0 if k is None else k.shape[2], d, 2 * inv_freq.shape[0])
    return (qo, ko) if k is not None else qo
