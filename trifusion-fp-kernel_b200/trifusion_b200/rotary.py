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
from ._autograd import has_tangent, written

_DTYPES = {torch.float32: _lib.TF_F32, torch.bfloat16: _lib.TF_BF16}
_LAYOUTS = {"half": 0, "interleaved": 1}
_launch = _lib.launcher("tf_rotary_positions_fwd", "6Q14qd8i")  # tf_rotary_io


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
      ``turns[1]`` kept, the ones between blended linearly in their turns (a model whose blend
      is linear in the index of the frequency has others there); amplitude ``0.1 ln(factor) + 1``.
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

    ``positions`` is int64 [B, T] or [T], any values (angles at 2^31 are within 1e-7 turns, and
    the error grows with the position);
    ``inv_freq`` FP64 [R/2] with ``R <= D``: elements R.. of each head are copied. Pairs are
    ``(i, i + R/2)`` (``layout "half"``) or ``(2 i, 2 i + 1)`` (``"interleaved"``); a pair becomes ``amplitude * (x1 cos -
    x2 sin, x2 cos + x1 sin)``. q and k are FP32 or BF16 with any strides; R is at most 1024 and
    ``(H + Hk) * D`` at most 65535. Returns new contiguous tensors, or the arguments themselves
    when ``inplace`` (last stride 1, q and k apart from each other). There is no backward pass.
    """
    interleaved = _LAYOUTS.get(layout)
    if interleaved is None:
        raise ValueError(f"apply_rotary: layout must be 'half' or 'interleaved', got {layout!r}")
    shape = q.shape
    if len(shape) != 4:
        raise ValueError("apply_rotary: q must be [B,T,H,D] and k [B,T,Hk,D]")
    b, t, h, d = shape
    dtype, index = _DTYPES.get(q.dtype), q.get_device()
    if dtype is None:
        raise TypeError(f"apply_rotary: expected float32 or bfloat16, got {q.dtype}")
    if k is None:
        hk, same, grad = 0, True, q.requires_grad
    else:
        kb, kt, hk, kd = k.shape if k.dim() == 4 else (-1,) * 4
        if kb != b or kt != t or kd != d:
            raise ValueError("apply_rotary: q must be [B,T,H,D] and k [B,T,Hk,D]")
        if k.dtype != q.dtype:
            raise TypeError("apply_rotary: q and k must have one dtype")
        same, grad = k.get_device() == index, q.requires_grad or k.requires_grad
    half = inv_freq.numel()
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not 2 <= 2 * half <= d:
        raise ValueError("apply_rotary: inv_freq must be float64 [R/2] with 2 <= R <= D")
    if positions.dtype != torch.int64 or tuple(positions.shape) not in ((b, t), (t,)):
        raise ValueError("apply_rotary: positions must be int64 [B,T] or [T]")
    if inplace:
        if q.stride(3) != 1 or k is not None and k.stride(3) != 1:
            raise ValueError("apply_rotary: in place needs a unit stride in the last dimension")
        for x in (q, k):
            if x is not None and not x.is_contiguous() and _lib.overlaps_itself(x):
                raise ValueError("apply_rotary: in place needs tensors that do not overlap themselves")
        if k is not None and q.data_ptr() == k.data_ptr() and q.numel() and k.numel():
            raise ValueError("apply_rotary: in place needs q and k apart from each other")
    if (grad or inv_freq.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("apply_rotary: " + _lib.NO_GRADIENT)
    if has_tangent(q, k, inv_freq):
        raise RuntimeError("apply_rotary: " + _lib.NO_TANGENT)
    if index < 0 or not same or positions.get_device() != index or inv_freq.get_device() != index:
        raise RuntimeError("apply_rotary: all tensors must be CUDA tensors on one device")
    if not inv_freq.is_contiguous():
        inv_freq = inv_freq.contiguous()
    q0, q1, q2, q3 = q.stride()
    k0 = k1 = k2 = o0 = o1 = o2 = 0
    k3, kp, kop = 1, 0, 0
    if k is not None:
        k0, k1, k2, k3 = k.stride()
    if inplace:
        qo, ko, p0, p1, p2, o0, o1, o2 = q, k, q0, q1, q2, k0, k1, k2
    else:
        if q3 != 1:
            q = q.contiguous()
            q0, q1, q2, _ = q.stride()
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        p0, p1, p2, ko = t * h * d, h * d, d, None
        if k is not None:
            if k3 != 1:
                k = k.contiguous()
                k0, k1, k2, _ = k.stride()
            ko = torch.empty_like(k, memory_format=torch.contiguous_format)
            o0, o1, o2 = t * hk * d, hk * d, d
    if k is not None:
        kp, kop = k.data_ptr(), ko.data_ptr()
    s = positions.stride()
    _launch(index, q.data_ptr(), kp, qo.data_ptr(), kop, positions.data_ptr(), inv_freq.data_ptr(), q0, q1, q2, k0, k1, k2,
            p0, p1, p2, o0, o1, o2, 0 if len(s) == 1 else s[0], s[-1], amplitude, dtype, interleaved, b, t, h, hk, d,
            2 * half)
    if inplace:
        written(q)
        if k is not None:
            written(k)
    return qo if k is None else (qo, ko)
