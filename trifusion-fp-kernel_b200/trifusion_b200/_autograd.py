"""What operators without derivatives owe to PyTorch's automatic differentiation."""

from __future__ import annotations

from torch.autograd import forward_ad
from torch.autograd.graph import increment_version


def has_tangent(*tensors):
    """Whether one of the tensors (None among them) carries a tangent of forward-mode differentiation.
    (Also under ``torch.no_grad()``, which leaves that mode on.)"""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside any dual level, as nearly always
        return False
    return any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors)


def written(x):
    """Counts a write to ``x``, as PyTorch's own in-place operations do, so that a backward pass which
    had saved it is refused instead of using the new values. (Tensors of inference mode count none.)"""
    if not x.is_inference():
        increment_version(x)
