"""Rotary frequencies scaled by parts: the band between the two limits (no GPU)."""

import math

import pytest
import torch

from trifusion_b200 import rotary_frequencies


@pytest.mark.parametrize("dim,base,factor,length,turns", [
    (64, 10000.0, 4.0, 2048, (1.0, 32.0)), (128, 500000.0, 8.0, 8192, (1.0, 4.0)), (96, 10000.0, 1.5, 451, (0.0, 7.5))])
def test_parts_blend_linearly_in_turns(dim, base, factor, length, turns):
    """The share that stays as it is goes from 0 at the low limit to 1 at the high one with the turns that a
    frequency makes within the trained length (not with its index)."""
    got, amplitude = rotary_frequencies(dim, base, scaling="parts", factor=factor, trained_length=length, turns=turns,
                                        device="cpu")
    low, high = turns
    band = 0
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        t = length * f / (2.0 * math.pi)
        share = min(max((t - low) / (high - low), 0.0), 1.0)
        band += 0.0 < share < 1.0
        assert got[i].item() == pytest.approx(share * f + (1.0 - share) * f / factor, rel=1e-13)
    assert band >= 3
    assert amplitude == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)


def test_parts_halfway():
    """dim 2, base 1: one frequency, one radian a position. 2 pi 10 positions are ten turns, halfway from 5 to 15."""
    f, _ = rotary_frequencies(2, 1.0, scaling="parts", factor=4.0, trained_length=20.0 * math.pi, turns=(5.0, 15.0),
                              device="cpu")
    assert torch.allclose(f, torch.tensor([0.5 + 0.5 / 4.0], dtype=torch.float64), rtol=1e-14)
