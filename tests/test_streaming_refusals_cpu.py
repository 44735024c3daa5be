"""Arguments of the streaming operators that are refused before anything is launched (no GPU)."""

import itertools

import pytest
import torch

from trifusion_b200 import _lib, apply_rotary, linear_attention, linear_attention_step, rotary_frequencies


def prompt(b=2, t=5, h=4, hq=2, n=64, p=64):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    return [z(b, t, hq, n), z(b, t, hq, n), z(b, t, h, p), torch.zeros(b, h, t)]


def step(b=2, h=4, hq=2, n=64, p=64):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    return [z(b, hq, n), z(b, hq, n), z(b, h, p), torch.zeros(b, h)]


SIZE = 64 * 64


@pytest.mark.parametrize("strides", [(SIZE, SIZE), (2 * SIZE, SIZE), (SIZE, 2 * SIZE), (3 * SIZE, 2 * SIZE + 4),
                                     (5 * SIZE, 2 * SIZE + 4)])
def test_pools_whose_entries_meet_are_refused(strides):
    """Head 0 of one entry in head 1 (2, 3) of another, wholly or in part."""
    state = torch.zeros(40 * SIZE).as_strided((3, 4, 64, 64), (*strides, 64, 1))
    with pytest.raises(ValueError, match="linear_attention: .*overlap"):
        linear_attention(*prompt(b=3), state)
    with pytest.raises(ValueError, match="linear_attention_step: .*overlap"):
        linear_attention_step(*step(b=3), state)


def test_which_pools_meet():
    """The rule against every pair of entries, and pools that only look as if they met."""
    from trifusion_b200.linear_recurrence import _meet

    for s0, n0, s1, n1 in itertools.product(range(4, 30), (2, 3, 5), range(4, 30), (2, 4)):
        at = sorted(i * s0 + j * s1 for i in range(n0) for j in range(n1))
        assert _meet(s0, n0, s1, n1, 4) == any(b - a < 4 for a, b in zip(at, at[1:])), (s0, n0, s1, n1)
    for strides in ((4 * SIZE, SIZE), (SIZE, 3 * SIZE), (3 * SIZE, 5 * SIZE)):  # (nested, transposed, interleaved)
        state = torch.zeros(40 * SIZE).as_strided((3, 4 if strides[0] != 3 * SIZE else 2, 64, 64), (*strides, 64, 1))
        h = state.shape[1]
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            linear_attention(*prompt(b=3, h=h), state)


def test_written_tensors_that_overlap_in_part_are_refused():
    """Windows that slide by less than they hold: two tokens, or two heads, share elements."""
    f, _ = rotary_frequencies(32, device="cpu")
    row = torch.zeros(4096, dtype=torch.bfloat16)
    for strides in ((1280, 256, 32, 1), (1280, 192, 64, 1), (640, 256, 64, 1), (1280, 2, 512, 1)):
        x = row.as_strided((2, 5, 4, 64), strides)
        with pytest.raises(ValueError, match="linear_attention: .*overlap"):
            linear_attention(*prompt(), out=x)
        with pytest.raises(ValueError, match="apply_rotary: .*overlap"):
            apply_rotary(x, None, torch.arange(5), f, inplace=True)
        with pytest.raises(ValueError, match="apply_rotary: .*overlap"):
            apply_rotary(torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16), x, torch.arange(5), f, inplace=True)
    # Slices, transposed views and rows with a gap between them are apart.
    wide = torch.zeros(2, 4, 7, 80, dtype=torch.bfloat16)
    for x in (wide[:, :, 1:6, 8:72].transpose(1, 2), wide.transpose(1, 2)[:, :5, :, :64], wide[:, :1, :5, :64].transpose(1, 2)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            linear_attention(*prompt(h=x.shape[2], hq=1), out=x)
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            apply_rotary(x, None, torch.arange(5), f, inplace=True)


def test_rotating_one_tensor_twice_in_place_is_refused():
    f, _ = rotary_frequencies(32, device="cpu")
    x = torch.zeros(2, 5, 4, 64)
    for q, k in ((x, x), (x, x[:, :, :1]), (x[:, :, :2], x)):
        with pytest.raises(ValueError, match="apart"):
            apply_rotary(q, k, torch.arange(5), f, inplace=True)
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            apply_rotary(q, k, torch.arange(5), f)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        apply_rotary(x[:, :, :2], x[:, :, 2:], torch.arange(5), f, inplace=True)


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    """A dual tensor's tangent would be dropped; torch.no_grad() does not turn forward mode off."""
    import torch.autograd.forward_ad as fw

    f, _ = rotary_frequencies(32, device="cpu")
    x = torch.zeros(1, 5, 2, 64)
    state = torch.zeros(2, 4, 64, 64)
    with torch.set_grad_enabled(grad), fw.dual_level():
        dual = lambda y: fw.make_dual(y, torch.ones_like(y))  # noqa: E731
        for i in range(4):
            for make, call in ((prompt, linear_attention), (step, linear_attention_step)):
                args = make()
                args[i] = dual(args[i])
                with pytest.raises(RuntimeError, match=f"{call.__name__}: .*forward mode"):
                    call(*args, state)
        with pytest.raises(RuntimeError, match="linear_attention_step: .*forward mode"):
            linear_attention_step(*step(), dual(state))
        with pytest.raises(RuntimeError, match="linear_attention: .*forward mode"):
            linear_attention(*prompt(), out=dual(prompt()[2]))
        for args in ((dual(x), x, torch.arange(5), f), (x, dual(x), torch.arange(5), f), (x, None, torch.arange(5), dual(f))):
            with pytest.raises(RuntimeError, match="apply_rotary: .*forward mode"):
                apply_rotary(*args)
        with pytest.raises(RuntimeError, match="CUDA tensors"):  # other tensors' tangents do not matter
            linear_attention(*prompt())


def test_a_gradient_of_the_frequencies_is_refused():
    f, _ = rotary_frequencies(32, device="cpu")
    f.requires_grad_()
    x = torch.zeros(1, 5, 2, 64)
    with pytest.raises(RuntimeError, match="apply_rotary: .*backward"):
        apply_rotary(x, x, torch.arange(5), f)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors"):
        apply_rotary(x, x, torch.arange(5), f)


@pytest.mark.parametrize("error,text", [(1, "a recurrence kernel"), (2, "a recurrence kernel"), (3, "a linear attention kernel")])
def test_the_error_names_the_operator_that_gave_up(monkeypatch, error, text):
    class Fake:
        cleared = 0

        def tf_device_error_pending(self):
            return 0 if self.cleared else error

        def tf_device_error(self, reset):
            self.cleared += reset
            return error

    fake = Fake()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setitem(_lib._watch, "ready", True)
    with pytest.raises(RuntimeError, match=f"{text} gave up one of its bounded waits"):
        _lib.check_device_error()
    _lib.check_device_error()  # once
