"""What the streaming operators write counts as written for autograd (GPU only)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from trifusion_b200 import apply_rotary, linear_attention, linear_attention_step, rotary_frequencies  # noqa: E402

DEV = "cuda"


def written_by(call, x):
    """Whether a product that saved ``x`` refuses its backward pass once ``call`` has run."""
    w = torch.ones_like(x, requires_grad=True)
    y = (x * w).sum()
    call()
    try:
        y.backward()
    except RuntimeError as e:
        assert "inplace" in str(e)
        return True
    return False


@pytest.mark.parametrize("time", [5, 130])
def test_saved_tensors_that_are_written_refuse_their_backward_pass(time):
    r = lambda *s: torch.randn(*s, device=DEV).bfloat16()  # noqa: E731
    b, h, n, p = 2, 2, 64, 64
    q, k, v, decay = r(b, time, 1, n), r(b, time, 1, n), r(b, time, h, p), -torch.rand(b, h, time, device=DEV)
    state, out = torch.zeros(b, h, n, p, device=DEV), r(b, time, h, p)
    one = q[:, 0].clone(), k[:, 0].clone(), v[:, 0].clone(), decay[:, :, 0].contiguous()
    f, _ = rotary_frequencies(n)
    pos = torch.arange(time, device=DEV)
    assert written_by(lambda: linear_attention(q, k, v, decay, state), state)
    assert written_by(lambda: linear_attention(q, k, v, decay, out=out), out)
    assert written_by(lambda: linear_attention_step(*one, state), state)
    assert written_by(lambda: linear_attention_step(*one, state, out=out[:, 0]), out)
    assert written_by(lambda: apply_rotary(q, k, pos, f, inplace=True), q)
    assert written_by(lambda: apply_rotary(q, k, pos, f, inplace=True), k)
    for x in (q, k, v, decay):
        assert not written_by(lambda: linear_attention(q, k, v, decay, state), x)
    assert not written_by(lambda: apply_rotary(q, k, pos, f), q)


def test_tensors_of_inference_mode():
    """They count no writes, inside the mode and behind it."""
    r = lambda *s: torch.randn(*s, device=DEV).bfloat16()  # noqa: E731
    f, _ = rotary_frequencies(64)
    with torch.inference_mode():
        q, k, v, decay = r(2, 70, 1, 64), r(2, 70, 1, 64), r(2, 70, 2, 64), -torch.rand(2, 2, 70, device=DEV)
        state = torch.zeros(2, 2, 64, 64, device=DEV)
        linear_attention(q, k, v, decay, state)
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay[:, :, 0], state)
        apply_rotary(q, k, torch.arange(70, device=DEV), f, inplace=True)
    before = state.clone()
    linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay[:, :, 0], state)
    apply_rotary(q, k, torch.arange(70, device=DEV), f, inplace=True)
    assert not torch.equal(state, before)
