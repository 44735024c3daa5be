"""Waits of the chunked linear attention that run out reach the caller as exceptions (GPU only).

With a limit of less than one try of 4 us, loads do not wait for room, so that all that wait for
their tiles give up. The launch must end by itself, the next call must raise, and the one after it
must give what it gave before. Nothing is faulted and the context stays usable.
"""

import pytest
import torch

from trifusion_b200 import _lib

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from trifusion_b200 import linear_attention  # noqa: E402

DEV = "cuda"
SHAPES = [  # rows, tokens, heads, key heads, N, P
    (1, 17, 1, 1, 64, 64),       # one partial chunk
    (2, 1200, 3, 1, 128, 64),    # segments, a pair and a single head
    (1, 2000, 2, 2, 128, 128),   # segments of one wide head
    (80, 300, 2, 1, 64, 128),    # many rows
]


@pytest.mark.parametrize("limit", [1, 3999, 1000000])
@pytest.mark.parametrize("shape", SHAPES)
def test_waits_that_run_out_raise_on_the_next_call(shape, limit):
    b, t, h, hq, n, p = shape
    g = torch.Generator(DEV).manual_seed(t)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    args = r(b, t, hq, n), r(b, t, hq, n), r(b, t, h, p), -torch.rand(b, h, t, generator=g, device=DEV)
    state = torch.randn(b, h, n, p, generator=g, device=DEV)
    ref = linear_attention(*args, state.clone())
    torch.cuda.synchronize()
    assert _lib.lib().tf_device_error(1) == 0
    _lib.set_flag_wait_ns(limit)
    try:
        linear_attention(*args, state.clone())
        torch.cuda.synchronize()
    finally:
        _lib.set_flag_wait_ns(0)
    gave_up = _lib.lib().tf_device_error_pending() != 0
    assert gave_up == (_lib.lib().tf_device_error(0) != 0)
    assert gave_up == (limit < 4000 and t > 17)  # (one chunk waits for no room)
    if gave_up:
        with pytest.raises(RuntimeError, match="linear attention kernel gave up one of its bounded waits"):
            linear_attention(*args, state.clone())
    assert _lib.lib().tf_device_error(0) == 0 and _lib.lib().tf_device_error_pending() == 0
    again = linear_attention(*args, state.clone())
    torch.cuda.synchronize()
    assert torch.equal(again[0], ref[0]) and torch.equal(again[1], ref[1])
    assert _lib.lib().tf_device_error_pending() == 0
