"""The linear attention held to the bounds of the form that a call runs in (GPU only)."""

import pytest
import torch

from streaming_reference import check_out, check_state, recurrence

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from trifusion_b200 import _lib, linear_attention  # noqa: E402

DEV = "cuda"


def inputs(b, t, h, hq, n, p, slow=0.1):
    g = torch.Generator(DEV).manual_seed(7 * t + n + p)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    decay = -torch.rand(b, h, t, generator=g, device=DEV) * slow
    return [r(b, t, hq, n).bfloat16(), r(b, t, hq, n).bfloat16(), r(b, t, h, p).bfloat16(), decay], r(b, h, n, p)


def in_chunks(b, t, h, hq, n, p):
    return bool(_lib.lib().tf_linear_attention_chunked(b, t, h, hq, n, p, _lib.TF_BF16))


@pytest.mark.parametrize("time", [1, 2, 7, 8, 9, 15, 16])
@pytest.mark.parametrize("b,h,hq,n,p", [(1, 4, 2, 64, 64), (80, 6, 2, 64, 64), (3, 4, 2, 64, 128), (2, 3, 1, 128, 96)])
def test_short_pieces_have_no_rounding_but_the_outputs(time, b, h, hq, n, p):
    assert not in_chunks(b, time, h, hq, n, p)
    args, state = inputs(b, time, h, hq, n, p)
    lengths = torch.arange(b, device=DEV) % (time + 1) if b == 3 else None
    new = state.clone()
    out, _ = linear_attention(*args, new, lengths=lengths)
    ref, s, mag, smag = recurrence(*args, state, lengths)
    check_out(out, ref, mag, time, n, False)
    check_state(new, s, smag, time, n)


@pytest.mark.parametrize("time,b", [(17, 2), (64, 2), (65, 80), (200, 2), (451, 3), (2000, 1)])
@pytest.mark.parametrize("n,p", [(64, 64), (128, 64), (64, 128), (128, 128), (40, 24)])
def test_outputs_of_chunks_as_a_whole(time, b, n, p):
    """Each output is rounded once, each of its terms (a weight, or an element of the state) once before,
    by at most 2^-8 of the value, 2^-8 / sqrt(3) r.m.s.; terms of independent signs add up as their squares,
    and so do their errors: sqrt(2 / 3) 2^-8 of the outputs' norm. Held to 2^-8 for what is correlated."""
    assert in_chunks(b, time, 4, 2, n, p)
    args, state = inputs(b, time, 4, 2, n, p)
    new = state.clone()
    out, _ = linear_attention(*args, new)
    ref, s, _, smag = recurrence(*args, state)
    err = (out.double() - ref).norm(dim=(1, 3)) / ref.norm(dim=(1, 3))  # of each row and head
    assert (err <= 2.0 ** -8).all(), err.max().item()
    check_state(new, s, smag, time, n)
