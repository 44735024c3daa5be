"""Infinite and undefined values in the states of the linear attention (GPU only)."""

import pytest
import torch

from streaming_reference import check_out, check_state, recurrence

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from trifusion_b200 import linear_attention, linear_attention_step  # noqa: E402

DEV = "cuda"
CHUNKED = ("chunks", "pair", "segments")
INF, NAN = float("inf"), float("nan")
FORMS = ["step", "tokens", "wide", "chunks", "pair", "segments"]


def operands(form, seed=0):
    """(q, k, v, decay, state, lengths) that a form of the operator takes; two rows, four heads."""
    t, n, p, dtype, lengths = {
        "step": (1, 64, 64, torch.bfloat16, None),
        "tokens": (21, 64, 64, torch.float32, [13, 21]),
        "wide": (11, 136, 64, torch.bfloat16, [11, 6]),
        "chunks": (200, 64, 128, torch.bfloat16, [200, 70]),
        "pair": (200, 128, 64, torch.bfloat16, [200, 70]),
        "segments": (1400, 64, 64, torch.bfloat16, [1400, 900]),
    }[form]
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    b, h, hq = 2, 4, 2
    q, k, v = r(b, t, hq, n).to(dtype), r(b, t, hq, n).to(dtype), r(b, t, h, p).to(dtype)
    decay = -torch.rand(b, h, t, generator=g, device=DEV) * 0.05
    lens = None if lengths is None else torch.tensor(lengths, device=DEV)
    return q, k, v, decay, r(b, h, n, p), lens


def run(form, q, k, v, decay, state, lengths):
    new = state.clone()
    if form == "step":
        out = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay[:, :, 0], new)[:, None]
    else:
        out, _ = linear_attention(q, k, v, decay, new, lengths=lengths)
    return out, new


def check_finite_part(got, ref, mag, t, n):
    good = ref.isfinite() & mag.isfinite()
    assert torch.equal(got.isfinite(), good)
    zero = torch.zeros((), device=DEV)
    check_state(torch.where(good, got, zero), torch.where(good, ref, zero.double()), torch.where(good, mag, zero.double()), t, n)


@pytest.mark.parametrize("form", FORMS)
def test_infinite_states_stay_infinite(form):
    """Under no decay, slow and fast ones and ones whose factor is zero in FP32, and behind a length."""
    q, k, v, decay, state, lengths = operands(form)
    decay[:, 0] = 0.0
    decay[:, 1] = -1e-4
    decay[:, 2] = -0.9
    decay[:, 3] = -200.0
    state[:, :, 3, 5] = INF
    state[:, :, 7, 6] = -INF
    out, new = run(form, q, k, v, decay, state, lengths)
    t, n = q.shape[1], q.shape[3]
    ref, s, _, smag = recurrence(q, k, v, decay, state, lengths)
    assert (new[:, :, 3, 5] == INF).all() and (new[:, :, 7, 6] == -INF).all()
    check_finite_part(new, s, smag, t, n)
    live = torch.ones(2, t, dtype=torch.bool, device=DEV) if lengths is None else (
        torch.arange(t, device=DEV)[None] < lengths[:, None])
    assert torch.equal(out.isfinite(), ref.isfinite()) and not out[live][..., 5:7].isfinite().any()
    # Before the factor of the output leaves FP32's range, their sign is the query's too.
    share = out.shape[2] // q.shape[2]
    sign = q[:, :, :, 3].sign().repeat_interleave(share, dim=2)[live][:, :2]
    assert (out[live][:, :2, 5].float() == sign * INF).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_resets_forget_states_that_are_not_finite(form, bad):
    """A decay of -inf on the first token, inside, on the last, on none and behind a length."""
    q, k, v, decay, state, lengths = operands(form, 1)
    t, n = q.shape[1], q.shape[3]
    first = t if lengths is None else int(lengths.min())
    decay[:, 0, 0] = decay[:, 1, first // 2] = decay[:, 2, t - 1] = -INF
    state[0] = bad
    state[1, :, 3, 5] = bad
    out, new = run(form, q, k, v, decay, state, lengths)
    ref, s, mag, smag = recurrence(q, k, v, decay, state, lengths)
    check_finite_part(new, s, smag, t, n)
    good = ref.isfinite() & mag.isfinite()
    assert torch.equal(out.isfinite(), good) and good[:, :, 0].all() and good[0, first // 2:, 1].all()
    keep = lambda x: torch.where(good, x, torch.zeros_like(x))  # noqa: E731
    check_out(keep(out), keep(ref), keep(mag), t, n, form in CHUNKED)
