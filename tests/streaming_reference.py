"""The streaming operators' definitions in 64 bits, and bounds on what rounding may do.

``recurrence`` also runs the recurrence of absolute values: ``mag`` (outputs) and
``state_mag`` (states) are what every term adds up to without cancellation, so a relative
error of each term by ``e`` is an absolute one of at most ``e * mag``.
"""

import torch

F32 = 2.0 ** -24  # half a step, relative to the value
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: F32}


def recurrence(q, k, v, decay, state=None, lengths=None, scale=None):
    """(out, state, mag, state_mag) of rows [B,T,...] in FP64; ``decay`` [B,H,T]."""
    b, t, h, p = v.shape
    hq, n = q.shape[2:]
    share = h // hq
    s = torch.zeros(b, h, n, p, dtype=torch.float64, device=v.device) if state is None else state.double()
    s = s.clone()
    m = s.abs()
    out = torch.zeros(b, t, h, p, dtype=torch.float64, device=v.device)
    mag = torch.zeros_like(out)
    scale = n ** -0.5 if scale is None else scale
    for i in range(t):
        live = torch.ones(b, dtype=torch.bool, device=v.device) if lengths is None else lengths > i
        qi, ki = (x[:, i].double().repeat_interleave(share, dim=1) for x in (q, k))
        a = decay[:, :, i].double().exp()[..., None, None]
        kv = ki[..., :, None] * v[:, i].double()[..., None, :]
        pick = live[:, None, None, None]
        s = torch.where(pick, torch.where(a == 0, 0.0, s * a) + kv, s)
        m = torch.where(pick, torch.where(a == 0, 0.0, m * a) + kv.abs(), m)
        row = live[:, None, None]
        out[:, i] = torch.where(row, scale * (qi[..., None] * s).sum(-2), 0.0)
        mag[:, i] = torch.where(row, abs(scale) * (qi.abs()[..., None] * m).sum(-2), 0.0)
    return out, s, mag, m


def term_error(t, n):
    """Relative error of a term after FP32 work on t tokens of key width n: one exponential
    (2 units in the last place and the rounding of its argument), one product and one sum a
    token, and a sum over n."""
    return (6 * t + n + 16) * F32


def check_out(got, ref, mag, t, n, chunked):
    """|got - ref| against the rounding of the result and of its terms. ``chunked``: the
    tensor-core form rounds each score and each state element to BF16 once more."""
    step = HALF_STEP[got.dtype]
    bound = step * ref.abs() + (term_error(t, n) + (2.0 ** -8 if chunked else 0.0)) * (1 + step) * mag
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), "non-finite output"
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert worst <= 0, f"{worst:.3e} over the bound; largest error {err.max().item():.3e}"


def check_state(got, ref, mag, t, n):
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), "non-finite state"
    worst = (err - term_error(t, n) * mag).max().item() if err.numel() else 0.0
    assert worst <= 0, f"{worst:.3e} over the bound; largest error {err.max().item():.3e}"


def rotate(x, positions, inv_freq, layout, amplitude):
    """FP64 rotation of x [B,T,H,D] by complex products."""
    r = 2 * inv_freq.shape[0]
    if positions.dim() == 1:
        positions = positions.expand(x.shape[0], -1)
    angle = (positions.double()[..., None] * inv_freq)[:, :, None]
    turn = amplitude * torch.complex(angle.cos(), angle.sin())
    y = x.double().clone()
    head = y[..., :r]
    if layout == "half":
        z = torch.complex(head[..., : r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        y[..., :r] = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(*x.shape[:3], r // 2, 2).contiguous()) * turn
        y[..., :r] = torch.view_as_real(z).flatten(-2)
    return y
