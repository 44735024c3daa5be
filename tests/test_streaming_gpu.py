"""The streaming operators on a B200 against their definitions in 64 bits (GPU only)."""

import pytest
import torch

from streaming_reference import F32, HALF_STEP, check_out, check_state, recurrence, rotate

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from trifusion_b200 import apply_rotary, linear_attention, linear_attention_step, rotary_frequencies  # noqa: E402

DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


# ---- rotary positions -----------------------------------------------------------------------

def check_rotated(got, x, positions, f, layout, amplitude):
    """One rounding to the type of a sum of two products; sine, cosine and the amplitude's
    product are each within two FP32 roundings, the angle within 2^-22 turns of FP32."""
    ref = rotate(x, positions, f, layout, amplitude)
    r = 2 * f.shape[0]
    assert got.dtype == x.dtype and got.shape == x.shape
    assert torch.equal(got[..., r:], x[..., r:])
    if layout == "half":
        mag = (x[..., : r // 2].double().abs() + x[..., r // 2: r].double().abs()).repeat(1, 1, 1, 2)
    else:
        mag = x[..., :r].double().abs().unflatten(-1, (r // 2, 2)).sum(-1).repeat_interleave(2, dim=-1)
    bound = HALF_STEP[x.dtype] * ref[..., :r].abs() + 16 * F32 * amplitude * mag
    err = (got[..., :r].double() - ref[..., :r]).abs()
    assert (err <= bound).all(), (err - bound).max().item()


ROTARY = [  # batch, time, heads, kv heads, head width, rotated width, first position
    (1, 1, 1, 1, 64, 64, 0), (3, 1, 32, 8, 128, 128, 1 << 31), (2, 7, 6, 6, 64, 32, -5), (1, 5, 3, 1, 6, 6, 11),
    (2, 33, 2, 1, 20, 12, 1000003), (1, 450, 12, 4, 96, 96, 7), (5, 3, 1, 2, 256, 128, 3), (1, 2000, 4, 4, 64, 64, 0),
    (1, 3, 2, 2, 10, 2, 5), (4, 600, 2, 1, 8, 4, 0),
]


@pytest.mark.parametrize("shape", ROTARY)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rotary(shape, layout, dtype):
    b, t, h, hk, d, r, first = shape
    g = torch.Generator(DEV).manual_seed(t + d)
    q = torch.randn(b, t, h, d, generator=g, device=DEV).to(dtype)
    k = torch.randn(b, t, hk, d, generator=g, device=DEV).to(dtype)
    pos = first + torch.randint(0, 50, (b, t), generator=g, device=DEV)
    f, a = rotary_frequencies(r, scaling="parts", factor=4.0, trained_length=512)
    qr, kr = apply_rotary(q, k, pos, f, layout=layout, amplitude=a)
    check_rotated(qr, q, pos, f, layout, a)
    check_rotated(kr, k, pos, f, layout, a)
    only = apply_rotary(q, None, pos, f, layout=layout, amplitude=a)
    assert torch.equal(only, qr)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_rotary_views_in_place(layout, offset):
    """q and k as views of one projection row that starts off a 16-byte boundary; [T] positions."""
    b, t, h, hk, d = 2, 37, 3, 1, 64
    width = (h + 2 * hk) * d
    f, a = rotary_frequencies(48)
    buf = torch.randn(b, t, width + 8, device=DEV).to(BF16)
    before = buf.clone()
    row = buf[..., offset: offset + width]
    q, k = row[..., : h * d].unflatten(-1, (h, d)), row[..., h * d: (h + hk) * d].unflatten(-1, (hk, d))
    pos = torch.arange(100, 100 + t, device=DEV)
    qr, kr = apply_rotary(q, k, pos, f, layout=layout)
    assert torch.equal(buf, before) and qr.is_contiguous()
    check_rotated(qr, q.clone(), pos, f, layout, a)
    check_rotated(kr, k.clone(), pos, f, layout, a)
    q2, k2 = apply_rotary(q, k, pos, f, layout=layout, inplace=True)
    assert q2.data_ptr() == q.data_ptr() and torch.equal(q2, qr) and torch.equal(k2, kr)
    assert torch.equal(row[..., (h + hk) * d:], before[..., offset + (h + hk) * d: offset + width])
    assert torch.equal(buf[..., :offset], before[..., :offset])


def test_rotary_transposed_heads_and_empty():
    f, a = rotary_frequencies(64)
    x = torch.randn(2, 3, 40, 64, device=DEV).transpose(1, 2)  # [B,T,H,D] held as [B,H,T,D]
    pos = torch.arange(40, device=DEV)
    check_rotated(apply_rotary(x, None, pos, f), x, pos, f, "half", a)
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64), (2, 3, 0, 64)):
        y = apply_rotary(torch.empty(shape, device=DEV), None, torch.zeros(shape[1], dtype=torch.int64, device=DEV), f)
        assert tuple(y.shape) == shape


# ---- linear attention -------------------------------------------------------------------------

def inputs(b, t, h, hq, n, p, dtype=BF16, seed=0, state=False, slow=0.1):
    g = torch.Generator(DEV).manual_seed(seed + t + n)
    r = lambda *s, d=dtype: torch.randn(*s, generator=g, device=DEV).to(d)  # noqa: E731
    decay = -torch.rand(b, h, t, generator=g, device=DEV) * slow * torch.arange(1, h + 1, device=DEV)[None, :, None]
    args = [r(b, t, hq, n), r(b, t, hq, n), r(b, t, h, p), decay]
    return args, (r(b, h, n, p, d=FP32) if state else None)


def chunked(args):
    """Whether the tensor-core form may run: its two more roundings are then allowed for."""
    return args[0].dtype == BF16 and args[0].shape[-1] <= 128 and args[2].shape[-1] <= 128


def check(args, state=None, lengths=None, **kw):
    given = None if state is None else state.clone()
    out, new = linear_attention(*args, given, lengths=lengths, **kw)
    decay = args[3]
    b, t, h = args[2].shape[:3]
    if decay.dim() == 1:
        decay = decay[None, :, None].expand(b, h, t)
    ref, s, mag, smag = recurrence(*args[:3], decay, state, lengths, kw.get("scale"))
    n = args[0].shape[-1]
    check_out(out, ref, mag, t, n, chunked(args))
    check_state(new, s, smag, t, n)
    if given is not None:
        assert new.data_ptr() == given.data_ptr()
    return out, new


@pytest.mark.parametrize("time", [1, 2, 31, 32, 63, 64, 65, 127, 129, 200, 451])
@pytest.mark.parametrize("n,p", [(128, 64), (64, 128), (128, 128), (64, 64)])
def test_prompt_lengths(time, n, p):
    args, state = inputs(2, time, 4, 2, n, p, state=True)
    check(args, state)


@pytest.mark.parametrize("n,p", [(8, 8), (32, 96), (96, 32), (72, 104), (40, 128), (128, 16), (136, 64), (64, 256),
                                 (256, 256)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_prompt_widths(n, p, dtype):
    args, state = inputs(2, 70, 3, 1, n, p, dtype, state=True)
    check(args, state)
    check(args)


@pytest.mark.parametrize("h,hq", [(1, 1), (6, 1), (6, 2), (6, 6)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_prompt_shared_heads(h, hq, dtype):
    args, _ = inputs(3, 150, h, hq, 64, 64, dtype)
    check(args, scale=0.5)


@pytest.mark.parametrize("b,t,h", [(1, 2000, 1), (2, 3601, 3), (1, 9000, 2), (40, 640, 8), (1, 1024, 4)])
def test_prompt_long(b, t, h):
    """Few long rows (the time axis is shared out) and many rows."""
    args, state = inputs(b, t, h, 1, 128, 64, state=True, slow=0.01)
    check(args, state)


@pytest.mark.parametrize("time,lengths", [(150, [150, 97, 1, 0, 64, 65]), (1300, [1300, 0, 451, 64]),
                                          (9, [9, 0, 1]), (100, [1000, -3])])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_ragged_rows_read_nothing_past_their_length(time, lengths, dtype):
    b = len(lengths)
    args, state = inputs(b, time, 4, 2, 64, 128, dtype, state=True)
    lens = torch.tensor(lengths, device=DEV)
    past = torch.arange(time, device=DEV)[None, :] >= lens[:, None]
    clean = [torch.where(past.view(b, time, 1, 1), 0.0, x) for x in args[:3]]
    clean.append(torch.where(past[:, None], 0.0, args[3]))
    for bad in (float("nan"), float("inf"), -float("inf")):
        dirty = [torch.where(past.view(b, time, 1, 1), bad, x).to(dtype) for x in args[:3]]
        dirty.append(torch.where(past[:, None], bad, args[3]))
        for s in (state, None):
            got = s.clone() if s is not None else None
            out, new = linear_attention(*dirty, got, lengths=lens)
            ref, sref, mag, smag = recurrence(*[x.to(dtype) for x in clean[:3]], clean[3], s, lens)
            check_out(out, ref, mag, time, 64, chunked(args))
            check_state(new, sref, smag, time, 64)
            assert (out[past] == 0).all()


def test_views_of_a_projection_row():
    """q, k, v as views of one row that starts off a 16-byte boundary, decay as a [B,T,H] view."""
    b, t, h, n, p = 2, 130, 4, 64, 64
    for offset in (0, 4, 3):
        buf = torch.randn(b, t, 2 * n + h * p + h + 8, device=DEV).to(BF16)
        row = buf[..., offset:]
        q, k = row[..., :n].unflatten(-1, (1, n)), row[..., n:2 * n].unflatten(-1, (1, n))
        v = row[..., 2 * n:2 * n + h * p].unflatten(-1, (h, p))
        decay = -torch.rand(b, t, h, device=DEV).transpose(1, 2)
        out = torch.full((b, t, h, p + 8), 7.0, device=DEV, dtype=BF16)
        got, _ = linear_attention(q, k, v, decay, out=out[..., :p])
        assert got.data_ptr() == out.data_ptr() and (out[..., p:] == 7).all()
        ref, _, mag, _ = recurrence(q, k, v, decay)
        check_out(got, ref, mag, t, n, True)
    # Heads before time, rows shared by the whole batch, and a constant decay for each head.
    q, k = (torch.randn(1, 1, t, n, device=DEV).to(BF16).transpose(1, 2).expand(b, t, 1, n) for _ in range(2))
    v = torch.randn(b, h, t, p, device=DEV).to(BF16).transpose(1, 2)
    check([q, k, v, -torch.tensor([0.0, 0.01, 0.3, 40.0], device=DEV)])


@pytest.mark.parametrize("time", [40, 200])
def test_decays_of_all_sizes(time):
    """No decay, decays that leave nothing, and resets (-inf) that forget what came before."""
    b, h, n, p = 2, 4, 64, 64
    args, state = inputs(b, time, h, 2, n, p, state=True)
    decay = args[3]
    decay[:, 0] = 0.0
    decay[:, 1] = -30.0
    decay[:, 2, ::7] = -float("inf")
    decay[:, 3, 5:] = -torch.logspace(-6, 3, time - 5, device=DEV)
    check(args, state)
    decay[:, :, -1] = -float("inf")
    decay[:, 1] = -float("inf")
    check(args, state)


@pytest.mark.parametrize("time", [7, 8, 9, 15, 16, 17, 18])
@pytest.mark.parametrize("b", [1, 80])
def test_short_prompts(time, b):
    """Around the length from which pieces run in chunks."""
    args, state = inputs(b, time, 6, 2, 64, 64, state=True)
    check(args, state)


@pytest.mark.parametrize("scale", [1e-12, -0.25, 1e12])
@pytest.mark.parametrize("rate", [-2.4, -3.0])
@pytest.mark.parametrize("n,p", [(64, 64), (128, 128)])
def test_scales_with_strong_decays(scale, rate, n, p):
    """Weights whose factors would leave FP32's range together with the scale."""
    args, state = inputs(1, 130, 2, 1, n, p, state=True)
    args[3][:] = rate
    check(args, state, scale=scale)


@pytest.mark.parametrize("form", ["chunks", "tokens", "steps"])
def test_slow_decays_over_a_long_memory(form):
    """Roundings of the state go both ways: 2^-24 r.m.s. at most for each of the two or three of a token,
    added up like a random walk, and no more than 2^-29 a token that go one way."""
    t, h, n, p = 2000, 2, 64, 64
    args, _ = inputs(1, t, h, 1, n, p, slow=1e-4)
    _, s, _, _ = recurrence(*args)
    if form == "chunks":
        _, new = linear_attention(*args)
    elif form == "tokens":
        _, new = linear_attention(*[x.float() for x in args])
    else:
        new = torch.zeros(1, h, n, p, device=DEV)
        for i in range(t):
            linear_attention_step(args[0][:, i], args[1][:, i], args[2][:, i], args[3][:, :, i], new)
    err = new.double() - s
    bias = abs(((new.double() * s).sum() / (s * s).sum() - 1).item())
    assert err.norm() <= 2.0 ** -24 * (3 * t) ** 0.5 * s.norm()
    assert bias <= t * 2.0 ** -29


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,p", [(64, 64), (128, 128), (128, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_where_non_finite_values_reach(dtype, n, p, bad):
    """A query's reaches its token, a key's its heads from its token on, a value's its column of its
    head (in the chunked form from the start of its chunk of 64 tokens on), a state's its column."""
    b, t, h, hq, at = 2, 200, 4, 2, 100
    args, state = inputs(b, t, h, hq, n, p, dtype, state=True)
    start = 64 if dtype == BF16 else at

    def run(i, *where):
        mine = [x.clone() for x in args] + [state.clone()]
        mine[i][where] = bad
        out, new = linear_attention(*mine)
        return out.isfinite(), new.isfinite()

    out, new = run(0, 0, at, 1)                     # heads 2 and 3 read key head 1
    assert new.all() and not out[0, at, 2:].any()
    out[0, at, 2:] = True
    assert out.all()
    out, new = run(1, 0, at, 1)
    assert not out[0, at:, 2:].any() and not new[0, 2:].any()
    out[0, at:, 2:] = new[0, 2:] = True
    assert out.all() and new.all()
    out, new = run(2, 0, at, 1, 5)
    assert not out[0, at:, 1, 5].any() and not new[0, 1, :, 5].any()
    out[0, start:, 1, 5] = new[0, 1, :, 5] = True
    assert out.all() and new.all()
    out, new = run(4, 0, 3, 7, 5)
    assert not out[0, :, 3, 5].any() and not new[0, 3, 7, 5]
    out[0, :, 3, 5] = new[0, 3, 7, 5] = True
    assert out.all() and new.all()


@pytest.mark.parametrize("time", [5, 300])
def test_pool_with_slots(time):
    b, h, n, p, pool = 6, 4, 64, 64, 9
    args, _ = inputs(b, time, h, 2, n, p)
    big = torch.randn(pool, h + 1, n, p, device=DEV)
    start = big.clone()
    slots = torch.tensor([4, -1, 8, 9, 4, 0], device=DEV)  # padding, past the pool, twice the same
    out, state = linear_attention(*args, big[:, :h], slots=slots)
    good = [0, 2, 5]
    ref, s, mag, smag = recurrence(*[x[good] for x in args], start[slots[good], :h])
    check_out(out[good], ref, mag, time, n, True)
    check_state(big[slots[good], :h], s, smag, time, n)
    assert (out[1] == 0).all() and out[3].isnan().all() and out[4].isnan().all()
    rest = [1, 2, 3, 5, 6, 7]
    assert torch.equal(big[rest], start[rest]) and torch.equal(big[:, h], start[:, h])


@pytest.mark.parametrize("n,p", [(64, 64), (128, 128), (40, 24)])
def test_long_ragged_rows_of_a_pool(n, p):
    """Slots, lengths, a pool with a gap between its heads and an output off a 16-byte boundary,
    on few rows (the time axis is shared out)."""
    b, t, h, pool = 5, 1400, 2, 6
    args, _ = inputs(b, t, h, 1, n, p, slow=0.01)
    big = torch.randn(pool, h + 1, n, p, device=DEV)
    start = big.clone()
    slots = torch.tensor([5, 0, -1, 5, 3], device=DEV)
    lengths = torch.tensor([1400, 0, 900, 300, 577], device=DEV)
    out = torch.full((b, t, h, p + 4), 7.0, device=DEV, dtype=BF16)
    linear_attention(*args, big[:, 1:], slots=slots, lengths=lengths, out=out[..., 4:])
    good = [0, 1, 4]
    ref, s, mag, smag = recurrence(*[x[good] for x in args], start[slots[good], 1:], lengths[good])
    check_out(out[good][..., 4:], ref, mag, t, n, True)
    check_state(big[slots[good], 1:], s, smag, t, n)
    assert (out[..., :4] == 7).all() and (out[2, :, :, 4:] == 0).all()
    assert out[3, :300, :, 4:].isnan().all() and (out[3, 300:, :, 4:] == 0).all()
    rest = [0, 1, 2, 4]
    assert torch.equal(big[rest], start[rest]) and torch.equal(big[:, 0], start[:, 0])


def test_two_streams_at_once():
    """Calls that share nothing but the device, on two streams without an order between them."""
    work = [inputs(1, 4000, 4, 1, 128, 64, seed=s, state=True, slow=0.01) for s in (1, 2)]
    alone = [linear_attention(*args, state.clone()) for args, state in work]
    states = [[state.clone() for _ in range(6)] for _, state in work]
    torch.cuda.synchronize()
    got = [[], []]
    streams = [torch.cuda.Stream() for _ in work]
    for i in range(6):
        for x, stream_ in enumerate(streams):
            with torch.cuda.stream(stream_):
                got[x].append(linear_attention(*work[x][0], states[x][i]))
    torch.cuda.synchronize()
    for x in range(2):
        for out, state in got[x]:
            assert torch.equal(out, alone[x][0]) and torch.equal(state, alone[x][1])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("b,h,hq,n,p", [(1, 1, 1, 64, 64), (5, 12, 1, 128, 64), (3, 4, 4, 40, 24), (2, 2, 1, 256, 136),
                                        (300, 2, 2, 32, 8)])
def test_step(dtype, b, h, hq, n, p):
    args, state = inputs(b, 1, h, hq, n, p, dtype, state=True)
    got = state.clone()
    q, k, v, decay = args[0][:, 0], args[1][:, 0], args[2][:, 0], args[3][:, :, 0]
    out = linear_attention_step(q, k, v, decay, got)
    ref, s, mag, smag = recurrence(*args, state)
    check_out(out, ref[:, 0], mag[:, 0], 1, n, False)
    check_state(got, s, smag, 1, n)
    again = state.clone()
    assert torch.equal(linear_attention_step(q, k, v, decay[0].contiguous().expand(b, h), again),
                       linear_attention_step(q, k, v, decay[0].contiguous(), state.clone()))


def test_step_slots_padding_and_wrong_slots():
    b, h, n, p, pool = 300, 2, 64, 32, 400
    args, _ = inputs(b, 1, h, 1, n, p)
    q, k, v, decay = args[0][:, 0], args[1][:, 0], args[2][:, 0], args[3][:, :, 0]
    start = torch.randn(pool, h, n, p, device=DEV)
    slots = torch.randperm(pool, device=DEV)[:b]
    slots[5], slots[7], slots[9] = -1, 1 << 40, -(1 << 40)
    slots[299] = slots[3]
    big = start.clone()
    out = linear_attention_step(q, k, v, decay, big, slots=slots)
    good = [i for i in range(b) if i not in (5, 7, 9, 299)]
    ref, s, mag, smag = recurrence(*[x[good] for x in args], start[slots[good]])
    check_out(out[good], ref[:, 0], mag[:, 0], 1, n, False)
    check_state(big[slots[good]], s, smag, 1, n)
    assert (out[5] == 0).all() and (out[9] == 0).all() and out[7].isnan().all() and out[299].isnan().all()
    untouched = torch.ones(pool, dtype=torch.bool, device=DEV)
    untouched[slots[good]] = False
    assert torch.equal(big[untouched], start[untouched])


def test_states_past_32_bit_offsets():
    """A pool of more than 2^31 values: its last slot."""
    h, n, p = 32, 128, 128
    pool = (1 << 31) // (h * n * p) + 2
    big = torch.empty(pool, h, n, p, device=DEV)
    args, state = inputs(1, 70, h, 8, n, p, state=True)
    slots = torch.tensor([pool - 1], device=DEV)
    big[-1] = state[0]
    linear_attention(*args, big, slots=slots)
    _, s, _, smag = recurrence(*args, state)
    check_state(big[-1:], s, smag, 70, n)
    one, before = inputs(1, 1, h, 8, n, p, seed=3)[0], big[-1:].clone()
    linear_attention_step(one[0][:, 0], one[1][:, 0], one[2][:, 0], one[3][:, :, 0], big, slots=slots)
    _, s, _, smag = recurrence(*one, before)
    check_state(big[-1:], s, smag, 1, n)


def test_empty_pieces():
    args, state = inputs(2, 0, 4, 2, 64, 64, state=True)
    out, new = linear_attention(*args, state.clone())
    assert tuple(out.shape) == (2, 0, 4, 64) and torch.equal(new, state)
    out, new = linear_attention(*args)
    assert tuple(new.shape) == (2, 4, 64, 64) and (new == 0).all()
    args, _ = inputs(0, 5, 4, 2, 64, 64)
    out, new = linear_attention(*args)
    assert tuple(out.shape) == (0, 5, 4, 64) and tuple(new.shape) == (0, 4, 64, 64)


@pytest.mark.parametrize("time", [3, 700])
def test_results_do_not_depend_on_the_run(time):
    args, state = inputs(2, time, 4, 1, 128, 64, state=True)
    first = linear_attention(*args, state.clone())
    for _ in range(3):
        again = linear_attention(*args, state.clone())
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


# ---- as they are used together -------------------------------------------------------------------

def stream(q, k, v, decay, pos, f, state, slots, pieces):
    """Rotation and recurrence of consecutive pieces: prompts of several tokens, steps of one."""
    outs, at = [], 0
    for piece in pieces:
        cut = slice(at, at + piece)
        qr, kr = apply_rotary(q[:, cut], k[:, cut], pos[:, cut], f)
        if piece == 1:
            outs.append(linear_attention_step(qr[:, 0], kr[:, 0], v[:, at], decay[:, :, at], state, slots=slots)[:, None])
        else:
            outs.append(linear_attention(qr, kr, v[:, cut], decay[:, :, cut], state, slots=slots)[0])
        at += piece
    return torch.cat(outs, 1)


def test_a_stream_in_pieces():
    """A prompt, another piece and single tokens equal the definition on the whole stream."""
    b, h, hq, n, p = 3, 4, 2, 64, 64
    pieces = [130, 1, 1, 65, 1, 7]
    t = sum(pieces)
    (q, k, v, decay), _ = inputs(b, t, h, hq, n, p)
    f, _ = rotary_frequencies(32)
    pos = torch.arange(t, device=DEV) + torch.tensor([[0], [5000], [70000]], device=DEV)
    slots = torch.tensor([2, 0, 4], device=DEV)
    pool = torch.zeros(5, h, n, p, device=DEV)
    out = stream(q, k, v, decay, pos, f, pool, slots, pieces)
    qr, kr = (rotate(x, pos, f, "half", 1.0).to(BF16) for x in (q, k))
    ref, s, mag, smag = recurrence(qr, kr, v, decay)
    # The operands' rounding to BF16 may fall on the other side where the FP64 value is near a tie:
    # a whole step (2^-7) of that element of q or k, so up to that much of each term.
    err = (out.double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + (2 * 2.0 ** -7 + 2.0 ** -8 + 1e-4) * mag).all()
    assert err.norm() / ref.norm() < 4e-3  # three roundings of 2^-9 r.m.s. at most, and the odd tie
    assert ((pool[slots].double() - s).abs() <= (2.0 ** -7 + 1e-4) * smag).all()
    assert (pool[[1, 3]] == 0).all()


def test_graph_replay_and_side_stream():
    """A captured stream of pieces gives what the eager one gives, replayed on new inputs, and beside
    another graph captured from the same calls."""
    b, h, hq, n, p = 2, 4, 1, 128, 64
    pieces = [600, 1, 33]
    t = sum(pieces)
    f, _ = rotary_frequencies(64)
    pos = torch.arange(t, device=DEV).expand(b, t)
    slots = torch.tensor([1, 2], device=DEV)
    (q, k, v, decay), _ = inputs(b, t, h, hq, n, p)
    graphs = []
    for _ in range(2):
        pool = torch.zeros(3, h, n, p, device=DEV)
        mine = [x.clone() for x in (q, k, v, decay)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            stream(*mine, pos, f, pool, slots, pieces)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pool.zero_()
            out = stream(*mine, pos, f, pool, slots, pieces)
        graphs.append((graph, mine, pool, out))
    for seed in (5, 6):
        expected = []
        for i, (graph, mine, pool, out) in enumerate(graphs):
            for x, y in zip(mine, inputs(b, t, h, hq, n, p, seed=seed + 10 * i)[0]):
                x.copy_(y)
            fresh = torch.zeros_like(pool)
            expected.append((stream(*mine, pos, f, fresh, slots, pieces), fresh))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, mine, pool, out), (eo, ep) in zip(graphs, expected):
            assert torch.equal(out, eo) and torch.equal(pool, ep)
