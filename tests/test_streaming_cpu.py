"""Host side of the streaming operators: refusals, frequencies and the C ABI's checks (no GPU)."""

import math
import struct

import pytest
import torch

from trifusion_b200 import _lib, apply_rotary, linear_attention, linear_attention_step, rotary_frequencies


def prompt(b=2, t=5, h=4, hq=2, n=64, p=64, dtype=torch.bfloat16):
    z = lambda *s, d=dtype: torch.zeros(*s, dtype=d)  # noqa: E731
    return [z(b, t, hq, n), z(b, t, hq, n), z(b, t, h, p), z(b, h, t, d=torch.float32)]


def step(b=2, h=4, hq=2, n=64, p=64, dtype=torch.bfloat16):
    z = lambda *s, d=dtype: torch.zeros(*s, dtype=d)  # noqa: E731
    return [z(b, hq, n), z(b, hq, n), z(b, h, p), z(b, h, d=torch.float32)]


STATE = torch.zeros(2, 4, 64, 64)


@pytest.mark.parametrize("change,error", [
    (lambda a: a.__setitem__(0, a[0][:, :, :1]), ValueError),            # q and k disagree
    (lambda a: a.__setitem__(2, a[2][:, :4]), ValueError),               # v has another length
    (lambda a: a.__setitem__(2, a[2][:, :, :3]), ValueError),            # H % Hq
    (lambda a: a.__setitem__(2, a[2][..., :60]), ValueError),            # P not a multiple of 8
    (lambda a: a.__setitem__(2, a[2].float()), TypeError),               # mixed types
    (lambda a: [a.__setitem__(i, a[i].half()) for i in range(3)], TypeError),
    (lambda a: a.__setitem__(3, a[3].bfloat16()), TypeError),            # decay type
    (lambda a: a.__setitem__(3, a[3].transpose(1, 2)), ValueError),      # decay layout
    (lambda a: a.__setitem__(0, a[0].float().requires_grad_()), TypeError),
    (lambda a: a.__setitem__(2, a[2].requires_grad_()), RuntimeError),   # no backward pass
])
def test_prompt_operands_refused(change, error):
    args = prompt()
    change(args)
    with pytest.raises(error, match="linear_attention"):
        linear_attention(*args)


@pytest.mark.parametrize("kw", [
    dict(state=torch.zeros(2, 4, 64, 64, dtype=torch.float64)),
    dict(state=torch.zeros(2, 4, 64, 32)),
    dict(state=torch.zeros(3, 4, 64, 64)),                               # no slots: one entry for each row
    dict(state=torch.zeros(2, 4, 64, 128)[..., :64]),                    # rows not contiguous
    dict(state=torch.zeros(1, 4, 64, 64).expand(2, 4, 64, 64)),          # overlapping states
    dict(state=torch.zeros(2 * 4 * 64 * 64 + 1)[1:].view(2, 4, 64, 64)),  # not on a 16-byte boundary
    dict(state=STATE, slots=torch.zeros(3, dtype=torch.int64)),
    dict(state=STATE, slots=torch.zeros(2, dtype=torch.int32)),
])
def test_states_refused(kw):
    with pytest.raises(ValueError, match="linear_attention"):
        linear_attention(*prompt(), **kw)
    with pytest.raises(ValueError, match="linear_attention_step"):
        linear_attention_step(*step(), **kw)


def test_prompt_options_refused():
    with pytest.raises(ValueError, match="slots need a state"):
        linear_attention(*prompt(), slots=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="lengths"):
        linear_attention(*prompt(), lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="out must be"):
        linear_attention(*prompt(), out=torch.zeros(2, 5, 4, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="out must be"):
        linear_attention_step(*step(), STATE, out=torch.zeros(2, 4, 64))


def test_written_arguments_refused():
    """What is written to may not overlap itself, nor hang in a gradient's graph."""
    out = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        linear_attention(*prompt(), out=out.expand(2, 5, 4, 64))
    with pytest.raises(ValueError, match="overlap"):
        linear_attention_step(*step(), STATE, out=out[:1, 0].expand(2, 4, 64))
    for kw in (dict(state=STATE.clone().requires_grad_()), dict(state=STATE, out=out[:, 0].clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="linear_attention_step: .*backward"):
            linear_attention_step(*step(), **kw)
    f, _ = rotary_frequencies(32, device="cpu")
    x = torch.zeros(1, 3, 2, 64)
    for q, k in ((x.expand(2, 3, 2, 64), x.repeat(2, 1, 1, 1)), (x, x[:, :, :1].expand(1, 3, 2, 64)),
                 (x[:, :1].expand(1, 3, 2, 64), None)):
        with pytest.raises(ValueError, match="overlap"):
            apply_rotary(q, k, torch.arange(3), f, inplace=True)


def test_cpu_tensors_fail_loudly():
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        linear_attention(*prompt())
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        linear_attention_step(*step(), STATE)
    f, _ = rotary_frequencies(32, device="cpu")
    x = torch.zeros(1, 3, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        apply_rotary(x, x, torch.arange(3), f)


def test_rotary_refused():
    f, _ = rotary_frequencies(32, device="cpu")
    x = torch.zeros(1, 3, 2, 64)
    pos = torch.arange(3)
    bad = [
        (ValueError, dict(layout="quarter")), (ValueError, dict(q=x[0])), (ValueError, dict(k=x[:, :2])),
        (TypeError, dict(k=x.bfloat16())), (TypeError, dict(q=x.double(), k=x.double())),
        (ValueError, dict(inv_freq=f.float())), (ValueError, dict(inv_freq=f[:0])),
        (ValueError, dict(q=x[..., :16], k=x[..., :16])), (ValueError, dict(positions=pos.int())),
        (ValueError, dict(positions=pos[None, :, None])), (ValueError, dict(positions=torch.arange(4))),
        (RuntimeError, dict(q=x.clone().requires_grad_())),
    ]
    for error, kw in bad:
        args = dict(q=x, k=x, positions=pos, inv_freq=f) | kw
        with pytest.raises(error, match="apply_rotary"):
            apply_rotary(**args)
    for kw in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=0.0),
               dict(rotary_dim=8, scaling="square"), dict(rotary_dim=8, scaling="parts", factor=2.0)):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            rotary_frequencies(device="cpu", **kw)


def test_frequencies():
    f, a = rotary_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and a == 1.0
    assert all(f[i].item() == pytest.approx(10000.0 ** (-2 * i / 64), rel=1e-14) for i in range(32))
    lin, a = rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin, f / 4) and a == 1.0
    base, a = rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert base[0] == 1.0 and base[-1].item() == pytest.approx(f[-1].item() / 4, rel=1e-12) and a == 1.0
    parts, a = rotary_frequencies(64, scaling="parts", factor=4.0, trained_length=2048, device="cpu")
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(parts[turns > 32], f[turns > 32])
    assert torch.allclose(parts[turns < 1], f[turns < 1] / 4, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (parts[mid] < f[mid]).all() and (parts[mid] > f[mid] / 4).all()
    assert a == pytest.approx(0.1 * math.log(4.0) + 1.0)


def test_c_abi_validates_on_the_host():
    lib = _lib.lib()
    buf = 4096

    def rotary(dtype=1, b=1, t=1, h=1, hk=1, d=8, r=8, q=buf):
        return lib.tf_rotary_positions_fwd(struct.pack("6Q14qd8i", q, buf, buf, buf, buf, buf, *[8] * 14, 1.0, dtype, 0,
                                                       b, t, h, hk, d, r), None)

    assert lib.tf_rotary_positions_fwd(None, None) == rotary(dtype=2) == rotary(b=-1) == rotary(r=7) == rotary(r=10) == _lib.TF_ERR_ARG
    assert rotary(q=0) == _lib.TF_ERR_ARG
    assert rotary(b=0) == rotary(t=0) == rotary(h=0, hk=0) == _lib.TF_OK
    assert rotary(d=2048, r=2048) == rotary(d=256, h=256) == rotary(b=1 << 16, t=1 << 16) == _lib.TF_ERR_SIZE

    def attention(dtype=1, state=buf, slots_n=4, fresh=0, slots=0, strides=(8,) * 17, b=2, t=3, h=4, hq=2, n=64, p=64, q=buf):
        return lib.tf_linear_attention_fwd(struct.pack("9Q2q17qd8i", q, buf, buf, buf, buf, state, slots, 0, 0, 0, slots_n,
                                                       *strides, 1.0, dtype, fresh, b, t, h, hq, n, p), None)

    assert lib.tf_linear_attention_fwd(None, None) == attention(dtype=3) == attention(h=5) == attention(hq=0) == _lib.TF_ERR_ARG
    assert attention(n=60) == attention(p=264) == attention(n=0) == attention(slots_n=1) == _lib.TF_ERR_ARG
    assert attention(state=0, slots=buf) == attention(q=0) == attention(t=-1) == _lib.TF_ERR_ARG
    assert attention(b=0) == attention(h=0, hq=1) == attention(t=0) == _lib.TF_OK
    assert attention(state=4100) == _lib.TF_ERR_LAYOUT
    sizes = dict(b=2, t=17, h=4, hq=2, n=128, p=64, dtype=1)
    chunked = lambda **kw: lib.tf_linear_attention_chunked(*(sizes | kw).values())  # noqa: E731
    assert chunked() == chunked(t=5000) == chunked(n=8, p=128) == 1
    assert chunked(t=16) == chunked(dtype=0) == chunked(n=136) == chunked(p=136) == chunked(b=0) == chunked(hq=3) == 0
    assert lib.tf_linear_attention_workspace_size(*(sizes | dict(t=16)).values()) == 0
    assert attention(strides=[8] * 15 + [6, 8]) == _lib.TF_ERR_LAYOUT


@pytest.mark.parametrize("first", ["linear_attention_step", "linear_attention", "apply_rotary", "linear_recurrence"])
def test_exports_do_not_depend_on_the_order_of_imports(first):
    """No export shares its name with a module of the package, which would take its place."""
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent / "trifusion-fp-kernel_b200"
    code = (f"import sys; sys.path.insert(0, {str(root)!r}); import trifusion_b200 as t; "
            f"exec('import trifusion_b200.{first}') if {first!r} == 'linear_recurrence' else getattr(t, {first!r}); "
            "assert all(callable(getattr(t, n)) for n in ('linear_attention', 'linear_attention_step', "
            "'apply_rotary', 'rotary_frequencies'))")
    subprocess.run([sys.executable, "-c", code], check=True)
