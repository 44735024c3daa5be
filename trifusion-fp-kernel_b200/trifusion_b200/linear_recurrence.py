"""Linear attention with a decay for each head and a carried state.

    S_t = e^(decay_t) S_(t-1) + k_t v_t^T          (N x P, FP32)
    o_t = scale * q_t S_t

``fused_mamba`` and ``fused_recurrence`` run a whole padded clip from a zero state.
These two run a causal recurrence of the same chunked kind over a stream:
``linear_attention`` a piece of any length (a prompt), ``linear_attention_step`` one
token for each row, both from and into states that the caller keeps, as one
tensor or as a pool with a slot for each row.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._autograd import has_tangent, written

_launch = _lib.launcher("tf_linear_attention_fwd", "9Q2q17qd8i")  # tf_linear_attention_io
_DTYPES = {torch.float32: _lib.TF_F32, torch.bfloat16: _lib.TF_BF16}


def _operands(op, dtype, q, k, v, decay, hq, h, n, p):
    """What both forms ask of their operands, shapes apart; returns the C ABI's dtype."""
    if hq < 1 or h % hq:
        raise ValueError(f"{op}: H must be divisible by Hq")
    if n % 8 or p % 8 or n < 8 or p < 8 or n > 256 or p > 256:
        raise ValueError(f"{op}: N and P must be multiples of 8 from 8 to 256")
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{op}: expected float32 or bfloat16, got {dtype}")
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"{op}: q, k and v must have one dtype")
    if decay.dtype != torch.float32:
        raise TypeError(f"{op}: decay must be float32")
    if (q.requires_grad or k.requires_grad or v.requires_grad or decay.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError(f"{op}: {_lib.NO_GRADIENT}")
    return code


def _meet(s0, n0, s1, n1, size):
    """Whether two of the n0 x n1 pieces of ``size`` values at i * s0 + j * s1 overlap (neither stride
    being below ``size``)."""
    if s0 >= s1 * (n1 - 1) + size or s1 >= s0 * (n0 - 1) + size:
        return False
    return any(0 < i < n0 and abs(j * s1 - i * s0) < size for j in range(1, n1) for i in (j * s1 // s0, j * s1 // s0 + 1))


def _check_state(op, state, slots, b, h, n, p):
    """Checks a state and its slots; returns the state's strides over slots and heads."""
    shape = state.shape
    if state.dtype != torch.float32 or len(shape) != 4 or shape[1:] != (h, n, p):
        raise ValueError(f"{op}: state must be float32 [slots,H,N,P]")
    s0, s1, s2, s3 = state.stride()
    if s3 != 1 or s2 != p or s0 % 4 or s1 % 4 or state.data_ptr() % 16:
        raise ValueError(f"{op}: state must be contiguous over [N,P], its heads on 16-byte boundaries")
    size, pool = n * p, shape[0]
    if (s1 < size and h > 1) or (s0 < size and pool > 1) or (h > 1 and pool > 1 and _meet(s0, pool, s1, h, size)):
        raise ValueError(f"{op}: the states of a pool must not overlap")
    if state.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{op}: {_lib.NO_GRADIENT}")
    if slots is None:
        if shape[0] != b:
            raise ValueError(f"{op}: without slots, state must have one entry for each row")
    elif slots.dtype != torch.int64 or slots.shape != (b,):
        raise ValueError(f"{op}: slots must be int64 [B]")
    return s0, s1


def _check_out(op, out, v):
    if out.shape != v.shape or out.dtype != v.dtype or out.stride(-1) != 1:
        raise ValueError(f"{op}: out must be like v with a unit stride in the last dimension")
    if out.numel() and not out.is_contiguous() and _lib.overlaps_itself(out):
        raise ValueError(f"{op}: out must not overlap itself")
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{op}: {_lib.NO_GRADIENT}")


def _on(index, x):
    return x is None or x.get_device() == index


def _aligned(x):
    """Whether tile loads and stores can address ``x`` ([B,T,heads,width] BF16)."""
    if x.data_ptr() % 16:
        return False
    (b, t, h, _), (sb, st, sh, _) = x.shape, x.stride()
    return not ((b > 1 and (sb % 8 or sb <= 0)) or (t > 1 and (st % 8 or st <= 0)) or (h > 1 and (sh % 8 or sh <= 0)))


@functools.lru_cache(maxsize=4096)
def _plan(device, *sizes):
    """Whether a piece of these sizes runs in chunks, and the bytes of workspace it takes then."""
    with torch.cuda.device(device):
        lib = _lib.lib()
        return lib.tf_linear_attention_chunked(*sizes), lib.tf_linear_attention_workspace_size(*sizes)


def linear_attention(q, k, v, decay, state=None, *, slots=None, lengths=None, scale=None, out=None):
    """A piece of T tokens for each row: returns ``(out, state)``.

    * ``q``, ``k`` [B,T,Hq,N], ``v`` [B,T,H,P], BF16 or FP32, H a multiple of Hq, N and P
      multiples of 8 up to 256; ``decay`` FP32 [B,H,T], or [H] for one decay a head: natural
      logs, at most 0 in use; ``-inf`` forgets everything before, states that are not finite
      included (an entry of a pool needs no clearing where its first decay is ``-inf``).
    * ``state`` FP32 [B,H,N,P] is the state before the first token and is overwritten by
      the state after the last. With ``slots`` (int64 [B]) it is a pool [slots,H,N,P] and row
      b works on entry ``slots[b]``. A row with a negative slot is padding: its output is
      zero and no state changes. A slot past the pool, or one that an earlier row has, gives
      NaN outputs and changes no state. ``None``: rows start at zero and a new [B,H,N,P] is
      returned.
    * ``lengths`` (int64 [B], on the device): tokens at or past a row's length are not
      read, and their output is zero.
    * ``scale`` defaults to ``N ** -0.5``; ``out``: a preallocated output like v with a unit
      stride in the last dimension. ``out`` and ``state`` overlap no other argument.

    BF16 operands with N and P up to 128 run on the tensor cores in chunks of 64 tokens
    (FP32 sums and state). A non-finite value in v then also reaches the earlier tokens of
    its chunk, and, with P up to 64, a non-finite weight (a NaN in a head's decays, say) the
    outputs of the head next to it under the same key head; a decay of ``-inf`` does not stop
    what is not finite in the tokens of its own chunk. FP32 operands, wider heads and
    pieces of up to 16 tokens run token by token. There is no backward pass.
    """
    op = "linear_attention"
    shape = q.shape
    if len(shape) != 4 or v.dim() != 4 or k.shape != shape:
        raise ValueError(f"{op}: q and k must be [B,T,Hq,N] and v [B,T,H,P]")
    b, t, hq, n = shape
    vb, vt, h, p = v.shape
    if vb != b or vt != t:
        raise ValueError(f"{op}: q and k must be [B,T,Hq,N] and v [B,T,H,P]")
    if has_tangent(q, k, v, decay, state, out):
        raise RuntimeError(f"{op}: {_lib.NO_TANGENT}")
    dtype, index = _operands(op, q.dtype, q, k, v, decay, hq, h, n, p), q.get_device()
    sg, shape = decay.stride(), decay.shape
    if shape == (h,) and sg:
        sg = (0, sg[0], 0)
    elif shape != (b, h, t):
        raise ValueError(f"{op}: decay must be [B,H,T] or [H]")
    fresh = state is None
    if not fresh:
        ss = _check_state(op, state, slots, b, h, n, p)
    elif slots is not None:
        raise ValueError(f"{op}: slots need a state")
    if lengths is not None and (lengths.dtype != torch.int64 or lengths.shape != (b,)):
        raise ValueError(f"{op}: lengths must be int64 [B]")
    if out is not None:
        _check_out(op, out, v)
    if (index < 0 or k.get_device() != index or v.get_device() != index or decay.get_device() != index
            or not (_on(index, state) and _on(index, slots) and _on(index, lengths) and _on(index, out))):
        raise RuntimeError(f"{op}: all tensors must be CUDA tensors on one device")
    q0, q1, q2, q3 = q.stride()
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if q3 != 1 or k3 != 1 or v3 != 1:
        q, k, v = [x if x.stride(3) == 1 else x.contiguous() for x in (q, k, v)]
        (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _) = q.stride(), k.stride(), v.stride()
    given = out is not None
    if not given:
        out, o0, o1, o2 = torch.empty_like(v, memory_format=torch.contiguous_format), t * h * p, h * p, p
    else:
        o0, o1, o2, _ = out.stride()
    if fresh:
        ss = (h * n * p, n * p)  # (the strided form is the faster call)
        state = torch.empty_strided((b, h, n, p), (*ss, p, 1), dtype=torch.float32, device=v.device)
    if not _lib._watch["ready"]:
        _lib.error_watch()
    _lib.check_device_error()
    chunked, nbytes = _plan(index, b, t, h, hq, n, p, dtype)
    slot, length, work, wp, into = 0, 0, None, 0, out
    qp, kp, vp, outp = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if chunked:  # its tile loads and stores need 16-byte rows
        strides = (q0, q1, q2, k0, k1, k2, v0, v1, v2, o0, o1, o2)
        if (qp | kp | vp | outp) & 15 or (q0 | q1 | q2 | k0 | k1 | k2 | v0 | v1 | v2 | o0 | o1 | o2) & 7 or min(strides) <= 0:
            q, k, v = [x if _aligned(x) else x.clone(memory_format=torch.contiguous_format) for x in (q, k, v)]
            if not _aligned(out):
                into = torch.empty((b, t, h, p), dtype=v.dtype, device=v.device)
            (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _) = q.stride(), k.stride(), v.stride()
            o0, o1, o2, _ = into.stride()
            qp, kp, vp, outp = q.data_ptr(), k.data_ptr(), v.data_ptr(), into.data_ptr()
        if nbytes:
            work = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=v.device)
            wp = work.data_ptr()
    if slots is not None:
        slots = slots.contiguous()
        slot = slots.data_ptr()
    if lengths is not None:
        lengths = lengths.contiguous()
        length = lengths.data_ptr()
    _launch(index, qp, kp, vp, outp, decay.data_ptr(), state.data_ptr(), slot, length, wp, nbytes, state.shape[0],
            q0, q1, q2, k0, k1, k2, v0, v1, v2, *sg, o0, o1, o2, *ss, n ** -0.5 if scale is None else scale,
            dtype, fresh, b, t, h, hq, n, p)
    if into is not out:
        out.copy_(into)
    if not fresh:
        written(state)
    if given:
        written(out)
    return out, state


def linear_attention_step(q, k, v, decay, state, *, slots=None, scale=None, out=None):
    """One token for each row: returns the output [B,H,P] and updates ``state`` in place.

    ``q``, ``k`` [B,Hq,N], ``v`` [B,H,P], BF16 or FP32; ``decay`` FP32 [B,H] or [H]; ``state``,
    ``slots``, ``scale`` and ``out`` as in :func:`linear_attention` (a batch padded for a
    captured graph gives its padding rows the slot -1).
    """
    op = "linear_attention_step"
    shape = q.shape
    if len(shape) != 3 or v.dim() != 3 or k.shape != shape:
        raise ValueError(f"{op}: q and k must be [B,Hq,N] and v [B,H,P]")
    b, hq, n = shape
    vb, h, p = v.shape
    if vb != b:
        raise ValueError(f"{op}: q and k must be [B,Hq,N] and v [B,H,P]")
    if has_tangent(q, k, v, decay, state, out):
        raise RuntimeError(f"{op}: {_lib.NO_TANGENT}")
    dtype, index = _operands(op, q.dtype, q, k, v, decay, hq, h, n, p), q.get_device()
    sg, shape = decay.stride(), decay.shape
    if shape == (h,) and sg:
        sg = (0, sg[0])
    elif shape != (b, h):
        raise ValueError(f"{op}: decay must be [B,H] or [H]")
    ss = _check_state(op, state, slots, b, h, n, p)
    if out is not None:
        _check_out(op, out, v)
    if (index < 0 or k.get_device() != index or v.get_device() != index or decay.get_device() != index
            or state.get_device() != index or not (_on(index, slots) and _on(index, out))):
        raise RuntimeError(f"{op}: all tensors must be CUDA tensors on one device")
    qb, qh, q1 = q.stride()
    kb, kh, k1 = k.stride()
    vb, vh, v1 = v.stride()
    if q1 != 1:
        q = q.contiguous()
        qb, qh, _ = q.stride()
    if k1 != 1:
        k = k.contiguous()
        kb, kh, _ = k.stride()
    if v1 != 1:
        v = v.contiguous()
        vb, vh, _ = v.stride()
    slot = 0
    if slots is not None:
        slots = slots.contiguous()
        slot = slots.data_ptr()
    given = out is not None
    if not given:
        out, ob, oh = torch.empty_like(v, memory_format=torch.contiguous_format), h * p, p
    else:
        ob, oh, _ = out.stride()
    _launch(index, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), decay.data_ptr(), state.data_ptr(), slot, 0,
            0, 0, state.shape[0], qb, 0, qh, kb, 0, kh, vb, 0, vh, *sg, 0, ob, 0, oh, *ss,
            n ** -0.5 if scale is None else scale, dtype, 0, b, 1, h, hq, n, p)
    written(state)
    if given:
        written(out)
    return out
