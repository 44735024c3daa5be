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

import torch

from . import _lib


def _prep(op, q, k, v, decay, time):
    """Shapes, types and devices of one call; ``time``: with a T dimension."""
    dims = 4 if time else 3
    lead = v.shape[:-2]
    if v.dim() != dims or q.dim() != dims or q.shape != k.shape or q.shape[:-2] != lead:
        raise ValueError(f"{op}: q and k must be {'[B,T,Hq,N]' if time else '[B,Hq,N]'} and v "
                         f"{'[B,T,H,P]' if time else '[B,H,P]'}")
    hq, n = q.shape[-2:]
    h, p = v.shape[-2:]
    if hq < 1 or h % hq:
        raise ValueError(f"{op}: H must be divisible by Hq")
    for w in (n, p):
        if w % 8 or not 8 <= w <= 256:
            raise ValueError(f"{op}: N and P must be multiples of 8 from 8 to 256")
    dtype = _lib.dtype_code(q, op)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{op}: q, k and v must have one dtype")
    shape = (lead[0], h, lead[1]) if time else (lead[0], h)
    if decay.dtype != torch.float32:
        raise TypeError(f"{op}: decay must be float32")
    if decay.dim() == 1 and decay.shape[0] == h:
        decay = decay.view(1, h, 1).expand(shape) if time else decay.view(1, h).expand(shape)
    elif tuple(decay.shape) != shape:
        raise ValueError(f"{op}: decay must be {'[B,H,T]' if time else '[B,H]'} or [H]")
    _lib.no_gradient(op, q, k, v, decay)
    q, k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (q, k, v))
    return q, k, v, decay, dtype


def _check_state(op, state, slots, b, h, n, p):
    if state.dtype != torch.float32 or state.dim() != 4 or tuple(state.shape[1:]) != (h, n, p):
        raise ValueError(f"{op}: state must be float32 [slots,H,N,P]")
    if (state.stride(3) != 1 or state.stride(2) != p or state.data_ptr() % 16
            or state.stride(0) % 4 or state.stride(1) % 4):
        raise ValueError(f"{op}: state must be contiguous over [N,P], its heads on 16-byte boundaries")
    if state.stride(1) < n * p or state.stride(0) < n * p:
        raise ValueError(f"{op}: the states of a pool must not overlap")
    if slots is None:
        if state.shape[0] != b:
            raise ValueError(f"{op}: without slots, state must have one entry for each row")
    elif slots.dtype != torch.int64 or tuple(slots.shape) != (b,):
        raise ValueError(f"{op}: slots must be int64 [B]")


def _aligned(x):
    return x.data_ptr() % 16 == 0 and all(e == 1 or (s > 0 and s % 8 == 0) for e, s in zip(x.shape[:3], x.stride()))


def linear_attention(q, k, v, decay, state=None, *, slots=None, lengths=None, scale=None, out=None):
    """A piece of T tokens for each row: returns ``(out, state)``.

    * ``q``, ``k`` [B,T,Hq,N], ``v`` [B,T,H,P], BF16 or FP32, H a multiple of Hq, N and P
      multiples of 8 up to 256; ``decay`` FP32 [B,H,T], or [H] for one decay a head: natural
      logs, at most 0 in use; ``-inf`` forgets everything before.
    * ``state`` FP32 [B,H,N,P] is the state before the first token and is overwritten by
      the state after the last. With ``slots`` (int64 [B]) it is a pool [slots,H,N,P] and row
      b works on entry ``slots[b]``. A row with a negative slot is padding: its output is
      zero and no state changes. A slot past the pool, or one that an earlier row has, gives
      NaN outputs and changes no state. ``None``: rows start at zero and a new [B,H,N,P] is
      returned.
    * ``lengths`` (int64 [B], on the device): tokens at or past a row's length are not
      read, and their output is zero.
    * ``scale`` defaults to ``N ** -0.5``; ``out``: a preallocated output like v with a unit
      stride in the last dimension.

    BF16 operands with N and P up to 128 run on the tensor cores in chunks of 64 tokens
    (FP32 sums and state); a non-finite value in v or k then also reaches the earlier
    tokens of its chunk. FP32 operands, wider heads and short pieces run token by token.
    There is no backward pass.
    """
    op = "linear_attention"
    q, k, v, decay, dtype = _prep(op, q, k, v, decay, True)
    b, t, hq, n = q.shape
    h, p = v.shape[2:]
    tensors = [q, k, v, decay]
    if slots is not None and state is None:
        raise ValueError(f"{op}: slots need a state")
    if state is not None:
        _check_state(op, state, slots, b, h, n, p)
        tensors.append(state)
    if slots is not None:
        slots = slots.contiguous()
        tensors.append(slots)
    if lengths is not None:
        if lengths.dtype != torch.int64 or tuple(lengths.shape) != (b,):
            raise ValueError(f"{op}: lengths must be int64 [B]")
        lengths = lengths.contiguous()
        tensors.append(lengths)
    if out is not None:
        if out.shape != v.shape or out.dtype != v.dtype or out.stride(3) != 1:
            raise ValueError(f"{op}: out must be like v with a unit stride in the last dimension")
        tensors.append(out)
    dev = _lib.require_cuda(op, *tensors)
    if out is None:
        out = torch.empty((b, t, h, p), dtype=v.dtype, device=dev)
    fresh = state is None
    if fresh:
        state = torch.empty((b, h, n, p), dtype=torch.float32, device=dev)
    _lib.error_watch()
    _lib.check_device_error()
    nbytes = _lib.lib().tf_linear_attention_workspace_size(b, t, h, hq, n, p, dtype)
    work, into = None, out
    if nbytes:  # the chunked form, whose tile loads need 16-byte rows
        q, k, v = (x if _aligned(x) else x.clone(memory_format=torch.contiguous_format) for x in (q, k, v))
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        if not _aligned(out):
            into = torch.empty((b, t, h, p), dtype=v.dtype, device=dev)
    strides = _lib.int64_array((*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *decay.stride(),
                                *into.stride()[:3], *state.stride()[:2]))
    _lib.launch("tf_linear_attention_fwd", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype, decay.data_ptr(),
                state.data_ptr(), state.shape[0], fresh, None if slots is None else slots.data_ptr(),
                None if lengths is None else lengths.data_ptr(), into.data_ptr(), strides, b, t, h, hq, n, p,
                n ** -0.5 if scale is None else float(scale), None if work is None else work.data_ptr(), nbytes)
    if into is not out:
        out.copy_(into)
    return out, state


def linear_attention_step(q, k, v, decay, state, *, slots=None, scale=None, out=None):
    """One token for each row: returns the output [B,H,P] and updates ``state`` in place.

    ``q``, ``k`` [B,Hq,N], ``v`` [B,H,P], BF16 or FP32; ``decay`` FP32 [B,H] or [H]; ``state``,
    ``slots``, ``scale`` and ``out`` as in :func:`linear_attention` (a batch padded for a
    captured graph gives its padding rows the slot -1).
    """
    op = "linear_attention_step"
    q, k, v, decay, dtype = _prep(op, q, k, v, decay, False)
    b, hq, n = q.shape
    h, p = v.shape[1:]
    _check_state(op, state, slots, b, h, n, p)
    tensors = [q, k, v, decay, state]
    if slots is not None:
        slots = slots.contiguous()
        tensors.append(slots)
    if out is not None:
        if out.shape != v.shape or out.dtype != v.dtype or out.stride(2) != 1:
            raise ValueError(f"{op}: out must be like v with a unit stride in the last dimension")
        tensors.append(out)
    dev = _lib.require_cuda(op, *tensors)
    if out is None:
        out = torch.empty((b, h, p), dtype=v.dtype, device=dev)
    (qb, qh), (kb, kh), (vb, vh), (ob, oh) = (x.stride()[:2] for x in (q, k, v, out))
    strides = _lib.int64_array((qb, 0, qh, kb, 0, kh, vb, 0, vh, *decay.stride(), 0, ob, 0, oh, *state.stride()[:2]))
    _lib.launch("tf_linear_attention_fwd", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype, decay.data_ptr(),
                state.data_ptr(), state.shape[0], 0, None if slots is None else slots.data_ptr(), None,
                out.data_ptr(), strides, b, 1, h, hq, n, p, n ** -0.5 if scale is None else float(scale), None, 0)
    return out
