"""The gated linear recurrence: a mixer whose decays depend on the token, for prompts, training and single tokens.

``gated_recurrence`` over sequences, ``gated_recurrence_step`` (one token per row on a pool of states). Types, streams,
derivatives and errors are those of the token operators (token_ops.py).
"""

from __future__ import annotations

import functools
import struct
from typing import Optional

import torch

from . import _lib, engine
from .engine import first_order
from .token_ops import _DTYPES, _addr, _device, _dtype, _last_contiguous, _launch, _work

_RECUR = struct.Struct("@4i3P6q3P3PP2qP3P2PPNP").pack  # ews_recur_args


@functools.lru_cache(maxsize=256)
def _sizes(B: int, T: int, C: int, code: int):
    """(carry, forward's and backward's workspace) in bytes: a function of the sizes alone."""
    lib, args = _lib.load(), _RECUR(B, T, C, code, *([0] * 27))
    return lib.ews_recur_carry_size(args), lib.ews_recur_work_size(args, 0), lib.ews_recur_work_size(args, 1)


def _forward(x, decay, gate, rate, initial, lengths, want_state, want_carry):
    (B, T, C), code = x.shape, _DTYPES[x.dtype]
    carry_bytes, size, _ = _sizes(B, T, C, code)
    out = x.new_empty((B, T, C))
    end = rate.new_empty((B, C)) if want_state else None
    carry = rate.new_empty(carry_bytes // 4) if want_carry else None
    work = _work(size, x)
    idx, xs, ds, gs = x.get_device(), x.stride(), decay.stride(), gate.stride()
    args = _RECUR(B, T, C, code, x.data_ptr(), decay.data_ptr(), gate.data_ptr(), xs[0], xs[1], ds[0], ds[1], gs[0], gs[1], rate.data_ptr(),
                  _addr(lengths), _addr(initial), out.data_ptr(), _addr(end), _addr(carry), 0, 0, 0, 0, 0, 0, 0, 0, 0, _addr(work), size,
                  engine.index_word(idx)[0])
    _launch(idx, "ews_recur_fwd", B * T, _lib.load().ews_recur_fwd, args)
    return out, end, carry


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, decay, gate, rate, initial, lengths, want_state):
        x, decay, gate = _last_contiguous(x), _last_contiguous(decay), _last_contiguous(gate)
        out, end, carry = _forward(x, decay, gate, rate, initial, lengths, want_state, True)
        ctx.save_for_backward(x, decay, gate, rate, initial, lengths, carry)
        ctx.set_materialize_grads(False)
        return out, end

    @staticmethod
    @first_order
    def backward(ctx, dout, dend):
        x, decay, gate, rate, initial, lengths, carry = ctx.saved_tensors
        (B, T, C), code = x.shape, _DTYPES[x.dtype]
        dout = None if dout is None else _last_contiguous(dout)
        dend = None if dend is None else dend.contiguous()
        dx, ddecay, dgate = x.new_empty((B, T, C)), x.new_empty((B, T, C)), x.new_empty((B, T, C))
        drate = rate.new_empty(C) if ctx.needs_input_grad[3] else None
        d0 = rate.new_empty((B, C)) if ctx.needs_input_grad[4] else None
        size = _sizes(B, T, C, code)[2]
        work = _work(size, x)
        idx, xs, ds, gs = x.get_device(), x.stride(), decay.stride(), gate.stride()
        os = (0, 0) if dout is None else dout.stride()
        args = _RECUR(B, T, C, code, x.data_ptr(), decay.data_ptr(), gate.data_ptr(), xs[0], xs[1], ds[0], ds[1], gs[0], gs[1],
                      rate.data_ptr(), _addr(lengths), _addr(initial), 0, 0, carry.data_ptr(), _addr(dout), os[0], os[1], _addr(dend),
                      dx.data_ptr(), ddecay.data_ptr(), dgate.data_ptr(), _addr(drate), _addr(d0), _addr(work), size, engine.index_word(idx)[0])
        _launch(idx, "ews_recur_bwd", B * T, _lib.load().ews_recur_bwd, args)
        return dx, ddecay, dgate, drate, d0, None, None


def _check(x, decay, gate, rate, axes):
    if not (x.dtype == decay.dtype == gate.dtype):
        raise TypeError(f"x, decay and gate must share a type, got {x.dtype}, {decay.dtype}, {gate.dtype}")
    _dtype(x, "x, decay and gate")
    shape = x.shape
    if len(shape) != axes or shape[-1] == 0 or decay.shape != shape or gate.shape != shape:
        raise ValueError(f"x, decay and gate must share a shape of {axes} axes with channels, got {tuple(shape)}, "
                         f"{tuple(decay.shape)}, {tuple(gate.shape)}")
    C = shape[-1]
    if rate.shape != (C,) or rate.dtype != torch.float32 or not rate.is_contiguous():
        raise ValueError(f"rate must be a contiguous float32 tensor of {C} values, got {rate.dtype} {tuple(rate.shape)}")
    return C


def gated_recurrence(x: torch.Tensor, decay: torch.Tensor, gate: torch.Tensor, rate: torch.Tensor, *,
                     initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                     return_state: bool = False):
    """A linear recurrence a channel whose decay and input the token gates:
    ``a_t = exp(-rate sigmoid(decay_t))``, ``h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_t) x_t``.

    x, decay, gate (B, T, C), float32 or bfloat16, any strides (views of one projection, for instance); rate (C,) float32,
    zero or larger (a negative one gives NaN): a diagonal generator's rates, with ``sigmoid(decay)`` as the clock's step.
    A decay of -inf, or of its type's lowest value, passes the state on unchanged and takes no input, whatever the token
    holds (NaN and infinities too). initial_state (B, C)
    float32 or None (zero). lengths (B,) int32: positions at or beyond a sample's length are not read, give zeros and
    leave the state.

    Returns h (B, T, C), with ``return_state`` also the state after the last token (B, C) float32, for
    ``gated_recurrence_step`` or the next piece of a long sequence; states and the scan are float32 whatever the type.
    Differentiable in x, decay, gate, rate and initial_state; results do not depend on timing."""
    C = _check(x, decay, gate, rate, 3)
    B = x.shape[0]
    if initial_state is not None:
        if initial_state.shape != (B, C) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state must be float32 {(B, C)}, got {initial_state.dtype} {tuple(initial_state.shape)}")
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.dtype != torch.int32:
            raise ValueError(f"lengths must be int32 ({B},), got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    _device(x, decay, gate, rate, initial_state, lengths)
    want = bool(return_state)
    if torch.is_grad_enabled() and (x.requires_grad or decay.requires_grad or gate.requires_grad or rate.requires_grad
                                    or initial_state is not None and initial_state.requires_grad):
        out, end = _Recurrence.apply(x, decay, gate, rate, initial_state, lengths, want)
    else:
        x, decay, gate = _last_contiguous(x), _last_contiguous(decay), _last_contiguous(gate)
        out, end, _ = _forward(x, decay, gate, rate, initial_state, lengths, want, False)
    return (out, end) if want else out


def gated_recurrence_step(x: torch.Tensor, decay: torch.Tensor, gate: torch.Tensor, rate: torch.Tensor, state: torch.Tensor, *,
                          slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token per row of ``gated_recurrence`` on a pool of states, updated in place.

    x, decay, gate (B, C); state (P, C) float32, contiguous. Row b works on state ``slots[b]`` (int32 (B,); None: b, with
    P >= B). A negative slot is a row without a request: its output is zero and no state is touched. Two rows must not share
    a slot; one out of range gives a zero row and IndexError on the next call. Returns h (B, C). For serving: no
    gradient; a backward that needs the states as they were raises, as after any operation in place."""
    C = _check(x, decay, gate, rate, 2)
    B, pool = x.shape[0], state.shape
    if len(pool) != 2 or pool[1] != C or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32 (P, {C}), got {state.dtype} {tuple(pool)}")
    if slots is None:
        if pool[0] < B:
            raise ValueError(f"{B} rows need as many states or slots, got {pool[0]} states")
    elif slots.shape != (B,) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError(f"slots must be contiguous int32 ({B},), got {slots.dtype} {tuple(slots.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or decay.requires_grad or gate.requires_grad or rate.requires_grad
                                    or state.requires_grad):
        raise RuntimeError("gated_recurrence_step has no gradient: call it under torch.no_grad()")
    idx = _device(x, decay, gate, rate, state, slots)
    (xs, x1), (ds, d1), (gs, g1) = x.stride(), decay.stride(), gate.stride()
    if (x1 != 1 or d1 != 1 or g1 != 1) and C > 1:
        x, decay, gate = x.contiguous(), decay.contiguous(), gate.contiguous()
        xs = ds = gs = C
    out = x.new_empty((B, C))
    args = _RECUR(B, 1, C, _DTYPES[x.dtype], x.data_ptr(), decay.data_ptr(), gate.data_ptr(), xs, 0, ds, 0, gs, 0, rate.data_ptr(),
                  0, 0, out.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, engine.index_word(idx)[0])
    _launch(idx, "ews_recur_step", B, _lib.load().ews_recur_step, args, 0 if slots is None else slots.data_ptr(), pool[0],
            state.data_ptr())
    if not state.is_inference():  # autograd cannot see the write: a backward that saved these states must
        torch.autograd.graph.increment_version(state)
    return out
