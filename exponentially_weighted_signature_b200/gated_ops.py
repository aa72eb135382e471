"""The gated linear layer: a block's channel stage up to its last projection.

``gated_linear``: both projections, the activation and the product in one kernel, with its gradients; for training, prompts and
single tokens. Types, streams, derivatives and errors are those of the token operators (token_ops.py).
"""

from __future__ import annotations

import functools
import struct

import torch

from . import _lib, engine
from .engine import first_order
from .token_ops import _DTYPES, _addr, _device, _dtype, _launch, _operand, _work

ACTIVATIONS = {"silu": 0, "gelu": 1}
_GATED = struct.Struct("@3q2i3P3q3Pq4PNP").pack  # ews_gated_args
_BF16 = _lib.EWS_DTYPE_BF16


@functools.lru_cache(maxsize=256)
def _size(rows, dim, inner, code, strides, at, wanted, backward):
    """Workspace bytes: a function of the sizes, the strides, the addresses modulo 16 and the gradients asked for."""
    args = _GATED(rows, dim, inner, code, 0, *at, *strides, 0, 0, 0, inner, *wanted, 0, 0, 0)
    return _lib.load().ews_gated_work_size(args, backward)


@functools.lru_cache(maxsize=256)
def _kept_size(rows, dim, inner, code):
    return _lib.load().ews_gated_kept_size(_GATED(rows, dim, inner, code, 0, 0, 0, 0, dim, dim, dim, *([0] * 10)))


def _forward(x, wg, wu, act, shape, keep):
    """The layer on operands: (tensor, stride) each. A single token's call is the host's time: what it can do without it does not
    ask for."""
    (x, xs), (wg, gs), (wu, us) = x, wg, wu
    rows, dim = x.shape
    inner, code = wg.shape[0], _DTYPES[x.dtype]
    xp, gp, up = x.data_ptr(), wg.data_ptr(), wu.data_ptr()
    out = x.new_empty(shape)
    kept = _work(_kept_size(rows, dim, inner, code), x) if keep else None
    work, size = 0, 0
    if code != _BF16 or (xs | gs | us | dim) & 7 or (xp | gp | up) & 15:  # else nothing is packed
        size = _size(rows, dim, inner, code, (xs, gs, us), (xp % 16, gp % 16, up % 16), (0, 0, 0), 0)
        space = _work(size, x)
        work = _addr(space)
    idx = x.get_device()
    args = _GATED(rows, dim, inner, code, act, xp, gp, up, xs, gs, us, out.data_ptr(), _addr(kept), 0, 0, 0, 0, 0, work, size,
                  engine.index_word(idx)[0])
    _launch(idx, "ews_gated_fwd", rows, _lib.load().ews_gated_fwd, args)
    return out, kept


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, act, shape):
        x, wg, wu = _operand(x), _operand(wg), _operand(wu)
        out, kept = _forward(x, wg, wu, act, shape, True)
        ctx.meta = act, x[1], wg[1], wu[1]
        ctx.save_for_backward(x[0], wg[0], wu[0], kept)
        return out

    @staticmethod
    @first_order
    def backward(ctx, dout):
        x, wg, wu, kept = ctx.saved_tensors
        act, xs, gs, us = ctx.meta
        (rows, dim), inner, code = x.shape, wg.shape[0], _DTYPES[x.dtype]
        dout, ds = _operand(dout if dout.dim() == 2 else dout.reshape(rows, inner))
        dx, dwg, dwu = (t.new_empty(t.shape) if need else None
                        for t, need in zip((x, wg, wu), ctx.needs_input_grad))
        xp, gp, up = x.data_ptr(), wg.data_ptr(), wu.data_ptr()
        size = _size(rows, dim, inner, code, (xs, gs, us), (xp % 16, gp % 16, up % 16),
                     (int(dx is not None), int(dwg is not None), int(dwu is not None)), 1)
        work = _work(size, x)
        idx = x.get_device()
        args = _GATED(rows, dim, inner, code, act, xp, gp, up, xs, gs, us, 0, _addr(kept), dout.data_ptr(), ds, _addr(dx), _addr(dwg),
                      _addr(dwu), _addr(work), size, engine.index_word(idx)[0])
        _launch(idx, "ews_gated_bwd", rows, _lib.load().ews_gated_bwd, args)
        return dx, dwg, dwu, None, None


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``act(x @ gate_weight.T) * (x @ up_weight.T)`` with both products, the activation and their product in one kernel.

    x (..., D); gate_weight and up_weight (F, D), all float32 or all bfloat16 (rows of any stride). activation: "silu",
    ``g sigmoid(g)``, or "gelu", ``g Phi(g)``. Returns (..., F). Sums are float32; the product is formed from them and rounded
    once. Differentiable in x and both weights (the two projections are kept for it, 6 bytes a pair for bfloat16, 8 for float32); in
    float32, gradients are NaN where an infinity, or a value that bfloat16 rounds to one, enters them."""
    inner = gate_weight.shape
    if len(inner) != 2 or up_weight.shape != inner or 0 in inner:
        raise ValueError(f"gate_weight and up_weight must be (F, D) with F, D > 0, got {tuple(inner)} and {tuple(up_weight.shape)}")
    shape = x.shape
    if not shape or shape[-1] != inner[1]:
        raise ValueError(f"x {tuple(shape)} and weights {tuple(inner)} do not fit together")
    if not (x.dtype == gate_weight.dtype == up_weight.dtype):
        raise TypeError(f"x and the weights must share a type, got {x.dtype}, {gate_weight.dtype}, {up_weight.dtype}")
    _dtype(x, "x and the weights")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}, got {activation!r}")
    _device(x, gate_weight, up_weight)
    flat = x if len(shape) == 2 else x.reshape(-1, inner[1])
    shape = (*shape[:-1], inner[0])
    if torch.is_grad_enabled() and (x.requires_grad or gate_weight.requires_grad or up_weight.requires_grad):
        return _Gated.apply(flat, gate_weight, up_weight, act, shape)
    return _forward(_operand(flat), _operand(gate_weight), _operand(up_weight), act, shape, False)[0]
