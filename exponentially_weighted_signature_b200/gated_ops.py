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
from .token_ops import _DTYPES, _addr, _device, _dtype, _launch, _row_stride, _rows, _work

ACTIVATIONS = {"silu": 0, "gelu": 1}
_GATED = struct.Struct("@3q2i3P3q3Pq4PNP").pack  # ews_gated_args


def _args(x, wg, wu, act, out=None, kept=None, dout=None, grads=(None, None, None), work=None):
    (rows, dim), inner = x.shape, wg.shape[0]
    return _GATED(rows, dim, inner, _DTYPES[x.dtype], act, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _row_stride(x),
                  _row_stride(wg), _row_stride(wu), _addr(out), _addr(kept), _addr(dout),
                  0 if dout is None else _row_stride(dout), *map(_addr, grads), _addr(work), 0 if work is None else work.numel(),
                  engine.index_word(x.get_device())[0])


@functools.lru_cache(maxsize=256)
def _size(rows, dim, inner, code, strides, at, wanted, backward):
    """Workspace bytes: a function of the sizes, the strides, the addresses modulo 16 and the gradients asked for."""
    args = _GATED(rows, dim, inner, code, 0, *at, *strides, 0, 0, 0, inner, *wanted, 0, 0, 0)
    return _lib.load().ews_gated_work_size(args, backward)


@functools.lru_cache(maxsize=256)
def _kept_size(rows, dim, inner, code):
    return _lib.load().ews_gated_kept_size(_GATED(rows, dim, inner, code, 0, 0, 0, 0, dim, dim, dim, *([0] * 10)))


def _workspace(x, wg, wu, wanted, backward):
    at = (x.data_ptr() % 16, wg.data_ptr() % 16, wu.data_ptr() % 16)
    strides = (_row_stride(x), _row_stride(wg), _row_stride(wu))
    return _work(_size(*x.shape, wg.shape[0], _DTYPES[x.dtype], strides, at, wanted, backward), x)


def _forward(x, wg, wu, act, shape, keep):
    lib = _lib.load()
    rows, inner = x.shape[0], wg.shape[0]
    out = torch.empty(shape, dtype=x.dtype, device=x.device)
    kept = _work(_kept_size(rows, x.shape[1], inner, _DTYPES[x.dtype]), x) if keep else None
    work = _workspace(x, wg, wu, (0, 0, 0), 0)
    _launch(x.get_device(), "ews_gated_fwd", rows, lib.ews_gated_fwd, _args(x, wg, wu, act, out, kept, work=work))
    return out, kept


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, act, shape):
        x, wg, wu = _rows(x), _rows(wg), _rows(wu)
        out, kept = _forward(x, wg, wu, act, shape, True)
        ctx.act = act
        ctx.save_for_backward(x, wg, wu, kept)
        return out

    @staticmethod
    @first_order
    def backward(ctx, dout):
        x, wg, wu, kept = ctx.saved_tensors
        lib = _lib.load()
        dout = _rows(dout.reshape(x.shape[0], wg.shape[0]))
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None
                 for t, need in zip((x, wg, wu), ctx.needs_input_grad)]
        work = _workspace(x, wg, wu, tuple(int(g is not None) for g in grads), 1)
        args = _args(x, wg, wu, ctx.act, None, kept, dout, grads, work)
        _launch(x.get_device(), "ews_gated_bwd", x.shape[0], lib.ews_gated_bwd, args)
        return (*grads, None, None)


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``act(x @ gate_weight.T) * (x @ up_weight.T)`` with both products, the activation and their product in one kernel.

    x (..., D); gate_weight and up_weight (F, D), all float32 or all bfloat16 (rows of any stride). activation: "silu",
    ``g sigmoid(g)``, or "gelu", ``g Phi(g)``. Returns (..., F). Sums are float32; the product is formed from them and rounded
    once. Differentiable in x and both weights (the two projections are kept for it, 6 bytes a pair for bfloat16, 8 for float32)."""
    if gate_weight.dim() != 2 or up_weight.shape != gate_weight.shape or 0 in gate_weight.shape:
        raise ValueError(f"gate_weight and up_weight must be (F, D) with F, D > 0, got {tuple(gate_weight.shape)} and {tuple(up_weight.shape)}")
    if x.dim() < 1 or x.shape[-1] != gate_weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weights {tuple(gate_weight.shape)} do not fit together")
    if not (x.dtype == gate_weight.dtype == up_weight.dtype):
        raise TypeError(f"x and the weights must share a type, got {x.dtype}, {gate_weight.dtype}, {up_weight.dtype}")
    _dtype(x, "x and the weights")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}, got {activation!r}")
    _device(x, gate_weight, up_weight)
    flat, shape = x.reshape(-1, x.shape[-1]), (*x.shape[:-1], gate_weight.shape[0])
    if torch.is_grad_enabled() and (x.requires_grad or gate_weight.requires_grad or up_weight.requires_grad):
        return _Gated.apply(flat, gate_weight, up_weight, act, shape)
    return _forward(_rows(flat), _rows(gate_weight), _rows(up_weight), act, shape, False)[0]
