"""Token operators beside the EWS engines: what a token model needs in front of, between and behind the blocks.

``token_embedding`` (scaled lookup, gradient by sorted tokens), ``decayed_attention`` (linear attention with a decay
per head, over prompts and in training) with ``decayed_attention_step`` (one token per row on a pool of states), and
``vocab_loss`` (softmax cross entropy over a large vocabulary whose logits are never kept). All run on the caller's
current stream through the C ABI, on float32 or bfloat16 CUDA tensors; states, sums, softmax statistics and losses
are float32. There is no CPU fallback. Indices out of range do not stop the GPU: the entry counts as absent and the
next token operator on the device raises IndexError (at once under ``configure(check_status=True)``).
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib, engine
from .engine import _ptr, _require_cuda, _stream_ptr, _timed

_DTYPES = {torch.float32: _lib.EWS_DTYPE_F32, torch.bfloat16: _lib.EWS_DTYPE_BF16}
MAX_HEAD = 128


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return code


def _indices(t: torch.Tensor, what: str) -> int:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what} must be int64 or int32, got {t.dtype}")
    return 1 if t.dtype == torch.int64 else 0


def _same_device(*tensors) -> torch.device:
    _require_cuda(*tensors)
    dev = tensors[0].device
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}")
    return dev


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-d tensor whose rows are contiguous and do not overlap (a view where it already is one)."""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _after(dev) -> None:
    if engine.CHECK_SYNC:
        torch.cuda.current_stream(dev).synchronize()
        engine.raise_index(dev)


# ----------------------------------------------------------------------------------------- token embedding


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_index):
        lib = _lib.load()
        dev = table.device
        code, wide = _DTYPES[table.dtype], _indices(ids, "ids")
        flat, rows = ids.reshape(-1), _rows(table)
        flat = flat.contiguous()
        n, (vocab, dim) = flat.numel(), table.shape
        out = torch.empty((*ids.shape, dim), dtype=table.dtype, device=dev)
        with torch.cuda.device(dev), _timed("ews_embed_fwd", dev, n, 1):
            _lib.check(lib.ews_embed_fwd(_ptr(flat), wide, _ptr(rows), code, n, vocab, dim, _row_stride(rows), scale,
                                         _ptr(out), engine.index_word(dev)[0], _stream_ptr(dev)), "ews_embed_fwd")
        ctx.meta = (code, wide, vocab, dim, scale, padding_index)
        ctx.save_for_backward(flat)
        _after(dev)
        return out

    @staticmethod
    def backward(ctx, dout):
        code, wide, vocab, dim, scale, padding_index = ctx.meta
        (flat,) = ctx.saved_tensors
        lib = _lib.load()
        dev = dout.device
        n = flat.numel()
        g = _rows(dout.reshape(n, dim))
        grad = torch.empty((vocab, dim), dtype=dout.dtype, device=dev)
        work = torch.empty(int(lib.ews_embed_work_size(n, vocab, dim)), dtype=torch.uint8, device=dev)
        skip = -1 if padding_index is None else padding_index
        with torch.cuda.device(dev), _timed("ews_embed_bwd", dev, n, 3):
            _lib.check(lib.ews_embed_bwd(_ptr(flat), wide, _ptr(g), code, n, vocab, dim, _row_stride(g), scale, skip,
                                         _ptr(grad), _ptr(work), work.numel(), None, _stream_ptr(dev)), "ews_embed_bwd")
        return None, grad, None, None


def token_embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
                    padding_index: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]``: ids of any shape (int64 or int32), table (V, D) -> (*ids.shape, D).

    Differentiable in the table. The gradient is the float32 sum of each token's rows in the order of their
    positions, rounded once and bit-reproducible; rows of ``padding_index`` (their token is looked up as any
    other) and of tokens that do not occur are zero. An id out of range gives a zero row and IndexError on the next
    call."""
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"table must be (V, D) with V, D > 0, got {tuple(table.shape)}")
    _dtype(table, "table")
    _indices(ids, "ids")
    dev = _same_device(table, ids)
    if padding_index is not None:
        if not -table.shape[0] <= padding_index < table.shape[0]:
            raise ValueError(f"padding_index {padding_index} is out of range for {table.shape[0]} rows")
        padding_index %= table.shape[0]
    engine.raise_index(dev)
    return _Embedding.apply(ids, table, float(scale), padding_index)


# ---------------------------------------------------------------------------------------- decayed attention


def _strides(t: torch.Tensor):
    return (ctypes.c_int64 * 3)(*t.stride()[:3])


def _last_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


class _Decayed(torch.autograd.Function):
    @staticmethod
    def _args(q, k, v, rate, lengths, scale):
        a = _lib.DecayArgs()
        a.batch, a.steps, a.heads, a.dk = q.shape
        a.kv_heads, a.dv = k.shape[2], v.shape[3]
        a.dtype, a.scale = _DTYPES[q.dtype], scale
        a.q, a.k, a.v = _ptr(q), _ptr(k), _ptr(v)
        a.q_stride, a.k_stride, a.v_stride = _strides(q), _strides(k), _strides(v)
        a.rate, a.lengths = _ptr(rate), _ptr(lengths)
        a.status = engine.index_word(q.device)[0]
        return a

    @staticmethod
    def forward(ctx, q, k, v, rate, initial, lengths, scale, want_state):
        lib = _lib.load()
        dev = q.device
        q, k, v = (_last_contiguous(t) for t in (q, k, v))
        B, T, H, dk = q.shape
        dv = v.shape[3]
        a = _Decayed._args(q, k, v, rate, lengths, scale)
        out = torch.empty((B, T, H, dv), dtype=q.dtype, device=dev)
        end = torch.empty((B, H, dk, dv), dtype=torch.float32, device=dev) if want_state else None
        a.initial, a.out, a.final_state = _ptr(initial), _ptr(out), _ptr(end)
        size = lib.ews_decay_work_size(ctypes.byref(a), 0)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        a.work, a.work_bytes = _ptr(work), size
        with torch.cuda.device(dev), _timed("ews_decay_fwd", dev, B * T):
            _lib.check(lib.ews_decay_fwd(ctypes.byref(a), _stream_ptr(dev)), "ews_decay_fwd")
        _after(dev)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, rate, initial, lengths)
        ctx.set_materialize_grads(False)
        return out, end

    @staticmethod
    def backward(ctx, dout, dend):
        q, k, v, rate, initial, lengths = ctx.saved_tensors
        lib = _lib.load()
        dev = q.device
        B, T, H, dk = q.shape
        dv = v.shape[3]
        dout = torch.zeros((B, T, H, dv), dtype=q.dtype, device=dev) if dout is None else _last_contiguous(dout)
        dend = None if dend is None else dend.contiguous()
        a = _Decayed._args(q, k, v, rate, lengths, ctx.scale)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v)]
        d0 = torch.empty((B, H, dk, dv), dtype=torch.float32, device=dev) if ctx.needs_input_grad[4] else None
        a.initial, a.dout, a.dout_stride, a.dfinal = _ptr(initial), _ptr(dout), _strides(dout), _ptr(dend)
        a.dq, a.dk_out, a.dv_out = (_ptr(g) for g in grads)
        a.dinitial = _ptr(d0)
        size = lib.ews_decay_work_size(ctypes.byref(a), 1)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        a.work, a.work_bytes = _ptr(work), size
        with torch.cuda.device(dev), _timed("ews_decay_bwd", dev, B * T):
            _lib.check(lib.ews_decay_bwd(ctypes.byref(a), _stream_ptr(dev)), "ews_decay_bwd")
        _after(dev)
        return (*grads, None, d0, None, None, None)


def _check_heads(q, k, v, rate, axes):
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k and v must share a type, got {q.dtype}, {k.dtype}, {v.dtype}")
    _dtype(q, "q, k and v")
    if q.dim() != axes or k.dim() != axes or v.dim() != axes:
        raise ValueError(f"q, k and v must have {axes} axes, got {q.dim()}, {k.dim()}, {v.dim()}")
    H, dk, Hk, dv = q.shape[-2], q.shape[-1], k.shape[-2], v.shape[-1]
    if k.shape != (*q.shape[:-2], Hk, dk) or v.shape != (*q.shape[:-2], Hk, dv):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    if Hk == 0 or H == 0 or H % Hk:
        raise ValueError(f"{H} query heads cannot share {Hk} key/value heads")
    if not (1 <= dk <= MAX_HEAD and 1 <= dv <= MAX_HEAD):
        raise NotImplementedError(f"head widths are 1 to {MAX_HEAD}, got {dk} and {dv}")
    if rate.shape != (H,) or rate.dtype != torch.float32 or not rate.is_contiguous():
        raise ValueError(f"rate must be a contiguous float32 tensor of {H} values, got {rate.dtype} {tuple(rate.shape)}")
    if rate.requires_grad:
        raise NotImplementedError("the rates are constants of the heads: no gradient is built for them")
    return H, dk, dv


def _scale(scale, dk):
    scale = dk**-0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or scale == 0.0:
        raise ValueError(f"scale must be finite and not zero, got {scale}")
    return scale


def decayed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rate: torch.Tensor, *,
                      scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                      lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """Linear attention with a decay per head: ``S_t = exp(-rate_h) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t``.

    q (B, T, H, dk), k (B, T, Hk, dk), v (B, T, Hk, dv), float32 or bfloat16, any strides (head h reads key/value
    head ``h // (H / Hk)``); dk, dv <= 128. rate (H,) float32, the heads' constants (exp(-rate) is the decay of one
    token, as an EWS generator's flow over a unit step). initial_state (B, H, dk, dv) float32 or None (zero).
    lengths (B,) int32: positions at or beyond a sample's length are not read, give zeros and leave the state.
    scale: default dk^-1/2.

    Returns o (B, T, H, dv), with ``return_state`` also the state after the last token (B, H, dk, dv) float32, for
    ``decayed_attention_step`` or the next piece of a long sequence. Differentiable in q, k, v and initial_state."""
    _, dk, dv = H_dk_dv = _check_heads(q, k, v, rate, 4)
    B, H = q.shape[0], H_dk_dv[0]
    if initial_state is not None:
        if initial_state.shape != (B, H, dk, dv) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state must be float32 {(B, H, dk, dv)}, got {initial_state.dtype} {tuple(initial_state.shape)}")
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.dtype != torch.int32:
            raise ValueError(f"lengths must be int32 ({B},), got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    engine.raise_index(_same_device(q, k, v, rate, initial_state, lengths))
    out, end = _Decayed.apply(q, k, v, rate, initial_state, lengths, _scale(scale, dk), bool(return_state))
    return (out, end) if return_state else out


def decayed_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rate: torch.Tensor, state: torch.Tensor, *,
                           scale: Optional[float] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token per row of ``decayed_attention`` on a pool of states, updated in place.

    q (B, H, dk), k (B, Hk, dk), v (B, Hk, dv); state (P, H, dk, dv) float32, contiguous. Row b works on state
    ``slots[b]`` (int32 (B,); None: b, with P >= B). A negative slot is a row without a request: its output is zero and
    no state is touched. Two rows must not share a slot; one out of range gives a zero row and IndexError on the
    next call. Returns o (B, H, dv). For serving: no gradient."""
    H, dk, dv = _check_heads(q, k, v, rate, 3)
    B = q.shape[0]
    if state.dim() != 4 or state.shape[1:] != (H, dk, dv) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32 (P, {H}, {dk}, {dv}), got {state.dtype} {tuple(state.shape)}")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError(f"{B} rows need as many states or slots, got {state.shape[0]} states")
    elif slots.shape != (B,) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError(f"slots must be contiguous int32 ({B},), got {slots.dtype} {tuple(slots.shape)}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError("decayed_attention_step has no gradient: call it under torch.no_grad()")
    dev = _same_device(q, k, v, rate, state, slots)
    engine.raise_index(dev)
    q, k, v = (_last_contiguous(t) for t in (q, k, v))
    out = torch.empty((B, H, dv), dtype=q.dtype, device=dev)
    a = _lib.DecayArgs()
    a.batch, a.steps, a.heads, a.kv_heads, a.dk, a.dv = B, 1, H, k.shape[1], dk, dv
    a.dtype, a.scale = _DTYPES[q.dtype], _scale(scale, dk)
    a.q, a.k, a.v, a.rate, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), rate.data_ptr(), out.data_ptr()
    a.status = engine.index_word(dev)[0]
    (a.q_stride[0], a.q_stride[2], _), (a.k_stride[0], a.k_stride[2], _), (a.v_stride[0], a.v_stride[2], _) = (
        q.stride(), k.stride(), v.stride())
    with torch.cuda.device(dev), _timed("ews_decay_step", dev, B, 1):
        _lib.check(_lib.load().ews_decay_step(ctypes.byref(a), _ptr(slots), state.shape[0], _ptr(state),
                                              _stream_ptr(dev)), "ews_decay_step")
    _after(dev)
    return out


# --------------------------------------------------------------------------------------------- vocabulary loss


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def _args(hidden, weight, targets, ignore):
        a = _lib.VocabArgs()
        a.rows, a.dim = hidden.shape
        a.vocab = weight.shape[0]
        a.dtype, a.targets_wide = _DTYPES[hidden.dtype], _indices(targets, "targets")
        a.hidden, a.weight, a.targets = _ptr(hidden), _ptr(weight), _ptr(targets)
        a.hidden_stride, a.weight_stride, a.ignore = _row_stride(hidden), _row_stride(weight), ignore
        return a

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore):
        lib = _lib.load()
        dev = hidden.device
        hidden, weight, targets = _rows(hidden), _rows(weight), targets.contiguous()
        a = _VocabLoss._args(hidden, weight, targets, ignore)
        loss = torch.empty(a.rows, dtype=torch.float32, device=dev)
        lse = torch.empty(a.rows, dtype=torch.float32, device=dev)
        size = int(lib.ews_vocab_work_size(ctypes.byref(a), 0))
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        a.loss, a.lse, a.work, a.work_bytes = _ptr(loss), _ptr(lse), _ptr(work), size
        a.status = engine.index_word(dev)[0]
        with torch.cuda.device(dev), _timed("ews_vocab_fwd", dev, a.rows):
            _lib.check(lib.ews_vocab_fwd(ctypes.byref(a), _stream_ptr(dev)), "ews_vocab_fwd")
        ctx.ignore = ignore
        ctx.save_for_backward(hidden, weight, targets, lse)
        _after(dev)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        hidden, weight, targets, lse = ctx.saved_tensors
        lib = _lib.load()
        dev = hidden.device
        dloss = dloss.contiguous()
        a = _VocabLoss._args(hidden, weight, targets, ctx.ignore)
        dh, dw = (torch.empty(t.shape, dtype=t.dtype, device=dev) if need else None
                  for t, need in ((hidden, ctx.needs_input_grad[0]), (weight, ctx.needs_input_grad[1])))
        size = int(lib.ews_vocab_work_size(ctypes.byref(a), 1))
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        a.lse, a.dloss, a.dhidden, a.dweight = _ptr(lse), _ptr(dloss), _ptr(dh), _ptr(dw)
        a.work, a.work_bytes = _ptr(work), size
        a.status = engine.index_word(dev)[0]
        with torch.cuda.device(dev), _timed("ews_vocab_bwd", dev, a.rows):
            _lib.check(lib.ews_vocab_bwd(ctypes.byref(a), _stream_ptr(dev)), "ews_vocab_bwd")
        _after(dev)
        return dh, dw, None, None


def vocab_loss(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100) -> torch.Tensor:
    """Softmax cross entropy of ``hidden @ weight.T`` against ``targets``, per position, in float32.

    hidden (..., D) and weight (V, D), both float32 or both bfloat16; targets (...) int64 or int32. Positions whose
    target is ``ignore_index`` have loss 0, no gradient, and their hidden rows do not enter the others'. Returns the
    losses with the shape of ``targets``; the logits (N, V) are formed in tiles and pieces and never kept.
    Differentiable in hidden and weight. A target out of range counts as ignored and raises IndexError on the next
    call."""
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not fit together")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden and weight must share a type, got {hidden.dtype} and {weight.dtype}")
    _dtype(hidden, "hidden and weight")
    _indices(targets, "targets")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} must have the shape {tuple(hidden.shape[:-1])}")
    dev = _same_device(hidden, weight, targets)
    engine.raise_index(dev)
    loss = _VocabLoss.apply(hidden.reshape(-1, hidden.shape[-1]), weight, targets.reshape(-1), int(ignore_index))
    return loss.reshape(targets.shape)
