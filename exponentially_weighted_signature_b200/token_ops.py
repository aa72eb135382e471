"""Token operators beside the EWS engines: what a token model needs in front of, between and behind the blocks.

``token_embedding`` (scaled lookup, gradient by sorted tokens), ``decayed_attention`` (linear attention with a decay
per head, over prompts and in training) with ``decayed_attention_step`` (one token per row on a pool of states), and
``vocab_loss`` (softmax cross entropy over a large vocabulary whose logits are never kept). All run on the caller's
current stream through the C ABI, on float32 or bfloat16 CUDA tensors; states, sums, softmax statistics and losses
are float32. There is no CPU fallback. Derivatives are reverse-mode and first-order: a dual tensor is refused, and so
is differentiating a gradient again. Indices out of range do not stop the GPU: the entry counts as absent and the next
token operator on the device raises IndexError (at once under ``configure(check_status=True)``).
"""

from __future__ import annotations

import functools
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib, engine
from .engine import _require_cuda, _timed, first_order

_DTYPES = {torch.float32: _lib.EWS_DTYPE_F32, torch.bfloat16: _lib.EWS_DTYPE_BF16}
_WIDE = {torch.int64: 1, torch.int32: 0}
MAX_HEAD = 128

# ews_decay_args and ews_vocab_args, packed in one call (native alignment; the fields in the header's order).
_DECAY = struct.Struct("@7if3P9q6P3q6PNP").pack
_VOCAB = struct.Struct("@3q2i3P3q7PNP").pack

_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without building a Stream


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return code


def _wide(t: torch.Tensor, what: str) -> int:
    wide = _WIDE.get(t.dtype)
    if wide is None:
        raise TypeError(f"{what} must be int64 or int32, got {t.dtype}")
    return wide


def _device(*tensors) -> int:
    """The index of the one CUDA device that all tensors are on, pending index errors on it raised. Dual tensors are
    refused: where no input requires a gradient no autograd function runs, and a tangent would vanish unseen."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the token operators have no forward-mode derivative")
    idx = tensors[0].get_device()
    for t in tensors:
        if t is not None and (idx < 0 or t.get_device() != idx):
            _require_cuda(*tensors)
            raise ValueError(f"all tensors must be on one device, got {tensors[0].device} and {t.device}")
    if engine.index_word(idx)[1].value:
        engine.raise_index(idx)
    return idx


def _launch(idx: int, name: str, units: int, fn, *args) -> None:
    """One library call on the device's current stream."""
    if engine.PROFILE is None and idx == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx), _timed(name, torch.device("cuda", idx), units):
            rc = fn(*args, _raw_stream(idx))
    if rc:
        _lib.check(rc, name)
    if engine.CHECK_SYNC:
        torch.cuda.current_stream(idx).synchronize()
        engine.raise_index(idx)


def _work(size: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


@functools.lru_cache(maxsize=256)
def _embed_size(n: int, vocab: int, dim: int) -> int:
    """Workspace bytes are a function of the sizes alone, so each set of sizes asks the library once."""
    return _lib.load().ews_embed_work_size(n, vocab, dim)


@functools.lru_cache(maxsize=256)
def _decay_size(B: int, T: int, H: int, Hk: int, dk: int, dv: int, code: int, backward: int) -> int:
    args = _DECAY(B, T, H, Hk, dk, dv, code, 1.0, *([0] * 27), 0, 0)
    return _lib.load().ews_decay_work_size(args, backward)


@functools.lru_cache(maxsize=256)
def _vocab_size(rows: int, vocab: int, dim: int, code: int, hidden_stride: int, weight_stride: int, weight_at: int, backward: int) -> int:
    """weight_at: the weight's address modulo 16."""
    args = _VOCAB(rows, vocab, dim, code, 1, 0, weight_at, 0, hidden_stride, weight_stride, 0, *([0] * 7), 0, 0)
    return _lib.load().ews_vocab_work_size(args, backward)


def _addr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-d tensor whose rows are contiguous and do not overlap (a view where it already is one)."""
    if t.is_contiguous():
        return t
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# ----------------------------------------------------------------------------------------- token embedding


def _embed(flat, table, scale, shape):
    idx, (vocab, dim), n = table.get_device(), table.shape, flat.numel()
    out = torch.empty((*shape, dim), dtype=table.dtype, device=table.device)
    _launch(idx, "ews_embed_fwd", n, _lib.load().ews_embed_fwd, flat.data_ptr(), _WIDE[flat.dtype], table.data_ptr(),
            _DTYPES[table.dtype], n, vocab, dim, _row_stride(table), scale, out.data_ptr(), engine.index_word(idx)[0])
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, flat, table, scale, padding_index, shape):
        rows = _rows(table)
        ctx.meta = (rows.shape, scale, padding_index)
        ctx.save_for_backward(flat)
        return _embed(flat, rows, scale, shape)

    @staticmethod
    @first_order
    def backward(ctx, dout):
        (vocab, dim), scale, padding_index = ctx.meta
        (flat,) = ctx.saved_tensors
        lib = _lib.load()
        n = flat.numel()
        g = _rows(dout.reshape(n, dim))
        grad = torch.empty((vocab, dim), dtype=dout.dtype, device=dout.device)
        work = _work(_embed_size(n, vocab, dim), dout)
        _launch(dout.get_device(), "ews_embed_bwd", n, lib.ews_embed_bwd, flat.data_ptr(), _WIDE[flat.dtype], g.data_ptr(),
                _DTYPES[dout.dtype], n, vocab, dim, _row_stride(g), scale, padding_index, grad.data_ptr(), _addr(work),
                0 if work is None else work.numel(), None)
        return None, grad, None, None, None


def token_embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
                    padding_index: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]``: ids of any shape (int64 or int32), table (V, D) -> (*ids.shape, D).

    Differentiable in the table. The gradient is the float32 sum of each token's rows in the order of their
    positions, rounded once and bit-reproducible; rows of ``padding_index`` (their token is looked up as any
    other) and of tokens that do not occur are zero. An id out of range gives a zero row and IndexError on the next
    call."""
    if table.dim() != 2 or 0 in table.shape:
        raise ValueError(f"table must be (V, D) with V, D > 0, got {tuple(table.shape)}")
    _dtype(table, "table")
    _wide(ids, "ids")
    if padding_index is not None and not -table.shape[0] <= padding_index < table.shape[0]:
        raise ValueError(f"padding_index {padding_index} is out of range for {table.shape[0]} rows")
    _device(table, ids)
    flat = ids.reshape(-1).contiguous()
    if table.requires_grad and torch.is_grad_enabled():
        skip = -1 if padding_index is None else padding_index % table.shape[0]
        return _Embedding.apply(flat, table, float(scale), skip, ids.shape)
    return _embed(flat, _rows(table.detach()), float(scale), ids.shape)


# ---------------------------------------------------------------------------------------- decayed attention


def _last_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _decay_args(q, k, v, rate, lengths, initial, scale, out=None, end=None, dout=None, dend=None, grads=(None, None, None),
                d0=None, work=None):
    B, T, H, dk = q.shape
    return _DECAY(B, T, H, k.shape[2], dk, v.shape[3], _DTYPES[q.dtype], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], rate.data_ptr(), _addr(lengths), _addr(initial),
                  _addr(out), _addr(end), _addr(dout), *((0, 0, 0) if dout is None else dout.stride()[:3]), _addr(dend),
                  _addr(grads[0]), _addr(grads[1]), _addr(grads[2]), _addr(d0), _addr(work), 0 if work is None else work.numel(),
                  engine.index_word(q.get_device())[0])


def _decayed(q, k, v, rate, initial, lengths, scale, want_state):
    lib = _lib.load()
    B, T, H, dk = q.shape
    dv = v.shape[3]
    out = torch.empty((B, T, H, dv), dtype=q.dtype, device=q.device)
    end = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device) if want_state else None
    work = _work(_decay_size(B, T, H, k.shape[2], dk, dv, _DTYPES[q.dtype], 0), q)
    args = _decay_args(q, k, v, rate, lengths, initial, scale, out, end, work=work)
    _launch(q.get_device(), "ews_decay_fwd", B * T, lib.ews_decay_fwd, args)
    return out, end


class _Decayed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, rate, initial, lengths, scale, want_state):
        q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, rate, initial, lengths)
        ctx.set_materialize_grads(False)
        return _decayed(q, k, v, rate, initial, lengths, scale, want_state)

    @staticmethod
    @first_order
    def backward(ctx, dout, dend):
        q, k, v, rate, initial, lengths = ctx.saved_tensors
        lib = _lib.load()
        B, T, H, dk = q.shape
        dv = v.shape[3]
        dout = torch.zeros((B, T, H, dv), dtype=q.dtype, device=q.device) if dout is None else _last_contiguous(dout)
        dend = None if dend is None else dend.contiguous()
        grads = [torch.empty(t.shape, dtype=t.dtype, device=q.device) for t in (q, k, v)]
        d0 = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device) if ctx.needs_input_grad[4] else None
        work = _work(_decay_size(B, T, H, k.shape[2], dk, dv, _DTYPES[q.dtype], 1), q)
        args = _decay_args(q, k, v, rate, lengths, initial, ctx.scale, None, None, dout, dend, grads, d0, work)
        _launch(q.get_device(), "ews_decay_bwd", B * T, lib.ews_decay_bwd, args)
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
    if rate.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("the rates are constants of the heads: no gradient is built for them")
    return H, dk, dv


def _scale(scale, dk):
    scale = dk**-0.5 if scale is None else float(scale)
    if not 2.0**-126 <= abs(scale) < 2.0**128 - 2.0**103:  # the kernels take it, and 1 / scale, in float32
        raise ValueError(f"scale must be finite, not zero and within float32's normal range, got {scale}")
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
    H, dk, dv = _check_heads(q, k, v, rate, 4)
    B = q.shape[0]
    if initial_state is not None:
        if initial_state.shape != (B, H, dk, dv) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state must be float32 {(B, H, dk, dv)}, got {initial_state.dtype} {tuple(initial_state.shape)}")
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.dtype != torch.int32:
            raise ValueError(f"lengths must be int32 ({B},), got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    _device(q, k, v, rate, initial_state, lengths)
    scale, want = _scale(scale, dk), bool(return_state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or initial_state is not None and initial_state.requires_grad):
        out, end = _Decayed.apply(q, k, v, rate, initial_state, lengths, scale, want)
    else:
        q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
        out, end = _decayed(q, k, v, rate, initial_state, lengths, scale, want)
    return (out, end) if want else out


def decayed_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rate: torch.Tensor, state: torch.Tensor, *,
                           scale: Optional[float] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token per row of ``decayed_attention`` on a pool of states, updated in place.

    q (B, H, dk), k (B, Hk, dk), v (B, Hk, dv); state (P, H, dk, dv) float32, contiguous. Row b works on state
    ``slots[b]`` (int32 (B,); None: b, with P >= B). A negative slot is a row without a request: its output is zero and
    no state is touched. Two rows must not share a slot; one out of range gives a zero row and IndexError on the
    next call. Returns o (B, H, dv). For serving: no gradient; a backward that needs the states as they were raises, as
    after any operation in place."""
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
    idx = _device(q, k, v, rate, state, slots)
    q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
    out = torch.empty((B, H, dv), dtype=q.dtype, device=q.device)
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    args = _DECAY(B, 1, H, k.shape[1], dk, dv, _DTYPES[q.dtype], _scale(scale, dk), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  qb, 0, qh, kb, 0, kh, vb, 0, vh, rate.data_ptr(), 0, 0, out.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                  engine.index_word(idx)[0])
    _launch(idx, "ews_decay_step", B, _lib.load().ews_decay_step, args, _addr(slots), state.shape[0], state.data_ptr())
    if not state.is_inference():  # autograd cannot see the write: a backward that saved these states must
        torch.autograd.graph.increment_version(state)
    return out


# --------------------------------------------------------------------------------------------- vocabulary loss


def _vocab_args(hidden, weight, targets, ignore, loss=None, lse=None, plan=None, dloss=None, dh=None, dw=None, work=None):
    rows, dim = hidden.shape
    return _VOCAB(rows, weight.shape[0], dim, _DTYPES[hidden.dtype], _WIDE[targets.dtype], hidden.data_ptr(), weight.data_ptr(),
                  targets.data_ptr(), _row_stride(hidden), _row_stride(weight), ignore, _addr(loss), _addr(lse), _addr(plan),
                  _addr(dloss), _addr(dh), _addr(dw), _addr(work), 0 if work is None else work.numel(), engine.index_word(hidden.get_device())[0])


def _vocab_work(hidden, weight, backward):
    return _work(_vocab_size(*hidden.shape[:1], *weight.shape, _DTYPES[hidden.dtype], _row_stride(hidden), _row_stride(weight),
                             weight.data_ptr() % 16, backward), hidden)


def _vocab(hidden, weight, targets, ignore, shape):
    lib = _lib.load()
    rows = hidden.shape[0]
    # of its own memory and shape: a loss that is a view cannot be changed in place by the caller
    loss = torch.empty(shape, dtype=torch.float32, device=hidden.device)
    lse = torch.empty(rows, dtype=torch.float32, device=hidden.device)
    work = _vocab_work(hidden, weight, 0)
    plan = torch.empty(3 * rows + 4, dtype=torch.int32, device=hidden.device)
    args = _vocab_args(hidden, weight, targets, ignore, loss, lse, plan, work=work)
    _launch(hidden.get_device(), "ews_vocab_fwd", rows, lib.ews_vocab_fwd, args)
    return loss, lse, plan


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore, shape):
        hidden, weight = _rows(hidden), _rows(weight)
        loss, lse, plan = _vocab(hidden, weight, targets, ignore, shape)
        ctx.ignore = ignore
        ctx.save_for_backward(hidden, weight, targets, lse, plan)
        return loss

    @staticmethod
    @first_order
    def backward(ctx, dloss):
        hidden, weight, targets, lse, plan = ctx.saved_tensors
        lib = _lib.load()
        dloss = dloss.contiguous()
        dh, dw = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None
                  for t, need in ((hidden, ctx.needs_input_grad[0]), (weight, ctx.needs_input_grad[1])))
        work = _vocab_work(hidden, weight, 1)
        args = _vocab_args(hidden, weight, targets, ctx.ignore, None, lse, plan, dloss, dh, dw, work)
        _launch(hidden.get_device(), "ews_vocab_bwd", hidden.shape[0], lib.ews_vocab_bwd, args)
        return dh, dw, None, None, None


def vocab_loss(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100) -> torch.Tensor:
    """Softmax cross entropy of ``hidden @ weight.T`` against ``targets``, per position, in float32.

    hidden (..., D) and weight (V, D), both float32 or both bfloat16; targets (...) int64 or int32. Positions whose
    target is ``ignore_index`` have loss 0 and no gradient, and cost nothing (only the other rows are computed). Returns the
    losses with the shape of ``targets``; the logits (N, V) are formed in tiles and pieces and never kept.
    Differentiable in hidden and weight. A target out of range counts as ignored and raises IndexError on the next
    call."""
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not fit together")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden and weight must share a type, got {hidden.dtype} and {weight.dtype}")
    _dtype(hidden, "hidden and weight")
    _wide(targets, "targets")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} must have the shape {tuple(hidden.shape[:-1])}")
    _device(hidden, weight, targets)
    flat, t = hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1).contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _VocabLoss.apply(flat, weight, t, int(ignore_index), targets.shape)
    return _vocab(_rows(flat), _rows(weight), t, int(ignore_index), targets.shape)[0]
