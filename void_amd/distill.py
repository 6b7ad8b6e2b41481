"""Distillation from a teacher's top logits on the gfx950 kernels
(void_distill_*): how a pruned model is trained back to its dense teacher.  The
reference has no counterpart.

A row of student logits s has k teacher entries (logit t_j at vocabulary index
i_j).  With the temperature T,

    p = softmax(t / T) over the row's entries,  q = softmax(s / T) over the vocabulary,
    loss = T^2 sum_j p_j (log p_j - log q_{i_j}) = T^2 KL(p || q),
    dloss / ds_v = T (q_v - sum_{j: i_j = v} p_j).

Entries with a negative index, or a logit of -inf, do not count, so that lists
of different lengths share one tensor; a row without entries (a prompt token)
has loss 0 and gradient 0 and is left out of the mean.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, Tuple

import torch
from torch.autograd import Function

from . import _lib, _runtime
from ._streams import raw_stream

MAX_ENTRIES = 1024  # VOID_DISTILL_MAX_ENTRIES
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}


def _checked(logits: torch.Tensor, teacher: torch.Tensor, index: torch.Tensor, temperature: float):
    """The three as 2-D rows and the C arguments over them."""
    if logits.dim() == 0:
        raise ValueError("logits need a vocabulary axis")
    if teacher.shape != index.shape or teacher.dim() == 0 or teacher.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"logits {list(logits.shape)} need teacher logits and indices [..., k] of the same rows, got "
                         f"{list(teacher.shape)} and {list(index.shape)}")
    if logits.shape[-1] >= _runtime.MAX_ROW:
        raise ValueError(f"a vocabulary of {logits.shape[-1]} values is too long")
    if teacher.shape[-1] > MAX_ENTRIES:
        raise ValueError(f"at most {MAX_ENTRIES} teacher entries a row, got {teacher.shape[-1]}")
    if index.dtype not in _INDEX_BYTES:
        raise TypeError(f"teacher indices must be int32 or int64, got {index.dtype}")
    _runtime.float_code(logits, "logits")
    _runtime.float_code(teacher, "teacher logits")
    temperature = float(temperature)
    if not (0 < temperature < math.inf):
        raise ValueError(f"the temperature must be positive, got {temperature}")
    _runtime.require_gpu(logits, "logits")
    for t, what in ((teacher, "teacher logits"), (index, "teacher indices")):
        if t.device != logits.device:
            raise ValueError(f"logits on {logits.device}, {what} on {t.device}")
    s, t, i = _runtime.flat_rows(logits), _runtime.flat_rows(teacher), _runtime.flat_rows(index)
    return s, t, i, _args(s, t, i, temperature)


def _args(s: torch.Tensor, t: torch.Tensor, i: torch.Tensor, temperature: float) -> "_lib.DistillArgs":
    """The C arguments over rows of logits, teacher logits and indices."""
    R, V = s.shape
    return _lib.DistillArgs(s.data_ptr(), s.stride(0), t.data_ptr(), t.stride(0), i.data_ptr(), i.stride(0), R, V,
                            t.shape[1], _runtime.FLOAT_CODES[s.dtype], _runtime.FLOAT_CODES[t.dtype],
                            _INDEX_BYTES[i.dtype], temperature)


def _losses(args: "_lib.DistillArgs", device: torch.device):
    """(row losses, parts, used) of one call."""
    R, V = args.rows, args.vocab
    if R == 0 or V == 0:
        zero = torch.zeros(R, dtype=torch.float32, device=device)
        return zero, zero, torch.zeros(R, dtype=torch.int32, device=device)
    lib = _lib.lib()
    loss = torch.empty(R, dtype=torch.float32, device=device)
    parts = torch.empty(R, lib.void_distill_slices(R, V), 2, dtype=torch.float32, device=device)
    used = torch.empty(R, dtype=torch.int32, device=device)
    st = lib.void_distill_loss(ctypes.byref(args), loss.data_ptr(), parts.data_ptr(), used.data_ptr(),
                               raw_stream(device))
    if st:
        _lib.check(st, "void_distill_loss")
    return loss, parts, used


def _reduced(loss: torch.Tensor, used: torch.Tensor, reduction: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """The reduced loss and the factor it was multiplied by."""
    out = torch.empty((), dtype=torch.float32, device=loss.device)
    factor = torch.empty((), dtype=torch.float32, device=loss.device)
    st = _lib.lib().void_distill_reduce(loss.data_ptr(), used.data_ptr(), loss.numel(), reduction == "mean",
                                        out.data_ptr(), factor.data_ptr(), raw_stream(loss.device))
    if st:
        _lib.check(st, "void_distill_reduce")
    return out, factor


class _Distillation(Function):
    @staticmethod
    def forward(ctx: Any, logits, teacher, index, temperature, reduction):
        s, t, i, args = _checked(logits, teacher, index, temperature)
        loss, parts, used = _losses(args, s.device)
        out, factor = (loss.view(logits.shape[:-1]), None) if reduction == "none" else _reduced(loss, used, reduction)
        ctx.save_for_backward(s, t, i, parts, factor)
        ctx.temperature, ctx.shape = args.temperature, logits.shape
        return out

    @staticmethod
    @_runtime.first_order
    def backward(ctx: Any, grad: torch.Tensor):
        # What a hook or a checkpoint gives back need not lie where the forward pass had it, nor in its layout.
        s, t, i, parts, factor = ctx.saved_tensors
        s, t, i, parts = _runtime.flat_rows(s), _runtime.flat_rows(t), _runtime.flat_rows(i), parts.contiguous()
        args = _args(s, t, i, ctx.temperature)
        ds = s.new_empty(ctx.shape)
        if not ds.numel():
            return ds, None, None, None, None
        g = grad.reshape(-1).to(torch.float32)
        st = _lib.lib().void_distill_grad(ctypes.byref(args), parts.data_ptr(), g.data_ptr(),
                                          g.stride(0) if factor is None else 0,
                                          factor.data_ptr() if factor is not None else None, ds.data_ptr(), s.shape[1],
                                          raw_stream(s.device))
        if st:
            _lib.check(st, "void_distill_grad")
        return ds, None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor,
                      temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """T^2 KL(teacher's top k || student), differentiable in the student's logits.

    logits [..., V]: fp32, bf16 or fp16; teacher_logits [..., k] (any of the
    three) and teacher_indices [..., k] (int32 or int64): the teacher's entries,
    k <= 1024, in any order.  Entries with a negative index or a logit of -inf
    do not count; an index that occurs twice counts twice; an index of V or
    more makes its row's loss and gradient NaN.

    reduction: "mean" over the rows that have an entry (0 if none has), "sum",
    or "none" for a loss per row.  The loss is float32, the gradient has the
    logits' type.  No gradient flows to the teacher.
    """
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if _runtime.differentiated(logits):
        return _Distillation.apply(logits, teacher_logits, teacher_indices, temperature, reduction)
    s, _, _, args = _checked(logits, teacher_logits, teacher_indices, temperature)
    loss, _, used = _losses(args, s.device)
    return loss.view(logits.shape[:-1]) if reduction == "none" else _reduced(loss, used, reduction)[0]


@torch.no_grad()
def distillation_loss_and_grad(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor,
                               temperature: float = 1.0, reduction: str = "mean",
                               grad_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, grad_scale * dloss/dlogits) in one pass over the logits, for loops
    that go on with ``logits.backward(grad)``; the arguments are
    distillation_loss's ("mean" or "sum"), grad_scale a loss scaler's factor
    (the loss itself is not scaled)."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    s, t, i, args = _checked(logits, teacher_logits, teacher_indices, temperature)
    R, V = s.shape
    lib = _lib.lib()
    loss = torch.empty((), dtype=torch.float32, device=s.device)
    grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
    ws = torch.empty(lib.void_distill_step_workspace_bytes(R, V), dtype=torch.uint8, device=s.device)
    st = lib.void_distill_step(ctypes.byref(args), reduction == "mean", float(grad_scale), loss.data_ptr(),
                               grad.data_ptr(), V, ws.data_ptr(), ws.numel(), raw_stream(s.device))
    if st:
        _lib.check(st, "void_distill_step")
    return loss, grad


__all__ = ["distillation_loss", "distillation_loss_and_grad"]
