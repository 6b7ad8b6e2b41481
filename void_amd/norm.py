"""Layer norm on the gfx950 kernels (void_layer_norm, void_layer_norm_grad):
the norm in front of a sparse layer, differentiable.  The reference has no
counterpart.

    y = (x - mean) / sqrt(var + eps) * weight + bias      over the last axis

Statistics are fp32 whatever x's type; y and the gradients are rounded once.
"""

from __future__ import annotations

import functools
from typing import Any, Optional

import torch
from torch.autograd import Function

from . import _lib, _runtime
from ._streams import raw_stream


def _forward(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
             with_stats: bool):
    """(y, the rows x was read as, their statistics or None)."""
    rows = _runtime.flat_rows(x)
    R, C = rows.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = torch.empty(R, 2, dtype=torch.float32, device=x.device) if with_stats else None
    param = weight if weight is not None else bias
    st = _lib.lib().void_layer_norm(
        rows.data_ptr(), rows.stride(0), weight.data_ptr() if weight is not None else None,
        bias.data_ptr() if bias is not None else None, _runtime.FLOAT_CODES[x.dtype if param is None else param.dtype],
        R, C, eps, _runtime.FLOAT_CODES[x.dtype], y.data_ptr(), C, stats.data_ptr() if stats is not None else None,
        raw_stream(x.device))
    if st:
        _lib.check(st, "void_layer_norm")
    return y, rows, stats


@functools.lru_cache(maxsize=256)
def _grad_workspace_bytes(R: int, C: int, code: int) -> int:
    return _lib.lib().void_layer_norm_grad_workspace_bytes(R, C, code)


class _LayerNorm(Function):
    @staticmethod
    def forward(ctx: Any, x, weight, bias, eps):
        y, rows, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_runtime.first_order
    def backward(ctx: Any, grad: torch.Tensor):
        # What a hook or a checkpoint gives back need not lie in the layout that the forward pass saved.
        rows, weight, stats = ctx.saved_tensors
        rows, stats = _runtime.flat_rows(rows), stats.contiguous()
        weight = None if weight is None else weight.contiguous()
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        R, C = rows.shape
        dy = _runtime.flat_rows(grad)
        dx = torch.empty_like(grad, memory_format=torch.contiguous_format) if need_x else None
        param = weight if weight is not None else rows.new_empty(C, dtype=ctx.bias_dtype or rows.dtype)
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(param) if need_b else None
        code, ws, ws_bytes = _runtime.FLOAT_CODES[rows.dtype], None, 0
        if need_w or need_b:
            ws_bytes = _grad_workspace_bytes(R, C, code)
            ws = stats.new_empty(ws_bytes // 4)
        st = _lib.lib().void_layer_norm_grad(
            dy.data_ptr(), dy.stride(0), rows.data_ptr(), rows.stride(0),
            weight.data_ptr() if weight is not None else None, _runtime.FLOAT_CODES[param.dtype], stats.data_ptr(), R, C,
            code, dx.data_ptr() if need_x else None, C, dw.data_ptr() if need_w else None,
            db.data_ptr() if need_b else None, ws.data_ptr() if ws is not None else None, ws_bytes,
            raw_stream(rows.device))
        if st:
            _lib.check(st, "void_layer_norm_grad")
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of x [..., C] over its last axis.

    x is fp32, bf16 or fp16 on the GPU, of any leading shape and row pitch;
    weight and bias are [C], of x's type or fp32 (other mixes are widened to
    fp32), each optional.  The result has x's type and shape.  Gradients of x,
    weight and bias come from one pass over x and the gradient; they are not
    differentiable themselves.
    """
    if x.dim() == 0:
        raise ValueError("layer_norm needs at least one axis")
    _runtime.float_code(x, "x")
    C = x.shape[-1]
    if C >= _runtime.MAX_ROW:
        raise ValueError(f"rows of {C} values are too long")
    for p, what in ((weight, "weight"), (bias, "bias")):
        if p is None:
            continue
        if p.shape != (C,):
            raise ValueError(f"{what} must be [{C}], got {list(p.shape)}")
        _runtime.float_code(p, what)
        if p.device != x.device:
            raise ValueError(f"x on {x.device}, {what} on {p.device}")
    _runtime.require_gpu(x, "x")
    wide = torch.float32
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.to(wide), bias.to(wide)
    if weight is not None:
        weight = (weight if weight.dtype in (x.dtype, wide) else weight.to(wide)).contiguous()
    if bias is not None:
        bias = (bias if bias.dtype in (x.dtype, wide) else bias.to(wide)).contiguous()
    if _runtime.differentiated(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


class LayerNorm(torch.nn.Module):
    """layer_norm over the last axis with a trainable weight (ones) and bias (zeros)."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True, dtype: Optional[torch.dtype] = None,
                 device=None):
        super().__init__()
        self.features, self.eps = features, eps
        self.weight = torch.nn.Parameter(torch.ones(features, dtype=dtype, device=device))
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(features, dtype=dtype, device=device))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}, bias={self.bias is not None}"


__all__ = ["layer_norm", "LayerNorm"]
