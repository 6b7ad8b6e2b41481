"""The dense layer with its epilogue on the gfx950 kernels (void_linear*): the
layers that pruning leaves dense, and the residual stream that a block's last
product is added to.  The reference has this epilogue on its sparse products
only (void/fusion.py:98-304), without the residual and without gradients.

    Z = x W^T + bias,   Y = activation(Z) + residual
    dZ = dY activation'(Z),   dx = dZ W,   dW = dZ^T x,   dbias = sum of dZ's rows

Products are summed in fp32 and Y is rounded once.  The forward pass keeps
activation'(Z) for the backward pass (fp32, or 2 bytes a value for 16-bit
inputs: within 2^-16, and from 2^-29 on within 2^-10 of itself); dZ is rounded
to the inputs' type, which the matrix cores take.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, Optional, Union

import torch
from torch.autograd import Function

from . import _lib, _runtime
from ._streams import raw_stream
from .fusion import _CODES, ActivationType, get_activation_code


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _whole(cols: int, t: torch.Tensor) -> int:
    """cols rounded up to whole 16-byte chunks of t's type."""
    per = 16 // t.element_size()
    return -(-cols // per) * per


_REACH = (1 << 31) - 1 - (1 << 16)  # bytes that 256 rows of the tiles' operands may span


def _far(t: torch.Tensor) -> bool:
    """Whether the rows of t (2-D) lie further apart than the tiles' 31-bit offsets reach."""
    R = t.shape[0]
    return R > 1 and min(R, 256) * t.stride(0) * t.element_size() > _REACH


def _padded(t: torch.Tensor, zero_tail: bool = False) -> torch.Tensor:
    """_runtime.padded_rows, copied too where the rows lie too far apart and a copy's do not."""
    rows = _runtime.padded_rows(t, zero_tail=zero_tail)
    if rows is t and t.numel() and _far(t) and t.stride(0) > _whole(t.shape[1], t):
        return _runtime.padded_copy(t, _whole(t.shape[1], t))
    return rows


def _chunked(t: torch.Tensor) -> torch.Tensor:
    """t with rows that can be read to the end of their last 16-byte chunk, whatever lies there."""
    rows = _padded(t)
    end = rows.storage_offset() + (rows.shape[0] - 1) * rows.stride(0) + _whole(rows.shape[1], rows)
    if rows is t and end * t.element_size() > t.untyped_storage().nbytes():
        return _padded(t, zero_tail=True)  # the storage ends inside the last row's last chunk
    return rows


def _forward(x, weight, bias, residual, code: int, with_slope: bool):
    """(y, x and weight as the kernel read them, activation'(Z) or None)."""
    lib = _lib.lib()
    N, K = weight.shape
    rows = x.reshape(math.prod(x.shape[:-1]), K)
    M = rows.shape[0]
    if lib.void_linear_any_alignment(M):
        rows = _runtime.flat_rows(rows)
        # Few rows far apart are copied for the tiles; a weight's stay, which few_kernel reads.
        if M > 1 and (rows.stride(0) < K or _far(rows)):
            rows = rows.contiguous()
        w = weight if weight.stride(1) == 1 and weight.stride(0) >= K else weight.contiguous()
        depth = K
    else:
        rows, w = _padded(rows, zero_tail=True), _padded(weight, zero_tail=True)
        depth = _whole(K, x)
    y = x.new_empty(x.shape[:-1] + (N,))
    slope = None
    if with_slope:
        slope = torch.empty(M, N, dtype=torch.float32 if x.dtype == torch.float32 else torch.int16, device=x.device)
    if not y.numel():
        return y, rows, w, slope
    if residual is not None:
        residual = _runtime.flat_rows(residual)
    dtype = _runtime.FLOAT_CODES[x.dtype]
    ws = _workspace(lib.void_linear_workspace_bytes(M, N, depth, dtype), x.device)
    args = _lib.LinearArgs(rows.data_ptr(), rows.stride(0), w.data_ptr(), w.stride(0), _ptr(bias), _ptr(residual),
                           0 if residual is None else residual.stride(0), y.data_ptr(), N, _ptr(slope), _ptr(ws),
                           0 if ws is None else ws.numel(), M, N, depth, dtype,
                           dtype if bias is None else _runtime.FLOAT_CODES[bias.dtype], code, 0)
    st = lib.void_linear(ctypes.byref(args), raw_stream(x.device))
    if st:
        _lib.check(st, "void_linear")
    return y, rows, w, slope


def _product(entry: str, a, b, M: int, N: int, K: int, out: torch.Tensor) -> torch.Tensor:
    """void_linear_grad_x / _grad_w of dZ [M, N] with W or X into out."""
    lib = _lib.lib()
    depth = N if entry == "void_linear_grad_x" else M
    code = _runtime.FLOAT_CODES[out.dtype]
    ws = _workspace(lib.void_linear_grad_workspace_bytes(out.shape[0], out.shape[1], depth, code), out.device)
    st = getattr(lib, entry)(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), M, N, K, code, out.data_ptr(), K,
                             _ptr(ws), 0 if ws is None else ws.numel(), raw_stream(out.device))
    if st:
        _lib.check(st, entry)
    return out


class _FusedLinear(Function):
    @staticmethod
    def forward(ctx: Any, x, weight, bias, residual, code):
        need_x, need_w, need_b, _, _ = ctx.needs_input_grad
        y, rows, w, slope = _forward(x, weight, bias, residual, code,
                                     code != _lib.ACT_NONE and (need_x or need_w or need_b))
        ctx.save_for_backward(rows if need_w else None, w if need_x else None, slope)
        ctx.x_shape, ctx.w_shape, ctx.bias_dtype = x.shape, weight.shape, None if bias is None else bias.dtype
        return y

    @staticmethod
    @_runtime.first_order
    def backward(ctx: Any, grad: torch.Tensor):
        # What a hook or a checkpoint gives back need not lie in the layout that the forward pass saved.
        rows, w, slope = ctx.saved_tensors
        slope = None if slope is None else slope.contiguous()
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        lib, (N, K) = _lib.lib(), ctx.w_shape
        M, dev, dtype = math.prod(ctx.x_shape[:-1]), grad.device, grad.dtype
        code = _runtime.FLOAT_CODES[dtype]
        dx = dw = db = None
        dy = grad.reshape(M, N)
        dz = None
        if need_x or need_w:
            if slope is None:
                dz = dy = _padded(dy, zero_tail=True)
            else:
                dz = torch.empty(M, _whole(N, grad), dtype=dtype, device=dev)
        if slope is not None or need_b:
            if N > 1 and dy.stride(1) != 1:
                dy = dy.contiguous()
            db = torch.empty(N, dtype=ctx.bias_dtype, device=dev) if need_b else None
            ws = _workspace(lib.void_linear_grad_z_workspace_bytes(M, N, code), dev) if need_b else None
            bias_code = code if db is None else _runtime.FLOAT_CODES[db.dtype]
            st = lib.void_linear_grad_z(dy.data_ptr(), dy.stride(0), _ptr(slope), M, N, code,
                                        _ptr(dz) if slope is not None else None, 0 if dz is None else dz.stride(0),
                                        _ptr(db), bias_code, _ptr(ws), 0 if ws is None else ws.numel(), raw_stream(dev))
            if st:
                _lib.check(st, "void_linear_grad_z")
        if need_x:
            dx = _product("void_linear_grad_x", dz, _chunked(w), M, N, K,
                          torch.empty(M, K, dtype=dtype, device=dev)).view(ctx.x_shape)
        if need_w:
            dw = _product("void_linear_grad_w", dz, _chunked(rows), M, N, K,
                          torch.empty(N, K, dtype=dtype, device=dev))
        return dx, dw, db, grad if need_r else None, None


def _code(activation: Union[str, ActivationType]) -> int:
    name = activation.value if isinstance(activation, ActivationType) else str(activation).lower()
    if name not in _CODES:
        raise ValueError(f"unknown activation {activation!r}")
    return get_activation_code(name)


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Union[str, ActivationType] = "none",
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual in one product, differentiable.

    x [..., K] and weight [N, K] share a type (fp32, bf16 or fp16); bias is [N]
    (another type than x's is widened to fp32); residual has the result's shape
    [..., N] and x's type.  activation: "none", "relu", "gelu" (tanh form) or
    "silu".  Any strides are taken; for more than 64 rows, operands whose rows
    are not whole 16-byte chunks are copied to such once, and so are rows so far
    apart that 256 of them (or all) span 2 GiB.  Gradients flow to all
    four tensors and are not differentiable themselves.
    """
    code = _code(activation)
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {list(x.shape)} needs a weight [N, {x.shape[-1] if x.dim() else '?'}], got "
                         f"{list(weight.shape)}")
    _runtime.float_code(x, "x")
    if weight.dtype != x.dtype:
        raise TypeError(f"x is {x.dtype}, weight {weight.dtype}")
    N = weight.shape[0]
    if bias is not None:
        _runtime.float_code(bias, "bias")
        if bias.shape != (N,):
            raise ValueError(f"bias must be [{N}], got {list(bias.shape)}")
    if residual is not None:
        if residual.shape != x.shape[:-1] + (N,):
            raise ValueError(f"residual must be {list(x.shape[:-1]) + [N]}, got {list(residual.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"x is {x.dtype}, residual {residual.dtype}")
    _runtime.require_gpu(x, "x")
    for t, what in ((weight, "weight"), (bias, "bias"), (residual, "residual")):
        if t is not None and t.device != x.device:
            raise ValueError(f"x on {x.device}, {what} on {t.device}")
    if bias is not None:
        bias = (bias if bias.dtype in (x.dtype, torch.float32) else bias.to(torch.float32)).contiguous()
    if _runtime.differentiated(x, weight, bias, residual):
        return _FusedLinear.apply(x, weight, bias, residual, code)
    return _forward(x, weight, bias, residual, code, False)[0]


class FusedLinear(torch.nn.Module):
    """nn.Linear with an activation and a residual: activation(x W^T + b) + residual."""

    def __init__(self, in_features: int, out_features: int, activation: str = "none", bias: bool = True,
                 dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        linear = torch.nn.Linear(in_features, out_features, bias=bias, dtype=dtype, device=device)
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        _code(activation)
        self.weight = linear.weight
        self.register_parameter("bias", linear.bias)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return fused_linear(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"activation={self.activation}, bias={self.bias is not None}")


__all__ = ["fused_linear", "FusedLinear"]
