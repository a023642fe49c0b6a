"""Layer norm over the last axis, forward and backward (lncc_layer_norm_* in include/lncc.h).

    y = fused_layer_norm(x, weight, bias, eps=1e-5)

x: (..., C) float32, bfloat16 or float16; weight and bias (C,) of x's type or float32, or None. y has x's type, the
gradients the types of what they belong to. Statistics and sums are fp32; the weight's and the bias' gradients are
summed in a fixed order, so they are the same bits run after run. Strided rows are read where they lie.
"""
from typing import Optional

import torch

from . import _lib
from ._host import DTYPES, check_tensor, ptr, rows_of, scratch_for, stream_of

_WHAT = "layer_norm"


def _on_device(dev):
    from . import _on_device as f
    return f(dev)


def _wdtype(x, weight, bias):
    p = weight if weight is not None else bias
    return DTYPES[x.dtype if p is None else p.dtype]


def _forward_impl(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                  keep: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd); mean and rstd (rows,) fp32, empty without keep."""
    lib = _lib.load()
    with _on_device(x.device):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        rows, width = x.numel() // x.shape[-1], x.shape[-1]
        stats = torch.empty((2, rows if keep else 0), dtype=torch.float32, device=x.device)
        mean, rstd = stats.unbind(0)
        if rows:
            xr = rows_of(x)
            w = weight if weight is None else weight.contiguous()
            b = bias if bias is None else bias.contiguous()
            st = lib.lncc_layer_norm_forward(xr.data_ptr(), xr.stride(0), ptr(w), ptr(b), DTYPES[x.dtype],
                                             _wdtype(x, weight, bias), rows, width, eps, y.data_ptr(),
                                             mean.data_ptr() if keep else None, rstd.data_ptr() if keep else None,
                                             stream_of(x.device))
            _lib.check(st, "fused_lncc layer_norm forward")
    return y, mean, rstd


def _backward_impl(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                   rstd: torch.Tensor, wdtype: torch.dtype, need_x: bool,
                   need_params: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias), each empty where it is not needed."""
    lib = _lib.load()
    with _on_device(x.device):
        width, dev = x.shape[-1], x.device
        rows = x.numel() // width
        dx = torch.empty(x.shape if need_x else (0,), dtype=x.dtype, device=dev)
        dw = torch.empty(width if need_params else 0, dtype=wdtype, device=dev)
        db = torch.empty(width if need_params else 0, dtype=wdtype, device=dev)
        xr, dr = (rows_of(x), rows_of(dy)) if rows else (x, dy)
        ws, n = scratch_for(dev, "lncc_layer_norm_scratch_bytes", rows, width) if need_params else (None, 0)
        w = weight if weight is None else weight.contiguous()
        st = lib.lncc_layer_norm_backward(dr.data_ptr(), dr.stride(0) if rows else width, xr.data_ptr(),
                                          xr.stride(0) if rows else width, ptr(w), DTYPES[x.dtype], DTYPES[wdtype], rows,
                                          width, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr() if need_x else None,
                                          dw.data_ptr() if need_params else None, db.data_ptr() if need_params else None,
                                          ptr(ws), n, stream_of(dev))
        _lib.check(st, "fused_lncc layer_norm backward")
    return dx, dw, db


# Custom ops for torch.compile; eager calls go to the functions above directly, as the loss does.
def _forward_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                keep: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    y, mean, rstd = _forward_impl(x, weight, bias, eps, keep)
    return y, mean.clone(), rstd.clone()  # outputs of an op may not share memory


_forward_custom = torch.library.custom_op("fused_lncc::layer_norm", mutates_args=())(_forward_op)
_backward_custom = torch.library.custom_op("fused_lncc::layer_norm_backward", mutates_args=())(_backward_impl)


@_forward_custom.register_fake
def _(x, weight, bias, eps, keep):
    rows = x.numel() // x.shape[-1] if keep else 0
    return (x.new_empty(x.shape), x.new_empty((rows,), dtype=torch.float32), x.new_empty((rows,), dtype=torch.float32))


@_backward_custom.register_fake
def _(dy, x, weight, mean, rstd, wdtype, need_x, need_params):
    n = x.shape[-1] if need_params else 0
    return (x.new_empty(x.shape if need_x else (0,)), x.new_empty((n,), dtype=wdtype), x.new_empty((n,), dtype=wdtype))


class FusedLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        f = torch.ops.fused_lncc.layer_norm if torch.compiler.is_compiling() else _forward_impl
        y, mean, rstd = f(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        p = weight if weight is not None else bias
        ctx.wdtype = x.dtype if p is None else p.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        f = torch.ops.fused_lncc.layer_norm_backward if torch.compiler.is_compiling() else _backward_impl
        dx, dw, db = f(dy, x, weight, mean, rstd, ctx.wdtype, need_x, need_w or need_b)
        return dx if need_x else None, dw if need_w else None, db if need_b else None, None


def fused_layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (..., C), with the biased variance.

    weight, bias: (C,) of x's type or float32 (both of one type), or None for ones and zeros. The result has x's type.
    RuntimeError for tensors that are not on one CUDA device, of another type or of the wrong shape. A row with a NaN or
    an infinity gives NaN in that row (and in the weight's gradient), as the formula does."""
    check_tensor(_WHAT, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("fused_lncc: layer_norm: expect x (..., C) with C >= 1")
    grad = x.requires_grad
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            check_tensor(_WHAT, name, p, x.device)
            if p.dtype != x.dtype and p.dtype != torch.float32:
                raise RuntimeError(f"fused_lncc: layer_norm: {name} must be {x.dtype} or float32, got {p.dtype}")
            if p.dim() != 1 or p.shape[0] != x.shape[-1]:
                raise RuntimeError(f"fused_lncc: layer_norm: {name} must be ({x.shape[-1]},), got {tuple(p.shape)}")
            grad = grad or p.requires_grad
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("fused_lncc: layer_norm: weight and bias must have one type")
    if grad and torch.is_grad_enabled():
        return FusedLayerNorm.apply(x, weight, bias, float(eps))
    if torch.compiler.is_compiling():
        return torch.ops.fused_lncc.layer_norm(x, weight, bias, float(eps), False)[0]
    return _forward_impl(x, weight, bias, float(eps), False)[0]
