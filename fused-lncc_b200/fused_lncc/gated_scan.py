"""The gated linear recurrence over a sequence, forward and backward (lncc_gated_scan_* in include/lncc.h).

    h, last = fused_gated_scan(x, gate, state=None, reverse=False)

    a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h_0 = state or 0

x, gate: (B, T, C) of one type, float32, bfloat16 or float16; state and last (B, C) float32. A sequence can be taken in
pieces, down to single tokens, by handing each call the state that the one before returned. The state is fp32
throughout; h is rounded to x's type as it is written, and no rounded value is carried on. The backward pass forms h
again from fp32 states that the forward pass kept, so nothing of h is saved.
"""
from typing import Optional

import torch

from . import _lib
from ._host import DTYPES, check_tensor, ptr, scratch_for, stream_of

_WHAT = "gated_scan"
KEEP = 16  # steps from one kept state to the next (lncc_gated_scan_kept_bytes)


def _on_device(dev):
    from . import _on_device as f
    return f(dev)


def _kept_numel(B, T, C):
    return B * ((T + KEEP - 1) // KEEP) * C


def _forward_impl(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor], reverse: bool,
                  keep: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(h, last, kept states); the states empty without keep."""
    lib = _lib.load()
    B, T, C = x.shape
    with _on_device(x.device):
        x = x if x.stride(2) == 1 else x.contiguous()
        gate = gate if gate.stride(2) == 1 else gate.contiguous()
        h = torch.empty((B, T, C), dtype=x.dtype, device=x.device)
        last = torch.empty((B, C), dtype=torch.float32, device=x.device)
        kept = torch.empty(_kept_numel(B, T, C) if keep else 0, dtype=torch.float32, device=x.device)
        s = None if state is None else state.contiguous()
        ws, n = scratch_for(x.device, "lncc_gated_scan_scratch_bytes", B, T, C)
        st = lib.lncc_gated_scan_forward(x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0),
                                         gate.stride(1), ptr(s), DTYPES[x.dtype], B, T, C, int(reverse), h.data_ptr(),
                                         last.data_ptr(), kept.data_ptr() if keep else None, ws.data_ptr(), n,
                                         stream_of(x.device))
        _lib.check(st, "fused_lncc gated_scan forward")
    return h, last, kept


def _backward_impl(dh: torch.Tensor, dlast: Optional[torch.Tensor], x: torch.Tensor, gate: torch.Tensor,
                   kept: torch.Tensor, reverse: bool,
                   need_state: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgate, dstate); dstate empty where it is not needed."""
    lib = _lib.load()
    B, T, C = x.shape
    with _on_device(x.device):
        x = x if x.stride(2) == 1 else x.contiguous()
        gate = gate if gate.stride(2) == 1 else gate.contiguous()
        dh = dh if dh.stride(2) == 1 else dh.contiguous()
        dx = torch.empty((B, T, C), dtype=x.dtype, device=x.device)
        dgate = torch.empty((B, T, C), dtype=x.dtype, device=x.device)
        dstate = torch.empty((B, C) if need_state else (0,), dtype=torch.float32, device=x.device)
        dl = None if dlast is None else dlast.contiguous()
        ws, n = scratch_for(x.device, "lncc_gated_scan_scratch_bytes", B, T, C)
        st = lib.lncc_gated_scan_backward(dh.data_ptr(), dh.stride(0), dh.stride(1), ptr(dl), x.data_ptr(), x.stride(0),
                                          x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1), kept.data_ptr(),
                                          DTYPES[x.dtype], B, T, C, int(reverse), dx.data_ptr(), dgate.data_ptr(),
                                          dstate.data_ptr() if need_state else None, ws.data_ptr(), n,
                                          stream_of(x.device))
        _lib.check(st, "fused_lncc gated_scan backward")
    return dx, dgate, dstate


# Custom ops for torch.compile; eager calls go to the functions above directly, as the loss does.
_forward_custom = torch.library.custom_op("fused_lncc::gated_scan", mutates_args=())(_forward_impl)
_backward_custom = torch.library.custom_op("fused_lncc::gated_scan_backward", mutates_args=())(_backward_impl)


@_forward_custom.register_fake
def _(x, gate, state, reverse, keep):
    B, T, C = x.shape
    return (x.new_empty((B, T, C)), x.new_empty((B, C), dtype=torch.float32),
            x.new_empty((_kept_numel(B, T, C) if keep else 0,), dtype=torch.float32))


@_backward_custom.register_fake
def _(dh, dlast, x, gate, kept, reverse, need_state):
    B, T, C = x.shape
    return (x.new_empty((B, T, C)), x.new_empty((B, T, C)),
            x.new_empty((B, C) if need_state else (0,), dtype=torch.float32))


class FusedGatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, reverse):
        f = torch.ops.fused_lncc.gated_scan if torch.compiler.is_compiling() else _forward_impl
        h, last, kept = f(x, gate, state, reverse, True)
        ctx.save_for_backward(x, gate, kept)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        x, gate, kept = ctx.saved_tensors
        if dh is None and dlast is None:
            return None, None, None, None
        if dh is None:
            dh = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        f = torch.ops.fused_lncc.gated_scan_backward if torch.compiler.is_compiling() else _backward_impl
        dx, dgate, dstate = f(dh, dlast, x, gate, kept, ctx.reverse, ctx.needs_input_grad[2])
        return (dx if ctx.needs_input_grad[0] else None, dgate if ctx.needs_input_grad[1] else None,
                dstate if ctx.needs_input_grad[2] else None, None)


def fused_gated_scan(x, gate, state=None, reverse=False):
    """h_t = sigmoid(gate_t) h_{t-1} + (1 - sigmoid(gate_t)) x_t along T: returns (h, last).

    x, gate: (B, T, C) of one type, any batch and time strides. state: (B, C), the state before the first step, or None
    for zeros. reverse: from the last step to the first. h: (B, T, C) of x's type; last: (B, C) float32, the state after
    the last step taken. Gradients flow to x, gate and state from both results.
    A gate of +inf keeps the state and ignores x_t, one of -inf forgets the state (x_t and the state have to be finite
    all the same: the formula multiplies them by zero). RuntimeError for wrong shapes, types or devices."""
    check_tensor(_WHAT, "x", x)
    if x.dim() != 3 or x.shape[2] < 1:
        raise RuntimeError(f"fused_lncc: gated_scan: expect x (B, T, C) with C >= 1, got {tuple(x.shape)}")
    check_tensor(_WHAT, "gate", gate, x.device, x.dtype)
    if gate.shape != x.shape:
        raise RuntimeError(f"fused_lncc: gated_scan: gate must be {tuple(x.shape)}, got {tuple(gate.shape)}")
    grad = x.requires_grad or gate.requires_grad
    if state is not None:
        check_tensor(_WHAT, "state", state, x.device)
        if state.shape != (x.shape[0], x.shape[2]):
            raise RuntimeError(f"fused_lncc: gated_scan: state must be {(x.shape[0], x.shape[2])}, got {tuple(state.shape)}")
        if state.dtype != torch.float32:
            state = state.float()
        grad = grad or state.requires_grad
    if grad and torch.is_grad_enabled():
        return FusedGatedScan.apply(x, gate, state, bool(reverse))
    f = torch.ops.fused_lncc.gated_scan if torch.compiler.is_compiling() else _forward_impl
    return f(x, gate, state, bool(reverse), False)[:2]
