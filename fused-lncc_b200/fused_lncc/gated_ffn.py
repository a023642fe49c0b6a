"""The gated feed-forward block, forward and backward (lncc_gated_ffn_* in include/lncc.h).

    y = fused_gated_ffn(x, w_gate, w_up, w_down, activation="silu")

    g = x w_gate^T,  u = x w_up^T,  h = act(g) u,  y = h w_down^T

x: (..., K); w_gate, w_up: (F, K); w_down: (N, F), as torch.nn.Linear lays its weights out; all of one type, float32,
bfloat16 or float16. Sums are fp32. Nothing of the hidden layer is saved for the backward pass: it forms g, u and h again.
"""
import torch

from . import _lib
from ._host import DTYPES, check_tensor, rows_of, scratch_for, stream_of

_WHAT = "gated_ffn"
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


def _on_device(dev):
    from . import _on_device as f
    return f(dev)


def _forward_impl(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                  act: int) -> torch.Tensor:
    lib = _lib.load()
    (F, K), N = w_gate.shape, w_down.shape[0]
    M, dt = x.numel() // K, DTYPES[x.dtype]
    with _on_device(x.device):
        y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
        if M:
            xr = rows_of(x)
            wg, wu, wd = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
            ws, n = scratch_for(x.device, "lncc_gated_ffn_scratch_bytes", M, K, F, N, dt, 0)
            st = lib.lncc_gated_ffn_forward(xr.data_ptr(), xr.stride(0), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dt,
                                            act, M, K, F, N, y.data_ptr(), ws.data_ptr(), n, stream_of(x.device))
            _lib.check(st, "fused_lncc gated_ffn forward")
    return y


def _backward_impl(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                   act: int, need_x: bool, need_gate: bool, need_up: bool,
                   need_down: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw_gate, dw_up, dw_down), each empty where it is not needed."""
    lib = _lib.load()
    (F, K), N = w_gate.shape, w_down.shape[0]
    M, dt, dev = x.numel() // K, DTYPES[x.dtype], x.device
    with _on_device(dev):
        out = [torch.empty(shape if need else (0,), dtype=x.dtype, device=dev)
               for need, shape in ((need_x, x.shape), (need_gate, (F, K)), (need_up, (F, K)), (need_down, (N, F)))]
        xr, dr = (rows_of(x), rows_of(dy)) if M else (x, dy)
        wg, wu, wd = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
        ws, n = scratch_for(dev, "lncc_gated_ffn_scratch_bytes", M, K, F, N, dt, 1)
        st = lib.lncc_gated_ffn_backward(dr.data_ptr(), dr.stride(0) if M else N, xr.data_ptr(), xr.stride(0) if M else K,
                                         wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dt, act, M, K, F, N,
                                         *(t.data_ptr() if need else None
                                           for t, need in zip(out, (need_x, need_gate, need_up, need_down))),
                                         ws.data_ptr(), n, stream_of(dev))
        _lib.check(st, "fused_lncc gated_ffn backward")
    return tuple(out)


# Custom ops for torch.compile; eager calls go to the functions above directly, as the loss does.
_forward_custom = torch.library.custom_op("fused_lncc::gated_ffn", mutates_args=())(_forward_impl)
_backward_custom = torch.library.custom_op("fused_lncc::gated_ffn_backward", mutates_args=())(_backward_impl)


@_forward_custom.register_fake
def _(x, w_gate, w_up, w_down, act):
    return x.new_empty((*x.shape[:-1], w_down.shape[0]))


@_backward_custom.register_fake
def _(dy, x, w_gate, w_up, w_down, act, need_x, need_gate, need_up, need_down):
    return tuple(x.new_empty(t.shape if need else (0,))
                 for need, t in ((need_x, x), (need_gate, w_gate), (need_up, w_up), (need_down, w_down)))


class FusedGatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        f = torch.ops.fused_lncc.gated_ffn if torch.compiler.is_compiling() else _forward_impl
        ctx.save_for_backward(x, w_gate, w_up, w_down)
        ctx.act = act
        return f(x, w_gate, w_up, w_down, act)

    @staticmethod
    def backward(ctx, dy):
        need = ctx.needs_input_grad[:4]
        f = torch.ops.fused_lncc.gated_ffn_backward if torch.compiler.is_compiling() else _backward_impl
        grads = f(dy, *ctx.saved_tensors, ctx.act, *need)
        return (*(g if n else None for g, n in zip(grads, need)), None)


def fused_gated_ffn(x, w_gate, w_up, w_down, activation="silu"):
    """act(x w_gate^T) * (x w_up^T) taken through w_down^T: (..., K) -> (..., N).

    w_gate, w_up: (F, K); w_down: (N, F); activation: 'silu', 'gelu' (the exact one, with erf) or 'relu'. x may have
    strided rows. RuntimeError for wrong shapes, types or devices, ValueError for another activation.
    A NaN or an infinity in a token reaches that token's output and gradient, and the weights' gradients."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"fused_lncc: gated_ffn: activation must be 'silu', 'gelu' or 'relu', got {activation!r}")
    check_tensor(_WHAT, "x", x)
    for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        check_tensor(_WHAT, name, w, x.device, x.dtype)
        if w.dim() != 2 or 0 in w.shape:
            raise RuntimeError(f"fused_lncc: gated_ffn: {name} must be a matrix, got {tuple(w.shape)}")
    if x.dim() < 1 or x.shape[-1] != w_gate.shape[1] or w_up.shape != w_gate.shape or w_down.shape[1] != w_gate.shape[0]:
        raise RuntimeError("fused_lncc: gated_ffn: expect x (..., K), w_gate and w_up (F, K), w_down (N, F), got "
                           f"{tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad):
        return FusedGatedFFN.apply(x, w_gate, w_up, w_down, act)
    f = torch.ops.fused_lncc.gated_ffn if torch.compiler.is_compiling() else _forward_impl
    return f(x, w_gate, w_up, w_down, act)
