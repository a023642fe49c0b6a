"""The gated feed-forward block, forward and backward (lncc_gated_ffn_* in include/lncc.h).

    y = fused_gated_ffn(x, w_gate, w_up, w_down, activation="silu")

    g = x w_gate^T,  u = x w_up^T,  h = act(g) u,  y = h w_down^T

x: (..., K); w_gate, w_up: (F, K); w_down: (N, F), as torch.nn.Linear lays its weights out; all of one type, float32,
bfloat16 or float16. Sums are fp32; for 16-bit types and more than four tokens the hidden values are rounded to the type's bits between
the products, in float16 too without its range: hidden values past 65504 and gradients below 2^-24 are held. Nothing of the
hidden layer is saved for the backward pass: it forms g, u and h again.
"""
import torch
from torch.overrides import has_torch_function

from . import _native

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


def fused_gated_ffn(x, w_gate, w_up, w_down, activation="silu"):
    """act(x w_gate^T) * (x w_up^T) taken through w_down^T: (..., K) -> (..., N).

    w_gate, w_up: (F, K); w_down: (N, F); activation: 'silu', 'gelu' (the exact one, with erf) or 'relu'. x may have
    strided rows. RuntimeError for wrong shapes, types or devices, ValueError for another activation.
    A NaN or an infinity in a token reaches that token's output and gradient, and the weights' gradients."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"fused_lncc: gated_ffn: activation must be 'silu', 'gelu' or 'relu', got {activation!r}")
    module = _native.load()
    if torch.compiler.is_compiling() or has_torch_function((x, w_gate, w_up, w_down)):
        return torch.ops.fused_lncc.fused_gated_ffn(x, w_gate, w_up, w_down, act)
    return module.gated_ffn(x, w_gate, w_up, w_down, act)
