"""The gated linear recurrence over a sequence, forward and backward (lncc_gated_scan_* in include/lncc.h).

    h, last = fused_gated_scan(x, gate, state=None, reverse=False)

    a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h_0 = state or 0

x, gate: (B, T, C) of one type, float32, bfloat16 or float16; state and last (B, C) float32. A sequence can be taken in
pieces, down to single tokens, by handing each call the state that the one before returned. The state is fp32
throughout; h is rounded to x's type as it is written, and no rounded value is carried on. The backward pass forms h
again from fp32 states that the forward pass kept, so nothing of h is saved.
"""
import torch
from torch.overrides import has_torch_function

from . import _native


def fused_gated_scan(x, gate, state=None, reverse=False):
    """h_t = sigmoid(gate_t) h_{t-1} + (1 - sigmoid(gate_t)) x_t along T: returns (h, last).

    x, gate: (B, T, C) of one type, any batch and time strides. state: (B, C), the state before the first step, or None
    for zeros. reverse: from the last step to the first. h: (B, T, C) of x's type; last: (B, C) float32, the state after
    the last step taken. Gradients flow to x, gate and state from both results.
    A gate of +inf keeps the state and ignores x_t, one of -inf forgets the state (x_t and the state have to be finite
    all the same: the formula multiplies them by zero). RuntimeError for wrong shapes, types or devices."""
    module = _native.load()
    if torch.compiler.is_compiling() or has_torch_function((x, gate, state)):
        return torch.ops.fused_lncc.fused_gated_scan(x, gate, state, reverse)
    return module.gated_scan(x, gate, state, reverse)
