"""Layer norm over the last axis, forward and backward (lncc_layer_norm_* in include/lncc.h).

    y = fused_layer_norm(x, weight, bias, eps=1e-5)

x: (..., C) float32, bfloat16 or float16; weight and bias (C,) of x's type or float32, or None. y has x's type, the
gradients the types of what they belong to. Statistics and sums are fp32; the weight's and the bias' gradients are
summed in a fixed order, so they are the same bits run after run. Strided rows are read where they lie.
"""
import torch
from torch.overrides import has_torch_function

from . import _native


def fused_layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (..., C), with the biased variance.

    weight, bias: (C,) of x's type or float32 (both of one type), or None for ones and zeros. The result has x's type.
    RuntimeError for tensors that are not on one CUDA device, of another type or of the wrong shape. A row with a NaN or
    an infinity gives NaN in that row (and in the weight's gradient), as the formula does."""
    module = _native.load()
    if torch.compiler.is_compiling() or has_torch_function((x, weight, bias)):
        return torch.ops.fused_lncc.fused_layer_norm(x, weight, bias, eps)
    return module.layer_norm(x, weight, bias, eps)
