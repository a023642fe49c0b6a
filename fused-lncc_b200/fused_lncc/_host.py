"""Host side shared by the token-block operators (layer_norm.py, gated_scan.py, gated_ffn.py): checks, row views, streams."""
import functools

import torch

from . import _lib

DTYPES = {torch.float32: _lib.LNCC_F32, torch.bfloat16: _lib.LNCC_BF16, torch.float16: _lib.LNCC_F16}


def check_tensor(what, name, t, device=None, dtype=None):
    """RuntimeErrors in the manner of the loss: CUDA tensors of one device, float32, bfloat16 or float16."""
    if not t.is_cuda:
        raise RuntimeError(f"fused_lncc: {what}: {name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise RuntimeError(f"fused_lncc: {what}: {name} must be on {device}, got {t.device}")
    if t.dtype not in DTYPES:
        raise RuntimeError(f"fused_lncc: {what}: float32, bfloat16 or float16 only, got {name} of {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"fused_lncc: {what}: {name} must be {dtype}, got {t.dtype}")


def rows_of(t):
    """t (..., C) as (rows, C) with contiguous rows at one stride of at least C: a view where its strides allow it."""
    if t.is_contiguous():
        return t.view(t.numel() // t.shape[-1], t.shape[-1])
    if t.dim() != 2:
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            return t.reshape(-1, t.shape[-1]).contiguous()
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t
    return t.contiguous()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_of(device):
    return torch.cuda.current_stream(device).cuda_stream


@functools.lru_cache(maxsize=4096)
def scratch_bytes(name, *sizes):
    """Bytes of a call's scratch as the library gives them; they depend on the sizes alone."""
    return getattr(_lib.load(), name)(*sizes)


def scratch_for(device, name, *sizes):
    n = scratch_bytes(name, *sizes)
    return torch.empty(n, dtype=torch.uint8, device=device), n
