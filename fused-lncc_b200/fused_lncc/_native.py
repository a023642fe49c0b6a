"""Loads libfused_lncc_torch.so, which gives torch the token-block operators (csrc/torch_ops.cpp), and tells torch.compile
their shapes. Like the C library it is built in-tree once where it is missing, or was built against another torch, and there
is no fallback. The loss needs none of it: a library that does not load is an error of the token-block functions alone."""
import importlib.machinery
import importlib.util
import os
import threading

import torch

from . import _lib

OPS_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libfused_lncc_torch.so")
KEEP = 16  # steps of the gated scan from one kept state to the next (lncc_gated_scan_kept_bytes)

_lock = threading.Lock()
_module = None


def _mark():
    """The last bytes of a library that is whole and was built against the torch that is installed (build.py: torch_mark)."""
    return f"fused_lncc token blocks for torch {torch.__version__}, cxx11 abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}".encode()


def _matches():
    mark = _mark()
    try:
        with open(OPS_PATH, "rb") as f:
            f.seek(-len(mark), os.SEEK_END)
            return f.read() == mark
    except OSError:
        return False


def _build():
    spec = importlib.util.spec_from_file_location(
        "_lncc_build", os.path.join(os.path.dirname(os.path.dirname(_lib.LIB_PATH)), "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.build_torch_ops()


def kept_numel(B, T, C):
    return B * ((T + KEEP - 1) // KEEP) * C


def load():
    """The library as a module: layer_norm, gated_scan and gated_ffn for eager calls. torch.ops.fused_lncc has the operators
    once it is loaded."""
    global _module
    if _module is None:
        with _lock:
            if _module is None:
                if not _matches():
                    _build()
                _lib.load()
                try:
                    loader = importlib.machinery.ExtensionFileLoader("libfused_lncc_torch", OPS_PATH)
                    module = importlib.util.module_from_spec(importlib.util.spec_from_loader(loader.name, loader))
                    loader.exec_module(module)
                except ImportError as e:
                    raise RuntimeError(f"fused_lncc: {OPS_PATH} does not load ({e}); build it again with "
                                       "build.py --force") from e
                _register_fakes()
                _module = module
    return _module


def _register_fakes():
    fake = torch.library.register_fake

    @fake("fused_lncc::layer_norm")
    def _(x, weight, bias, eps, keep):
        rows = x.numel() // x.shape[-1] if keep else 0
        return x.new_empty(x.shape), x.new_empty((rows,), dtype=torch.float32), x.new_empty((rows,), dtype=torch.float32)

    @fake("fused_lncc::layer_norm_backward")
    def _(dy, x, weight, mean, rstd, wdtype, need_x, need_params):
        n = x.shape[-1] if need_params else 0
        return x.new_empty(x.shape if need_x else (0,)), x.new_empty((n,), dtype=wdtype), x.new_empty((n,), dtype=wdtype)

    @fake("fused_lncc::gated_scan")
    def _(x, gate, state, reverse, keep):
        B, T, C = x.shape
        return (x.new_empty((B, T, C)), x.new_empty((B, C), dtype=torch.float32),
                x.new_empty((kept_numel(B, T, C) if keep else 0,), dtype=torch.float32))

    @fake("fused_lncc::gated_scan_backward")
    def _(dh, dlast, x, gate, kept, reverse, need_state):
        B, T, C = x.shape
        return (x.new_empty((B, T, C)), x.new_empty((B, T, C)),
                x.new_empty((B, C) if need_state else (0,), dtype=torch.float32))

    @fake("fused_lncc::gated_ffn")
    def _(x, w_gate, w_up, w_down, act):
        return x.new_empty((*x.shape[:-1], w_down.shape[0]))

    @fake("fused_lncc::gated_ffn_backward")
    def _(dy, x, w_gate, w_up, w_down, act, need_x, need_gate, need_up, need_down):
        return tuple(x.new_empty(t.shape if need else (0,))
                     for need, t in ((need_x, x), (need_gate, w_gate), (need_up, w_up), (need_down, w_down)))


if _matches():
    try:
        load()
    except (RuntimeError, OSError, AttributeError):  # the first call of a token-block function raises it
        pass
