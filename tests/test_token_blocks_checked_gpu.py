"""GPU: the token blocks in the bounds-checked build report no access outside an array, and its results are the product
library's up to rounding. (Not bit by bit: the compiler contracts multiplications and additions differently in the two. Each
result is within one rounding of its type and a few of fp32 of the exact one, so two of them are within 2u of the norm for
16-bit types, u = 2^-8 and 2^-11, and 1e-5 for fp32.)"""
import ctypes
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _open(checked):
    from fused_lncc import _lib
    if not checked:
        return _lib.load()
    path = os.path.join(os.path.dirname(_lib.LIB_PATH), "liblncc_sm100_checked.so")
    if not os.path.exists(path):
        import importlib.util
        spec = importlib.util.spec_from_file_location(
            "_b", os.path.join(os.path.dirname(os.path.dirname(_lib.LIB_PATH)), "build.py"))
        b = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(b)
        b.build_library(checked=True)
    lib = ctypes.CDLL(path)
    for name, (res, args) in _lib.SIGNATURES.items():
        f = getattr(lib, name)
        f.restype, f.argtypes = res, args
    assert lib.lncc_checked_build() == 1
    return lib


@pytest.fixture(scope="module")
def libs():
    return _open(False), _open(True)


def _rand(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _both(libs, call):
    """call(lib) -> (statuses, tensors), the same from both builds."""
    results = []
    for lib in libs:
        statuses, tensors = call(lib)
        torch.cuda.synchronize()
        assert statuses == [0] * len(statuses), statuses
        results.append(tensors)
    tol = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
    for a, b in zip(*results):
        assert (a.double() - b.double()).norm() <= tol[a.dtype] * b.double().norm()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,width", [(1, 1), (37, 97), (65, 384), (9, 1030), (3, 8192), (2, 9001)])
def test_norm(libs, rows, width, dtype):
    x, dy, w = _rand(1, rows, width, dtype=dtype), _rand(2, rows, width, dtype=dtype), _rand(3, width)
    dt = DT[dtype]

    def call(lib):
        y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        n = lib.lncc_layer_norm_scratch_bytes(rows, width)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        st = [lib.lncc_layer_norm_forward(x.data_ptr(), width, w.data_ptr(), None, dt, 0, rows, width, 1e-5, y.data_ptr(),
                                          mean.data_ptr(), rstd.data_ptr(), None),
              lib.lncc_layer_norm_backward(dy.data_ptr(), width, x.data_ptr(), width, w.data_ptr(), dt, 0, rows, width,
                                           mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                           ws.data_ptr(), n, None)]
        return st, (y, dx, dw, db)
    _both(libs, call)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (2, 17, 33), (1, 130, 96), (3, 1001, 40)])
@pytest.mark.parametrize("reverse", [0, 1])
def test_scan(libs, B, T, C, dtype, reverse):
    x, gate, dh = (_rand(s, B, T, C, dtype=dtype) for s in (1, 2, 3))
    state, dlast = _rand(4, B, C), _rand(5, B, C)
    dt = DT[dtype]

    def call(lib):
        h, dx, dgate = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        last, dstate = torch.empty_like(state), torch.empty_like(state)
        kept = torch.empty(lib.lncc_gated_scan_kept_bytes(B, T, C) // 4, device="cuda")
        n = lib.lncc_gated_scan_scratch_bytes(B, T, C)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        st = [lib.lncc_gated_scan_forward(x.data_ptr(), T * C, C, gate.data_ptr(), T * C, C, state.data_ptr(), dt, B, T, C, reverse,
                                          h.data_ptr(), last.data_ptr(), kept.data_ptr(), ws.data_ptr(), n, None),
              lib.lncc_gated_scan_backward(dh.data_ptr(), T * C, C, dlast.data_ptr(), x.data_ptr(), T * C, C, gate.data_ptr(),
                                           T * C, C, kept.data_ptr(), dt, B, T, C, reverse, dx.data_ptr(), dgate.data_ptr(),
                                           dstate.data_ptr(), ws.data_ptr(), n, None)]
        return st, (h, last, dx, dgate, dstate)
    _both(libs, call)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("M,K,F,N", [(1, 64, 128, 64), (3, 33, 51, 27), (130, 72, 200, 40), (301, 97, 130, 259)])
def test_ffn(libs, M, K, F, N, act, dtype):
    x, dy = _rand(1, M, K, dtype=dtype), _rand(2, M, N, dtype=dtype)
    wg, wu, wd = (_rand(s, *shape, dtype=dtype, scale=0.1) for s, shape in ((3, (F, K)), (4, (F, K)), (5, (N, F))))
    dt = DT[dtype]

    def call(lib):
        y, grads = torch.empty_like(dy), [torch.empty_like(t) for t in (x, wg, wu, wd)]
        nf, nb = (lib.lncc_gated_ffn_scratch_bytes(M, K, F, N, dt, b) for b in (0, 1))
        ws = torch.empty(max(nf, nb), dtype=torch.uint8, device="cuda")
        st = [lib.lncc_gated_ffn_forward(x.data_ptr(), K, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dt, act, M, K, F, N,
                                         y.data_ptr(), ws.data_ptr(), nf, None),
              lib.lncc_check_abort(ws.data_ptr(), None),  # no wait ran out
              lib.lncc_gated_ffn_backward(dy.data_ptr(), N, x.data_ptr(), K, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dt, act,
                                          M, K, F, N, *(g.data_ptr() for g in grads), ws.data_ptr(), nb, None),
              lib.lncc_check_abort(ws.data_ptr(), None)]
        return st, (y, *grads)
    _both(libs, call)
