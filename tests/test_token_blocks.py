"""CPU: the token-block oracle's gradients against differences and autograd, the operators' refusals that need no GPU,
and the C entry points' argument checks."""
import pytest
import torch

import fused_lncc
from oracle import token_blocks as ob


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=torch.float64)


def _differences(f, args, names, grads, gen, step=1e-6):
    """Central differences of the scalar f along a random direction of each argument, against <gradient, direction>."""
    for i, name in enumerate(names):
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * v, args[i] - step * v
        got = (f(*up) - f(*down)) / (2 * step)
        want = (grads[name] * v).sum()
        # truncation ~ step^2, rounding ~ 1e-16 * |f| / step: both below 1e-8 of values of order 100
        assert abs(got - want) <= 1e-6 * (1 + abs(want)), name


def test_norm_oracle_gradients():
    gen = torch.Generator().manual_seed(0)
    x, w, b, dy = _rand(gen, 5, 7), _rand(gen, 7), _rand(gen, 7), _rand(gen, 5, 7)
    o = ob.layer_norm(x, w, b, 1e-3, dy)
    _differences(lambda *a: (ob.layer_norm(*a, 1e-3)["y"] * dy).sum(), (x, w, b), ("dx", "dw", "db"), o, gen)


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_oracle_gradients(reverse):
    gen = torch.Generator().manual_seed(1)
    x, gate, state = _rand(gen, 2, 9, 3), _rand(gen, 2, 9, 3), _rand(gen, 2, 3)
    dh, dlast = _rand(gen, 2, 9, 3), _rand(gen, 2, 3)
    o = ob.gated_scan(x, gate, state, reverse, dh, dlast)

    def f(*a):
        r = ob.gated_scan(*a, reverse)
        return (r["h"] * dh).sum() + (r["last"] * dlast).sum()
    _differences(f, (x, gate, state), ("dx", "dgate", "dstate"), o, gen)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_ffn_oracle_gradients(act):
    gen = torch.Generator().manual_seed(2)
    x, wg, wu, wd = _rand(gen, 4, 5), _rand(gen, 6, 5), _rand(gen, 6, 5), _rand(gen, 3, 6)
    dy = _rand(gen, 4, 3)
    o = ob.gated_ffn(x, wg, wu, wd, act, dy)
    _differences(lambda *a: (ob.gated_ffn(*a, act)["y"] * dy).sum(), (x, wg, wu, wd),
                 ("dx", "dw_gate", "dw_up", "dw_down"), o, gen)


def test_refusals_without_gpu():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_lncc.fused_layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_lncc.fused_gated_scan(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_lncc.fused_gated_ffn(x, torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))
    with pytest.raises(ValueError, match="activation"):
        fused_lncc.fused_gated_ffn(x, x, x, x, activation="tanh")


def test_refusals_of_fake_cuda_tensors():
    """Every check of shapes, types and devices, without a GPU: fake tensors that say they are on one."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ln, scan, ffn = fused_lncc.fused_layer_norm, fused_lncc.fused_gated_scan, fused_lncc.fused_gated_ffn
    with FakeTensorMode():
        x, w, d = (torch.zeros(s, device="cuda") for s in ((4, 8), (16, 8), (8, 16)))
        half = torch.zeros(8, device="cuda", dtype=torch.float16)
        for call, why in ((lambda: ln(x.double()), "float32"), (lambda: ln(x, torch.zeros(7, device="cuda")), r"\(7\)"),
                          (lambda: ln(x, torch.zeros(8)), "CUDA"), (lambda: ln(x, half), "Half"),
                          (lambda: ln(x.half(), torch.zeros(8, device="cuda"), half), "one type"),
                          (lambda: ln(x[:, :0]), "C >= 1"), (lambda: scan(x, x), r"\(B, T, C\)"),
                          (lambda: scan(x[None], x[None].half()), "Half"), (lambda: scan(x[None], x[None, :3]), r"\(1, 3, 8\)"),
                          (lambda: scan(x[None], x[None], x), r"\(4, 8\)"), (lambda: ffn(x, w, w, w), r"w_down \(N, F\)"),
                          (lambda: ffn(x, w, w[:8], d), r"\(8, 8\)"), (lambda: ffn(x.half(), w, w, d), "Half"),
                          (lambda: ffn(x, w[0], w, d), "matrix"), (lambda: ffn(x, w, w, d.cpu()), "CUDA")):
            with pytest.raises(RuntimeError, match=why):
                call()


def test_torch_library_brings_no_second_libstdcxx():
    """One that defines std::ostream itself crashes on the first number in an error message."""
    import subprocess

    from fused_lncc import _native
    _native.load()
    out = subprocess.run(["nm", "-D", "--defined-only", _native.OPS_PATH], capture_output=True, text=True, check=True).stdout
    assert "_ZNSo9_M_insert" not in out


def test_custom_ops_registered():
    for name in ("layer_norm", "layer_norm_backward", "gated_scan", "gated_scan_backward", "gated_ffn",
                 "gated_ffn_backward"):
        assert hasattr(torch.ops.fused_lncc, name)


def test_fake_impls_give_shapes_and_types():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 5, 8, dtype=torch.bfloat16)
        y, mean, rstd = torch.ops.fused_lncc.layer_norm(x, None, None, 1e-5, True)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == (10,) and rstd.dtype == torch.float32
        h, last, kept = torch.ops.fused_lncc.gated_scan(x, x, None, False, True)
        assert h.shape == x.shape and last.shape == (2, 8) and last.dtype == torch.float32 and kept.dim() == 1
        w = torch.empty(12, 8, dtype=torch.bfloat16)
        y = torch.ops.fused_lncc.gated_ffn(x, w, w, torch.empty(6, 12, dtype=torch.bfloat16), 0)
        assert y.shape == (2, 5, 6) and y.dtype == torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from fused_lncc import _lib
    return _lib.load()


BAD_ARG, DTYPE, WORKSPACE, TOO_LARGE = 1, 3, 6, 8


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=5), DTYPE), (dict(dtype=1, wdtype=2), DTYPE), (dict(rows=-1), BAD_ARG), (dict(width=0), BAD_ARG),
    (dict(width=1 << 31), TOO_LARGE), (dict(x=None), BAD_ARG), (dict(x=2), BAD_ARG), (dict(y=None), BAD_ARG),
    (dict(x_stride=4), BAD_ARG), (dict(mean=None), BAD_ARG), (dict(rows=0), 0),
])
def test_norm_rejects_bad_arguments(lib, kw, status):
    a = dict(x=64, x_stride=8, w=None, b=None, dtype=0, wdtype=0, rows=2, width=8, eps=1e-5, y=64, mean=64, rstd=64, s=None)
    a.update(kw)
    assert lib.lncc_layer_norm_forward(*a.values()) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dy=None), BAD_ARG), (dict(dy_stride=3), BAD_ARG), (dict(mean=None), BAD_ARG), (dict(ws=None), WORKSPACE),
    (dict(n=4), WORKSPACE), (dict(dx=None, dw=None, db=None), 0), (dict(rows=0, dw=None, db=None), 0),
])
def test_norm_backward_rejects_bad_arguments(lib, kw, status):
    a = dict(dy=64, dy_stride=8, x=64, x_stride=8, w=None, dtype=0, wdtype=0, rows=2, width=8, mean=64, rstd=64, dx=64,
             dw=64, db=64, ws=64, n=1 << 20, s=None)
    a.update(kw)
    assert lib.lncc_layer_norm_backward(*a.values()) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=-1), DTYPE), (dict(B=-1), BAD_ARG), (dict(T=-1), BAD_ARG), (dict(C=0), BAD_ARG), (dict(B=70000), TOO_LARGE),
    (dict(x=None), BAD_ARG), (dict(gate=3), BAD_ARG), (dict(h=None), BAD_ARG), (dict(last=None), BAD_ARG),
    (dict(ws=None), WORKSPACE), (dict(n=1), WORKSPACE), (dict(B=0), 0),
])
def test_scan_rejects_bad_arguments(lib, kw, status):
    a = dict(x=64, x_b=8, x_t=8, gate=64, g_b=8, g_t=8, state=None, dtype=0, B=1, T=100, C=8, reverse=0, h=64, last=64,
             kept=None, ws=64, n=1 << 30, s=None)
    a.update(kw)
    assert lib.lncc_gated_scan_forward(*a.values()) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=9), DTYPE), (dict(dh=None), BAD_ARG), (dict(kept=None), BAD_ARG), (dict(dgate=None), BAD_ARG),
    (dict(ws=None), WORKSPACE), (dict(B=0), 0),
])
def test_scan_backward_rejects_bad_arguments(lib, kw, status):
    a = dict(dh=64, dh_b=8, dh_t=8, dlast=None, x=64, x_b=8, x_t=8, gate=64, g_b=8, g_t=8, kept=64, dtype=0, B=1, T=100,
             C=8, reverse=0, dx=64, dgate=64, dstate=None, ws=64, n=1 << 30, s=None)
    a.update(kw)
    assert lib.lncc_gated_scan_backward(*a.values()) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=4), DTYPE), (dict(act=3), BAD_ARG), (dict(act=-1), BAD_ARG), (dict(M=-1), BAD_ARG), (dict(K=0), BAD_ARG),
    (dict(F=1 << 21), TOO_LARGE), (dict(M=1 << 31), TOO_LARGE), (dict(x=None), BAD_ARG), (dict(x_stride=1), BAD_ARG),
    (dict(wd=None), BAD_ARG), (dict(y=None), BAD_ARG), (dict(ws=None), WORKSPACE), (dict(n=16), WORKSPACE), (dict(M=0), 0),
])
def test_ffn_rejects_bad_arguments(lib, kw, status):
    a = dict(x=64, x_stride=8, wg=64, wu=64, wd=64, dtype=0, act=0, M=300, K=8, F=16, N=8, y=64, ws=1024, n=1 << 30, s=None)
    a.update(kw)
    assert lib.lncc_gated_ffn_forward(*a.values()) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=4), DTYPE), (dict(act=3), BAD_ARG), (dict(dy=None), BAD_ARG), (dict(dy_stride=2), BAD_ARG),
    (dict(dx=2), BAD_ARG), (dict(ws=None), WORKSPACE), (dict(n=16), WORKSPACE),
])
def test_ffn_backward_rejects_bad_arguments(lib, kw, status):
    a = dict(dy=64, dy_stride=8, x=64, x_stride=8, wg=64, wu=64, wd=64, dtype=0, act=0, M=300, K=8, F=16, N=8, dx=64,
             dwg=64, dwu=64, dwd=64, ws=1024, n=1 << 30, s=None)
    a.update(kw)
    assert lib.lncc_gated_ffn_backward(*a.values()) == status


def test_kept_size_is_the_bindings(lib):
    from fused_lncc import _native
    for B, T, C in ((1, 1, 1), (2, 16, 5), (3, 17, 8), (1, 1000, 33)):
        assert lib.lncc_gated_scan_kept_bytes(B, T, C) == 4 * _native.kept_numel(B, T, C)
