"""CPU: the token blocks' C entry points refuse every pointer that is off its element's alignment, before any launch."""
import pytest

from fused_lncc import _lib

BAD_ARG = 1


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("wdtype,name,at", [(0, n, 66) for n in ("w", "b", "mean", "rstd")] + [(1, n, 65) for n in ("x", "w", "b", "y")])
def test_norm_forward(lib, wdtype, name, at):
    a = dict(x=64, x_stride=8, w=64, b=64, dtype=1, wdtype=wdtype, rows=2, width=8, eps=1e-5, y=64, mean=64, rstd=64, s=None)
    a[name] = at
    assert lib.lncc_layer_norm_forward(*a.values()) == BAD_ARG


@pytest.mark.parametrize("wdtype,name,at", [(0, n, 66) for n in ("w", "mean", "rstd", "dw", "db")] +
                         [(1, n, 65) for n in ("dy", "x", "w", "dx", "dw", "db")])
def test_norm_backward(lib, wdtype, name, at):
    a = dict(dy=64, dy_stride=8, x=64, x_stride=8, w=64, dtype=1, wdtype=wdtype, rows=2, width=8, mean=64, rstd=64, dx=64,
             dw=64, db=64, ws=64, n=1 << 20, s=None)
    a[name] = at
    assert lib.lncc_layer_norm_backward(*a.values()) == BAD_ARG


@pytest.mark.parametrize("name,at", [(n, 65) for n in ("x", "gate", "h")] + [(n, 66) for n in ("state", "last", "kept")])
def test_scan_forward(lib, name, at):
    a = dict(x=64, x_b=8, x_t=8, gate=64, g_b=8, g_t=8, state=64, dtype=1, B=1, T=100, C=8, reverse=0, h=64, last=64,
             kept=64, ws=64, n=1 << 30, s=None)
    a[name] = at
    assert lib.lncc_gated_scan_forward(*a.values()) == BAD_ARG


@pytest.mark.parametrize("name,at", [(n, 65) for n in ("dh", "x", "gate", "dx", "dgate")] + [(n, 66) for n in ("dlast", "kept", "dstate")])
def test_scan_backward(lib, name, at):
    a = dict(dh=64, dh_b=8, dh_t=8, dlast=64, x=64, x_b=8, x_t=8, gate=64, g_b=8, g_t=8, kept=64, dtype=1, B=1, T=100,
             C=8, reverse=0, dx=64, dgate=64, dstate=64, ws=64, n=1 << 30, s=None)
    a[name] = at
    assert lib.lncc_gated_scan_backward(*a.values()) == BAD_ARG


@pytest.mark.parametrize("dtype,at", [(0, 66), (1, 65)])
@pytest.mark.parametrize("name", ["x", "wg", "wu", "wd", "y"])
def test_ffn_forward(lib, name, dtype, at):
    a = dict(x=64, x_stride=8, wg=64, wu=64, wd=64, dtype=dtype, act=0, M=300, K=8, F=16, N=8, y=64, ws=1024, n=1 << 30, s=None)
    a[name] = at
    assert lib.lncc_gated_ffn_forward(*a.values()) == BAD_ARG


@pytest.mark.parametrize("dtype,at", [(0, 66), (1, 65)])
@pytest.mark.parametrize("name", ["dy", "x", "wg", "wu", "wd", "dx", "dwg", "dwu", "dwd"])
def test_ffn_backward(lib, name, dtype, at):
    a = dict(dy=64, dy_stride=8, x=64, x_stride=8, wg=64, wu=64, wd=64, dtype=dtype, act=0, M=300, K=8, F=16, N=8, dx=64,
             dwg=64, dwu=64, dwd=64, ws=1024, n=1 << 30, s=None)
    a[name] = at
    assert lib.lncc_gated_ffn_backward(*a.values()) == BAD_ARG
