"""GPU: the 16-bit feed-forward block's activations and their derivatives, gate by gate, far into the lower tail.

One-hot tokens and a unit matrix make every hidden value a result of its own: y[f] = act(v_f) u_f with one rounding, and
dWg[f, 0] = M dh u_f act'(v_f) with one. A result may be off by that rounding and by 3e-5 of what it is made of: the
polynomial's 7.5e-6, and the fast exponential's and reciprocal's few 2^-24, of which the exponential's argument adds
|log2| (up to 100) x 2^-24. u_f is a power of 2 that brings the value near 1, within fp16's range."""
import math

import pytest
import torch

import fused_lncc
from oracle import token_blocks as ob

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _tensors(v, about, M, dtype):
    """Tokens and weights for gates v and up projections that bring `about` near 1."""
    F = len(v)
    limit = 15 if dtype == torch.float16 else 60
    power = (-torch.log2(about.abs()).round()).clamp(-limit, 2 * limit)
    first = torch.full_like(power, limit).minimum(power.clamp(min=0))
    x = torch.zeros(M, 64, device="cuda")
    x[:, 0], x[:, 1] = 1, 1
    wg, wu = torch.zeros(F, 64, device="cuda"), torch.zeros(F, 64, device="cuda")
    wg[:, 0] = v
    wu[:, 1] = 2.0 ** first
    scale = 2.0 ** (power - first)        # what one factor cannot hold goes into the unit matrix
    return x.to(dtype), wg.to(dtype), wu.to(dtype), torch.diag(scale).to(dtype), 2.0 ** first, scale


def _gates(dtype, low):
    g = torch.Generator(device="cuda").manual_seed(7)
    v = torch.rand(120, generator=g, device="cuda") * (6 - low) + low
    v = torch.cat([v, torch.tensor([low, -4.5, -5.0, -6.0, -1e-3, 0.0, 1e-3, 6.0], device="cuda")])
    return v.to(dtype).float().double()


@pytest.mark.parametrize("dtype,act,low", [(torch.float16, "gelu", -6.0), (torch.bfloat16, "gelu", -11.0),
                                           (torch.float16, "silu", -15.0), (torch.bfloat16, "silu", -60.0)])
@pytest.mark.parametrize("M", [1, 4, 8, 130])
def test_activation(dtype, act, low, M):
    v = _gates(dtype, low)
    a, _ = ob.activation(v, act)
    x, wg, wu, wd, u, scale = _tensors(v, torch.where(a == 0, torch.ones_like(a), a), M, dtype)
    y = fused_lncc.fused_gated_ffn(x, wg, wu, wd, activation=act).double()
    want = a * u * scale
    assert ((y - want).abs() <= (U[dtype] * 1.01 + 3e-5) * want.abs()).all(), ((y - want) / want).abs().max()


@pytest.mark.parametrize("dtype,act,low", [(torch.float16, "gelu", -6.0), (torch.bfloat16, "gelu", -11.0),
                                           (torch.float16, "silu", -15.0), (torch.bfloat16, "silu", -60.0)])
def test_derivative(dtype, act, low):
    v = _gates(dtype, low)
    _, da = ob.activation(v, act)
    if act == "gelu":
        made_of = (v * torch.exp(-v * v / 2)).abs() / math.sqrt(2 * math.pi) + 0.5 * torch.erfc(-v / math.sqrt(2))
    else:
        made_of = torch.sigmoid(v) * (1 + (v * torch.sigmoid(-v)).abs())
    M = 8
    x, wg, wu, wd, u, scale = _tensors(v, made_of, M, dtype)
    wg.requires_grad_(True)
    y = fused_lncc.fused_gated_ffn(x, wg, wu, wd, activation=act)
    (dwg,) = torch.autograd.grad(y, wg, torch.ones_like(y))
    got, want = dwg[:, 0].double(), M * da * u * scale
    tol = U[dtype] * 1.01 * want.abs() + 3e-5 * M * made_of * u * scale
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
