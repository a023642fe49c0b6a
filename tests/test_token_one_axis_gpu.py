"""GPU: x with one axis, a single token: strided, and with the expanded upstream gradient of a sum or a mean. The same call on x
as a matrix of one row is the reference, bit by bit (the kernels see the same row)."""
import pytest
import torch

import fused_lncc

pytestmark = pytest.mark.gpu


def _rand(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def _norm(x):
    return fused_lncc.fused_layer_norm(x, _rand(11, x.shape[-1]), _rand(12, x.shape[-1]))


def _ffn(x):
    n = x.shape[-1]
    return fused_lncc.fused_gated_ffn(x, _rand(11, 24, n), _rand(12, 24, n), _rand(13, 20, 24))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 33, 64])
@pytest.mark.parametrize("step", [1, 2, 3])
def test_norm_and_ffn_of_one_axis(n, step, dtype):
    for f in (_norm, _ffn) if dtype == torch.float32 else (lambda x: fused_lncc.fused_layer_norm(x),):
        x = _rand(1, n * step).to(dtype)[::step].detach().requires_grad_(True)
        row = x.detach().clone()[None].requires_grad_(True)
        y, want = f(x), f(row)
        assert y.shape == want.shape[1:] and torch.equal(y, want[0])
        for reduce in (torch.sum, torch.mean):
            (g,) = torch.autograd.grad(reduce(y), x, retain_graph=True)
            (w,) = torch.autograd.grad(reduce(want), row, retain_graph=True)
            assert g.shape == x.shape and torch.equal(g, w[0])
        up = _rand(2, y.numel() * 2).to(y.dtype)[::2]     # a strided upstream gradient
        (g,) = torch.autograd.grad(y, x, up)
        (w,) = torch.autograd.grad(want, row, up.clone()[None])
        assert torch.equal(g, w[0])
