"""GPU: the fp32 feed-forward block with ReLU where many gates are exactly 0 (padded tokens, pruned units), NaN, or formed from
rows whose squares leave the range of fp32."""
import pytest
import torch

import fused_lncc
from oracle import token_blocks as ob

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _grads(x, wg, wu, wd, dy):
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    return torch.autograd.grad(fused_lncc.fused_gated_ffn(*leaves, activation="relu"), leaves, dy)


def _near(got, want):
    """Sums of up to 1100 terms of 24 bits wander by some sqrt(1100) u32; 64 u32 of the norm."""
    assert (got.double() - want).norm() <= 64 * U32 * want.norm()


def _case(M, K, F, N):
    # gates that are whole numbers: their sign is the same in any order of summation
    g = torch.Generator(device="cuda").manual_seed(1)
    x, wg = (torch.randint(-2, 3, s, generator=g, device="cuda").float() for s in ((M, K), (F, K)))
    return x, wg, _rand(2, F, K, scale=K ** -0.5), _rand(3, N, F, scale=F ** -0.5), _rand(4, M, N)


def test_zero_rows():
    x, wg, wu, wd, dy = _case(300, 70, 120, 40)
    x[::2] = 0
    x[5, :69] = 0
    wg[::3] = 0
    for got, name in zip(_grads(x, wg, wu, wd, dy), ("dx", "dw_gate", "dw_up", "dw_down")):
        _near(got, ob.gated_ffn(x, wg, wu, wd, "relu", dy)[name])


def test_nan_rows_reach_their_own_gradient_alone():
    x, wg, wu, wd, dy = _case(200, 70, 120, 40)
    x[7, 3] = float("nan")
    dx = _grads(x, wg, wu, wd, dy)[0]
    keep = torch.arange(200, device="cuda") != 7
    assert dx[7].isnan().all()
    _near(dx[keep], ob.gated_ffn(x[keep], wg, wu, wd, "relu", dy[keep])["dx"])


@pytest.mark.parametrize("power", [-75, 0, 60])
def test_gates_at_zero_of_very_small_and_large_rows(power):
    """Gates closer to 0 than any order of summation can tell get the sign of the plain sum, whatever x's scale: a power of 2
    changes no rounding. (At 2^60 and 2^-75 the squares of a row pass fp32's range.)"""
    M, K, F = 130, 300, 72
    x, wg = _rand(1, M, K), _rand(2, F, K)
    x[:, K // 2:], wg[:, K // 2:] = x[:, :K // 2], -wg[:, :K // 2]
    wu, wd, dy = _rand(3, F, K, scale=K ** -0.5), _rand(4, 64, F, scale=F ** -0.5), _rand(5, M, 64)
    xs, ws = x.cpu(), wg.cpu()
    g = torch.zeros(M, F, dtype=torch.float64)
    for k in range(K):  # a multiply-add rounds once
        g = (g + xs[:, k, None].double() * ws[None, :, k].double()).float().double()
    on = (g > 0).double().cuda()
    assert 0 < on.mean() < 1
    dh = dy.double() @ wd.double()
    want = (dh * (x.double() @ wu.double().T) * on) @ wg.double() + (dh * g.cuda().clamp(min=0)) @ wu.double()
    got = _grads(x * 2.0 ** power, wg, wu, wd, dy)[0]
    _near(got.double() * 2.0 ** -power, want)


def test_zero_tokens_cost_no_more():
    """Half of the tokens padded: less work, not 24 times the time (which forming each of their gates again took)."""
    x, wg, wu, wd, dy = _rand(1, 4096, 512), _rand(2, 1024, 512), _rand(3, 1024, 512), _rand(4, 512, 1024), _rand(5, 4096, 512)

    def time(x):
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = fused_lncc.fused_gated_ffn(*leaves, activation="relu")
        best = float("inf")
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            torch.autograd.grad(y, leaves, dy, retain_graph=True)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    dense = time(x)
    x[::2] = 0
    assert time(x) < 2 * dense
