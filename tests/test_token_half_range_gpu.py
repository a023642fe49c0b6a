"""GPU: the fp16 feed-forward block where hidden values or their gradients leave fp16's range, though inputs and results do not.

Tolerances as for the block at large: a result has its own rounding and that of h, dg or du, two independent relative errors of at
most u = 2^-11 and under u/2 in the mean, so u of the norm, and half the smallest subnormal, 2^-25, for each element. Rows of a
result are looked at one by one where tokens differ in size."""
import pytest
import torch

import fused_lncc
from oracle import token_blocks as ob

pytestmark = pytest.mark.gpu
U, TINY = 2.0 ** -11, 2.0 ** -25
H = torch.float16


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _weights(K, F, N, seed=10, down=1.0):
    return [t.to(H) for t in (_rand(seed, F, K, scale=K ** -0.5), _rand(seed + 1, F, K, scale=K ** -0.5),
                              _rand(seed + 2, N, F, scale=down * F ** -0.5))]


def _near(got, want, rows=False):
    assert got.dtype == H and got.shape == want.shape
    off = got.double() - want
    if rows:
        assert (off.norm(dim=1) <= U * want.norm(dim=1) + TINY * want.shape[1] ** 0.5).all()
    else:
        assert off.norm() <= U * want.norm() + TINY * want.numel() ** 0.5, (off.norm() / want.norm()).item()


def _run(x, w, dy, act):
    leaves = [t.detach().requires_grad_(True) for t in (x, *w)]
    y = fused_lncc.fused_gated_ffn(*leaves, activation=act)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,K,F,N", [(4, 96, 256, 96), (5, 96, 256, 96), (8, 768, 2048, 768), (300, 97, 130, 41), (512, 768, 2048, 768)])
def test_hidden_values_past_65504(M, K, F, N, act):
    x = _rand(1, M, K, scale=300).to(H)
    w = _weights(K, F, N, down=2.0 ** -10)
    dy = _rand(2, M, N, scale=2.0 ** -10).to(H)
    ref = ob.gated_ffn(x, *w, act, dy)
    g = x.double() @ w[0].double().T
    assert (ob.activation(g, act)[0] * (x.double() @ w[1].double().T)).abs().max() > 1.2e5
    got = _run(x, w, dy, act)
    for name, t in zip(NAMES, got):
        if ref[name].abs().max() < 6e4:
            assert t.isfinite().all()
            _near(t, ref[name])
    assert ref["y"].abs().max() < 6e4


@pytest.mark.parametrize("scale", [1.0, 1e-3, 1e-5, 1e-6])
@pytest.mark.parametrize("M,K,F,N", [(5, 96, 256, 96), (4096, 96, 256, 96), (700, 33, 70, 50)])
def test_small_upstream_gradients(M, K, F, N, scale):
    """As a mean over tokens leaves them."""
    x, w, dy = _rand(1, M, K).to(H), _weights(K, F, N), _rand(2, M, N, scale=scale).to(H)
    for act in ("silu", "gelu"):
        ref = ob.gated_ffn(x, *w, act, dy)
        for name, t in zip(NAMES, _run(x, w, dy, act)):
            _near(t, ref[name])


def test_small_tokens_and_weights():
    """Hidden values of 1e-9 and less, brought back by the down projection."""
    x, dy = _rand(1, 200, 96, scale=1e-2).to(H), _rand(2, 200, 96, scale=1e-2).to(H)
    w = _weights(96, 256, 96)
    w = [w[0] * 2.0 ** -6, w[1] * 2.0 ** -6, (w[2].float() * 2.0 ** 14).to(H)]
    for act in ("silu", "relu"):
        if act == "relu":  # the sign of a gate near 0 is the oracle's only where the sum is exact
            x, w[0] = (x * 64).round().to(H) / 64, (w[0].float() * 2 ** 12).round().to(H) * 2.0 ** -12
        ref = ob.gated_ffn(x, *w, act, dy)
        for name, t in zip(NAMES, _run(x, w, dy, act)):
            _near(t, ref[name])


def test_tokens_of_different_size():
    """Each token is as exact as it would be by itself, from 2^-8 to 2^8 and with one of 2^12 among them; the sums over tokens
    are exact relative to their norm."""
    M, K, F, N = 260, 96, 256, 80
    g = torch.Generator(device="cuda").manual_seed(3)
    size_x = 2.0 ** torch.randint(-8, 9, (M, 1), generator=g, device="cuda")
    size_dy = 2.0 ** torch.randint(-12, 5, (M, 1), generator=g, device="cuda")
    size_x[7], size_dy[7] = 2.0 ** 12, 2.0 ** -14
    x, dy = (_rand(1, M, K) * size_x).to(H), (_rand(2, M, N) * size_dy).to(H)
    w = _weights(K, F, N, down=2.0 ** -8)
    ref = ob.gated_ffn(x, *w, "silu", dy)
    got = dict(zip(NAMES, _run(x, w, dy, "silu")))
    for name in ("y", "dx"):
        fine = ref[name].abs().amax(1) < 6e4
        assert fine.sum() > 200
        _near(got[name][fine], ref[name][fine], rows=True)
    for name in NAMES[2:]:
        if ref[name].abs().max() < 6e4:
            _near(got[name], ref[name])


@pytest.mark.parametrize("power", [-14, -8, 6])
def test_a_power_of_2_changes_no_rounding(power):
    """Upstream gradients times a power of 2 give the same gradients times it, bit by bit, as far as fp16 holds them."""
    x, w = _rand(1, 500, 72).to(H), _weights(72, 200, 72)
    dy = _rand(2, 500, 72, scale=2.0 ** -2).to(H)
    dy = torch.where(dy.abs() < 2.0 ** -9, torch.zeros_like(dy), dy)   # 11 bits of the rest are left at 2^-24
    base, other = _run(x, w, dy, "gelu"), _run(x, w, (dy.float() * 2.0 ** power).to(H), "gelu")
    exact = (dy.float() * 2.0 ** power).to(H).float() == dy.float() * 2.0 ** power
    if not exact.all():
        dy = torch.where(exact, dy, torch.zeros_like(dy))
        base, other = _run(x, w, dy, "gelu"), _run(x, w, (dy.float() * 2.0 ** power).to(H), "gelu")
    assert torch.equal(base[0], other[0])
    some = 0
    for a, b in zip(base[1:], other[1:]):
        want = a.float() * 2.0 ** power
        held = (want.abs() >= 2.0 ** -14) & (a.float().abs() >= 2.0 ** -14) & (want.abs() < 65504)
        assert torch.equal(b.float()[held], want[held])
        some += int(held.sum())
    assert some > 1000


def test_rows_of_zeros():
    x, w, dy = _rand(1, 300, 96, scale=100).to(H), _weights(96, 256, 96, down=2.0 ** -8), _rand(2, 300, 96, scale=1e-4).to(H)
    x[::3], dy[1::3] = 0, 0
    x[30:60], dy[60:90] = 0, 0
    for act in ("silu", "gelu", "relu"):
        ref = ob.gated_ffn(x, *w, act, dy)
        for name, t in zip(NAMES, _run(x, w, dy, act)):
            assert t.isfinite().all()
            if act != "relu":
                _near(t, ref[name])
    for zero in ((0, 1, 2), (0,), (2,)):
        z = [torch.zeros_like(t) if i in zero else t for i, t in enumerate(w)]
        ref = ob.gated_ffn(x, *z, "silu", dy)
        for name, t in zip(NAMES, _run(x, z, dy, "silu")):
            _near(t, ref[name])
    for t in _run(torch.zeros_like(x), w, dy, "silu") + _run(x, w, torch.zeros_like(dy), "silu")[1:]:
        assert (t == 0).all()


def test_nan_and_infinity_stay_in_their_tokens():
    x, w, dy = _rand(1, 300, 96, scale=100).to(H), _weights(96, 256, 96, down=2.0 ** -8), _rand(2, 300, 96, scale=1e-4).to(H)
    clean = _run(x, w, dy, "silu")
    x[5, 3], x[6, 4], dy[7, 5], dy[8, 6] = float("nan"), float("inf"), float("inf"), float("nan")
    x[9] = float("inf")
    y, dx = _run(x, w, dy, "silu")[:2]
    assert not y[[5, 6, 9]].isfinite().any() and not dx[5:10].isfinite().any()
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[5:10] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert torch.equal(y[7:9], clean[0][7:9])


def test_strides_of_tokens_and_gradients():
    """Rows off the 16-byte boundary and rows that repeat, for the copies that the sums over tokens take."""
    big, up = _rand(1, 140, 200, scale=100).to(H), _rand(2, 140, 90, scale=1e-5).to(H)
    w = _weights(72, 160, 80, down=2.0 ** -8)
    for x, dy in ((big[:, 5:77], up[:, 3:83]), (big[:, 8:80], up[:1, :80].expand(140, 80)), (big.t()[:140, :72], up[:, 8:88])):
        ref = ob.gated_ffn(x, *w, "silu", dy)
        for name, t in zip(NAMES, _run(x, w, dy, "silu")):
            _near(t, ref[name])


def test_network_trains_in_fp16():
    from fused_lncc import tokenreg
    from fused_lncc.registration import identity_grid, make_pair
    torch.manual_seed(0)
    fixed, moving, _ = make_pair(32)
    net = tokenreg.TokenRegistration(width=64, hidden=128, depth=2, dtype=H).cuda()
    losses = tokenreg.train(net, [(fixed, moving)], identity_grid(32, 32, 32, "cuda"), iters=40)
    assert all(v == v for v in losses) and losses[-1] < 0.8 * losses[0], (losses[0], losses[-1])
    assert all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())
