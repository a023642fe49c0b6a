"""GPU: the token-block registration network (fused_lncc/tokenreg.py) against the same network in plain torch, and its
training on the LNCC loss."""
import pytest
import torch
import torch.nn.functional as F

from fused_lncc import tokenreg
from fused_lncc.registration import identity_grid, make_pair

pytestmark = pytest.mark.gpu


def _plain_block(b, u):
    def scan(x, gate):
        a, h, out = torch.sigmoid(gate), torch.zeros_like(x[:, 0]), []
        for t in range(x.shape[1]):
            h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
            out.append(h)
        return torch.stack(out, 1)

    half = u.shape[-1] // 2
    n = F.layer_norm(u, u.shape[-1:], b.norm1.weight, b.norm1.bias, b.norm1.eps)
    x, gate = F.linear(n, b.mix_in.weight, b.mix_in.bias).chunk(2, -1)
    ahead = scan(x[..., :half], gate[..., :half])
    back = scan(x[..., half:].flip(1), gate[..., half:].flip(1)).flip(1)
    u = u + F.linear(torch.cat([ahead, back], -1), b.mix_out.weight, b.mix_out.bias)
    n = F.layer_norm(u, u.shape[-1:], b.norm2.weight, b.norm2.bias, b.norm2.eps)
    return u + F.linear(F.silu(F.linear(n, b.w_gate)) * F.linear(n, b.w_up), b.w_down)


def test_block_matches_plain_torch():
    """fp32 block against the same block in 64 bits: some ten operators deep, 1e-5 of the norms."""
    torch.manual_seed(0)
    block = tokenreg.TokenBlock(48, 120).cuda()
    u = torch.randn(2, 70, 48, device="cuda", requires_grad=True)
    g = torch.randn(2, 70, 48, device="cuda")
    params = list(block.parameters())
    got = block(u)
    grads = torch.autograd.grad(got, [u, *params], g)
    block64 = tokenreg.TokenBlock(48, 120).cuda().double()
    block64.load_state_dict(block.state_dict())
    u64 = u.detach().double().requires_grad_(True)
    want = _plain_block(block64, u64)
    want_grads = torch.autograd.grad(want, [u64, *block64.parameters()], g.double())
    assert (got - want).norm() <= 1e-5 * want.norm()
    for a, b in zip(grads, want_grads):
        assert (a - b).norm() <= 1e-5 * b.norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_lowers_the_loss(dtype):
    torch.manual_seed(0)
    fixed, moving, _ = make_pair(32)
    net = tokenreg.TokenRegistration(width=64, hidden=128, depth=2, dtype=dtype).cuda()
    losses = tokenreg.train(net, [(fixed, moving)], identity_grid(32, 32, 32, "cuda"), iters=40)
    assert all(x == x for x in losses)
    assert losses[-1] < 0.8 * losses[0], (losses[0], losses[-1])
    assert all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())


def test_main_prints_one_line(capsys):
    import json
    tokenreg.main(["--size", "32", "--iters", "4"])
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["tokens"] == 512 and line["ms_per_iter"] > 0
