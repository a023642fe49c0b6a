"""Learned registration on the token blocks: a network over the tokens of a volume, trained on the fused LNCC loss.

registration.py optimises one displacement field for one pair; here a network predicts the field. The moving and the fixed
volume are cut into patches of 4^3 voxels, each patch is a token, and `depth` blocks mix and transform the tokens:

    n = layer norm(u);  u = u + scan of n's projection, forward for one half of the channels and backward for the other
    n = layer norm(u);  u = u + gated feed-forward(n)

(fused_layer_norm, fused_gated_scan, fused_gated_ffn). A linear scan keeps the cost linear in the tokens: 32768 for a 128^3
volume, 107520 for 160 x 192 x 224. A head turns each token into a displacement, which is interpolated to the volume's
resolution, warps the moving volume, and is trained under LNCC + lam * diffusion. The projections in and out
and the head are ordinary torch products.

    python -m fused_lncc.tokenreg --size 64
"""
import argparse
import json

import torch
import torch.nn.functional as F
from torch import nn

from . import fused_gated_ffn, fused_gated_scan, fused_layer_norm, fused_lncc_loss
from .registration import diffusion, identity_grid, make_pair, warp

PATCH = 4


class TokenBlock(nn.Module):
    """One pre-norm block over tokens (B, T, C), C even: two scans in opposite directions, then the gated feed-forward."""

    def __init__(self, width, hidden, activation="silu"):
        super().__init__()
        self.norm1, self.norm2 = nn.LayerNorm(width), nn.LayerNorm(width)  # parameters alone; the kernels read them
        self.mix_in = nn.Linear(width, 2 * width)
        self.mix_out = nn.Linear(width, width)
        with torch.no_grad():  # in either direction gates that remember from a few tokens to some hundreds
            for part in self.mix_in.bias[width:].split([width // 2, width - width // 2]):
                part.copy_(torch.linspace(1.0, 6.0, len(part)))
        self.w_gate = nn.Parameter(torch.randn(hidden, width) * width ** -0.5)
        self.w_up = nn.Parameter(torch.randn(hidden, width) * width ** -0.5)
        self.w_down = nn.Parameter(torch.randn(width, hidden) * hidden ** -0.5 * 0.5)
        self.activation = activation

    def forward(self, u):
        dt, half = u.dtype, u.shape[-1] // 2
        n = fused_layer_norm(u, self.norm1.weight, self.norm1.bias, self.norm1.eps)
        p = F.linear(n, self.mix_in.weight.to(dt), self.mix_in.bias.to(dt))
        x, gate = p.chunk(2, -1)
        ahead, _ = fused_gated_scan(x[..., :half], gate[..., :half])
        back, _ = fused_gated_scan(x[..., half:], gate[..., half:], reverse=True)
        u = u + F.linear(torch.cat([ahead, back], -1), self.mix_out.weight.to(dt), self.mix_out.bias.to(dt))
        n = fused_layer_norm(u, self.norm2.weight, self.norm2.bias, self.norm2.eps)
        return u + fused_gated_ffn(n, self.w_gate.to(dt), self.w_up.to(dt), self.w_down.to(dt), self.activation)


class TokenRegistration(nn.Module):
    """Displacement field (B, 3, D, H, W), in grid_sample's normalised coordinates, of a moving and a fixed volume
    (B, 1, D, H, W) whose sides are multiples of 4. dtype: the tokens' type; parameters and the field are fp32."""

    def __init__(self, width=96, hidden=256, depth=2, dtype=torch.bfloat16):
        super().__init__()
        self.dtype = dtype
        self.embed = nn.Linear(2 * PATCH ** 3, width)
        self.blocks = nn.ModuleList(TokenBlock(width, hidden) for _ in range(depth))
        self.norm = nn.LayerNorm(width)
        self.head = nn.Linear(width, 3)
        nn.init.zeros_(self.head.weight)
        nn.init.zeros_(self.head.bias)

    def forward(self, moving, fixed):
        B, _, D, H, W = moving.shape
        d, h, w = D // PATCH, H // PATCH, W // PATCH
        pair = torch.cat([moving, fixed], 1).reshape(B, 2, d, PATCH, h, PATCH, w, PATCH)
        patches = pair.permute(0, 2, 4, 6, 1, 3, 5, 7).reshape(B, d * h * w, 2 * PATCH ** 3)
        u = F.linear(patches.to(self.dtype), self.embed.weight.to(self.dtype), self.embed.bias.to(self.dtype))
        for block in self.blocks:
            u = block(u)
        n = fused_layer_norm(u, self.norm.weight, self.norm.bias, self.norm.eps)
        field = F.linear(n.float(), self.head.weight, self.head.bias).transpose(1, 2).reshape(B, 3, d, h, w)
        return F.interpolate(field, size=(D, H, W), mode="trilinear", align_corners=True)


def train(net, pairs, base, iters=60, lr=2e-3, lam=0.5, kernel_size=7, opt=None):
    """Adam (or the given optimiser, which goes on from its state) on the network over (fixed, moving) pairs in turn; returns
    the loss of each step."""
    opt = opt or torch.optim.Adam(net.parameters(), lr=lr)
    losses = []
    for i in range(iters):
        fixed, moving = pairs[i % len(pairs)]
        opt.zero_grad(set_to_none=True)
        field = net(moving, fixed)
        loss = fused_lncc_loss(warp(moving, field, base), fixed, kernel_size) + lam * diffusion(field)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).float().cpu().tolist()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--size", type=int, default=64)
    ap.add_argument("--iters", type=int, default=600)
    ap.add_argument("--width", type=int, default=96)
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--depth", type=int, default=2)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    pairs = [make_pair(a.size, seed=s)[:2] for s in range(2)]
    base = identity_grid(a.size, a.size, a.size, "cuda")
    net = TokenRegistration(a.width, a.hidden, a.depth).cuda()
    n = len(pairs)
    # One optimiser throughout: Adam begun anew two steps later left about half of the runs in a poor minimum.
    opt = torch.optim.Adam(net.parameters(), lr=2e-3)
    first = train(net, pairs, base, n, opt=opt)  # one pass over the pairs, which also warms up
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    t0.record()
    losses = train(net, pairs, base, a.iters, opt=opt)
    t1.record()
    torch.cuda.synchronize()
    print(json.dumps({"size": a.size, "tokens": (a.size // PATCH) ** 3, "width": a.width, "depth": a.depth, "iters": a.iters,
                      "loss_first": sum(first) / n, "loss_last": sum(losses[-n:]) / n,
                      "ms_per_iter": t0.elapsed_time(t1) / a.iters}))


if __name__ == "__main__":
    main()
