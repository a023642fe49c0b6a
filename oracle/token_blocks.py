"""Layer norm, the gated linear recurrence and the gated feed-forward block from their definitions, in 64 bits.

Test infrastructure, on the CPU or the GPU, step by step and without the package's kernels. Each function returns the
results and, given the upstream gradients, every gradient by its formula; `tests/test_token_blocks.py` checks the
gradients against differences. Beside each result stands, under `scale_<name>`, the size of what was summed up to it: a
computation whose every step is off by at most a relative u is off by at most some number of u times that.
"""
import math

import torch


def _d(t):
    return None if t is None else t.detach().double()


def layer_norm(x, weight=None, bias=None, eps=1e-5, dy=None):
    """x (R, C)."""
    x, weight, bias, dy = _d(x), _d(weight), _d(bias), _d(dy)
    w = torch.ones_like(x[0]) if weight is None else weight
    b = torch.zeros_like(x[0]) if bias is None else bias
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    n = (x - mu) * r
    big = r * ((x - mu).abs() + x.abs().mean(1, keepdim=True))  # what n is made of
    out = {"y": n * w + b, "scale_y": big * w.abs() + b.abs()}
    if dy is not None:
        g = dy * w
        out["dx"] = r * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
        out["scale_dx"] = r * (g.abs() + g.abs().mean(1, keepdim=True) + big * (g.abs() * big).mean(1, keepdim=True))
        out["dw"], out["scale_dw"] = (dy * n).sum(0), (dy.abs() * big).sum(0)
        out["db"], out["scale_db"] = dy.sum(0), dy.abs().sum(0)
    return out


def gated_scan(x, gate, state=None, reverse=False, dh=None, dlast=None):
    """x, gate (B, T, C). The scales hold the roundings of every earlier step, faded as the values themselves fade."""
    x, gate, state, dh, dlast = _d(x), _d(gate), _d(state), _d(dh), _d(dlast)
    B, T, C = x.shape
    order = range(T - 1, -1, -1) if reverse else range(T)
    a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    first = x.new_zeros(B, C) if state is None else state
    h, size, err = first, first.abs(), first.abs()
    out = {"h": torch.empty_like(x), "scale_h": torch.empty_like(x)}
    before, err_before = torch.empty_like(x), torch.empty_like(x)
    for t in order:
        before[:, t], err_before[:, t] = h, err
        h = a[:, t] * h + keep[:, t] * x[:, t]
        size = a[:, t] * size + keep[:, t] * x[:, t].abs()
        err = a[:, t] * err + size
        out["h"][:, t], out["scale_h"][:, t] = h, err
    out["last"], out["scale_last"] = h, err
    if dh is not None:
        q = x.new_zeros(B, C) if dlast is None else dlast
        size, err = q.abs(), q.abs()
        for n in ("dx", "dgate"):
            out[n], out["scale_" + n] = torch.empty_like(x), torch.empty_like(x)
        for t in reversed(order):
            q, size = q + dh[:, t], size + dh[:, t].abs()
            err = err + size
            ak = a[:, t] * keep[:, t]
            out["dx"][:, t], out["scale_dx"][:, t] = keep[:, t] * q, keep[:, t] * err
            out["dgate"][:, t] = q * (before[:, t] - x[:, t]) * ak
            out["scale_dgate"][:, t] = ak * (err * (before[:, t].abs() + x[:, t].abs()) + size * err_before[:, t])
            q, size, err = a[:, t] * q, a[:, t] * size, a[:, t] * err
        out["dstate"], out["scale_dstate"] = q, err + size
    return out


def activation(g, act):
    """act(g) and act'(g)."""
    if act == "relu":
        return g.clamp(min=0), (g > 0).to(g.dtype)
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    p = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def gated_ffn(x, w_gate, w_up, w_down, act, dy=None):
    """x (M, K)."""
    x, wg, wu, wd, dy = _d(x), _d(w_gate), _d(w_up), _d(w_down), _d(dy)
    g, u = x @ wg.T, x @ wu.T
    a, slope = activation(g, act)
    out = {"y": (a * u) @ wd.T}
    if dy is not None:
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        out.update(dx=dg @ wg + du @ wu, dw_gate=dg.T @ x, dw_up=du.T @ x, dw_down=dy.T @ (a * u))
    return out
