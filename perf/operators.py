"""What is measured of the token-block operators: layer norm, the gated linear recurrence and the gated feed-forward block.

They make up the block of a network that predicts a displacement field from the tokens of a volume and is trained on the
LNCC loss. Token counts come from the volumes of bench.py in 4^3 patches (64^3: 4096 tokens, 128^3: 32768,
160x192x224: 107520); widths are generic.

`run` computes an operator in its plain form (elementary torch operations in fp32, rounded once at the end), or, with
`own`, through fused_lncc. A training pass is the forward and the backward: it returns the output and every gradient.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one token of a streamed sequence through a norm: latency
        {"name": "norm-step", "op": "norm", "rows": 1, "width": 768, "dtype": "bf16", "weight": "bf16", "train": False},
        # a residual stream of a 160x192x224 volume's tokens, weights kept in fp32 as mixed-precision training does
        {"name": "norm-train", "op": "norm", "rows": 107520, "width": 384, "dtype": "bf16", "weight": "fp32", "train": True},
        # fp32 training on a batch whose last tokens were cut off, with an odd width
        {"name": "norm-train-odd", "op": "norm", "rows": 32749, "width": 97, "dtype": "fp32", "weight": "fp32", "train": True},
        # one more token for each of 32 running sequences, from their carried states
        {"name": "scan-step", "op": "scan", "batch": 32, "length": 1, "width": 768, "dtype": "bf16", "state": True,
         "reverse": False, "train": False},
        # inference over 128^3 volumes' tokens
        {"name": "scan-long", "op": "scan", "batch": 2, "length": 32768, "width": 256, "dtype": "fp16", "state": True,
         "reverse": False, "train": False},
        # training over one 160x192x224 volume's tokens, back to front: few channels, the longest axis
        {"name": "scan-train-long", "op": "scan", "batch": 1, "length": 107520, "width": 96, "dtype": "bf16", "state": False,
         "reverse": True, "train": True},
        # fp32 training over a ragged batch of 64^3 volumes' tokens with an odd width
        {"name": "scan-train-odd", "op": "scan", "batch": 6, "length": 4093, "width": 389, "dtype": "fp32", "state": True,
         "reverse": False, "train": True},
        # one token through the block: the weights' bytes and latency
        {"name": "ffn-step", "op": "ffn", "rows": 1, "width": 1024, "hidden": 2816, "dtype": "bf16", "act": "silu", "train": False},
        # inference over a 64^3 volume's tokens
        {"name": "ffn-tokens", "op": "ffn", "rows": 4096, "width": 768, "hidden": 2048, "dtype": "fp16", "act": "gelu", "train": False},
        # training of a narrow network over a 160x192x224 volume's tokens
        {"name": "ffn-train-narrow", "op": "ffn", "rows": 107520, "width": 96, "hidden": 256, "dtype": "bf16", "act": "gelu", "train": True},
        # training of a wide network over a batch: the matrix products' rate
        {"name": "ffn-train-wide", "op": "ffn", "rows": 16384, "width": 1024, "hidden": 4096, "dtype": "bf16", "act": "silu", "train": True},
        # fp32 training at odd sizes
        {"name": "ffn-train-odd", "op": "ffn", "rows": 4093, "width": 389, "hidden": 1037, "dtype": "fp32", "act": "relu", "train": True},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "scan", "ffn"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.6
    if op == "norm":
        while True:
            rows, width = _log(rng, 1, 131072), _log(rng, 16, 8192)
            if rng.random() < 0.5:
                width = max(16, width // 8 * 8)
            if rows * width <= 107520 * 384:
                return {"op": op, "rows": rows, "width": width, "dtype": dtype, "weight": rng.choice([dtype, "fp32"]), "train": train}
    if op == "scan":
        while True:
            batch, length, width = _log(rng, 1, 64), _log(rng, 1, 107520), _log(rng, 16, 2048)
            if rng.random() < 0.5:
                width = max(16, width // 8 * 8)
            if batch * length * width <= 107520 * 96:
                return {"op": op, "batch": batch, "length": length, "width": width, "dtype": dtype,
                        "state": rng.random() < 0.5, "reverse": rng.random() < 0.5, "train": train}
    while True:
        rows, width, ratio = _log(rng, 1, 107520), _log(rng, 32, 1024), rng.uniform(1.0, 4.0)
        hidden = round(width * ratio)
        if rng.random() < 0.5:
            width, hidden = max(32, width // 8 * 8), max(32, hidden // 8 * 8)
        if rows * width * hidden <= 16384 * 1024 * 2048:
            return {"op": op, "rows": rows, "width": width, "hidden": hidden, "dtype": dtype,
                    "act": rng.choice(["silu", "gelu", "relu"]), "train": train}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=DTYPES[case["dtype"]], scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    s = {"case": case}
    train = case["train"]
    if case["op"] == "norm":
        R, C = case["rows"], case["width"]
        wtype = DTYPES[case["weight"]]
        # a residual stream: channels of different scale, rows of different mean
        chan = torch.exp(0.5 * torch.randn(C, generator=gen, device="cuda"))
        s["x"] = (torch.randn(R, C, generator=gen, device="cuda") * chan
                  + 0.5 * torch.randn(R, 1, generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
        s["w"] = normal(C, dtype=wtype, scale=0.1, shift=1.0)
        s["b"] = normal(C, dtype=wtype, scale=0.1)
        s["dy"] = normal(R, C) if train else None
        leaves = ("x", "w", "b")
    elif case["op"] == "scan":
        B, T, C = case["batch"], case["length"], case["width"]
        s["x"] = normal(B, T, C)
        # forget gates that remember some tens of tokens, and now and then a cut between sequences
        gate = torch.randn(B, T, C, generator=gen, device="cuda") * 1.5 + 2.0
        cut = torch.rand(B, T, 1, generator=gen, device="cuda") < 1.0 / 2048
        s["gate"] = gate.masked_fill_(cut, -1e4).to(DTYPES[case["dtype"]])
        s["state"] = normal(B, C, dtype=torch.float32, scale=0.3) if case["state"] else None
        s["dh"] = normal(B, T, C) if train else None
        s["dlast"] = normal(B, C, dtype=torch.float32) if train else None
        leaves = ("x", "gate", "state")
    else:
        M, K, F = case["rows"], case["width"], case["hidden"]
        s["x"] = normal(M, K)
        s["wg"] = normal(F, K, scale=K ** -0.5)
        s["wu"] = normal(F, K, scale=K ** -0.5)
        s["wd"] = normal(K, F, scale=F ** -0.5)
        s["dy"] = normal(M, K) if train else None
        leaves = ("x", "wg", "wu", "wd")
    if train:
        for n in leaves:
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    d = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    n = d * r
    y = (n * w + b).to(s["x"].dtype)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * n).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["b"].dtype)}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0, by doubling the span that each position has summed up."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _plain_scan(s):
    x, gate = s["x"].float(), s["gate"].float()
    if s["case"]["reverse"]:
        x, gate = x.flip(1), gate.flip(1)
    state = torch.zeros_like(x[:, 0]) if s["state"] is None else s["state"]
    a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    b = keep * x
    b = torch.cat([b[:, :1] + a[:, :1] * state[:, None], b[:, 1:]], 1)
    h = _doubling(a, b)

    def out(t):
        return (t.flip(1) if s["case"]["reverse"] else t).to(s["x"].dtype)

    res = {"h": out(h), "last": h[:, -1]}
    if s["dh"] is None:
        return res
    dh = s["dh"].float()
    if s["case"]["reverse"]:
        dh = dh.flip(1)
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dlast"][:, None]], 1)
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    q = _doubling(later.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([state[:, None], h[:, :-1]], 1)
    res["dx"] = out(keep * q)
    res["dgate"] = out(q * (before - x) * a * keep)
    if s["state"] is not None:
        res["dstate"] = a[:, 0] * q[:, 0]
    return res


def _act(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    p = 0.5 * (1 + torch.erf(g * 2 ** -0.5))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_ffn(s):
    t = s["x"].dtype
    x, wg, wu, wd = s["x"].float(), s["wg"].float(), s["wu"].float(), s["wd"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, s["case"]["act"])
    h = a * u
    y = (h @ wd.T).to(t)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return {"y": y, "dx": (dg @ wg + du @ wu).to(t), "dwg": (dg.T @ x).to(t), "dwu": (du.T @ x).to(t), "dwd": (dy.T @ h).to(t)}


# ---------------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------------
def _framework():
    if "fused_lncc" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fused-lncc_b200"))
    import fused_lncc
    return fused_lncc


def _own(s):
    lib, case = _framework(), s["case"]
    if case["op"] == "norm":
        y = lib.fused_layer_norm(s["x"], s["w"], s["b"], EPS)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if case["op"] == "scan":
        h, last = lib.fused_gated_scan(s["x"], s["gate"], state=s["state"], reverse=case["reverse"])
        if not case["train"]:
            return {"h": h, "last": last}
        names = ["x", "gate"] + (["state"] if s["state"] is not None else [])
        grads = torch.autograd.grad((h, last), [s[n] for n in names], (s["dh"], s["dlast"]))
        return {"h": h.detach(), "last": last.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    y = lib.fused_gated_ffn(s["x"], s["wg"], s["wu"], s["wd"], activation=case["act"])
    if not case["train"]:
        return {"y": y}
    dx, dwg, dwu, dwd = torch.autograd.grad(y, (s["x"], s["wg"], s["wu"], s["wd"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dwg": dwg, "dwu": dwu, "dwd": dwd}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "scan": _plain_scan, "ffn": _plain_ffn}[state["case"]["op"]](state)


def work(case):
    """Each input read once and each output written once, and the operations of the formulas."""
    e, train = SIZE[case["dtype"]], case["train"]
    if case["op"] == "norm":
        n, c, we = case["rows"] * case["width"], case["width"], SIZE[case["weight"]]
        return {"bytes": n * e * (4 if train else 2) + c * we * (4 if train else 2), "flops": n * (22 if train else 8)}
    if case["op"] == "scan":
        n, c = case["batch"] * case["length"] * case["width"], case["batch"] * case["width"]
        carried = c * 4 * (1 + case["state"]) * (2 if train else 1)
        return {"bytes": n * e * (6 if train else 3) + carried, "flops": n * (22 if train else 9)}
    m, k, f = case["rows"], case["width"], case["hidden"]
    return {"bytes": e * (m * k * (4 if train else 2) + 3 * f * k * (2 if train else 1)), "flops": 6 * m * k * f * (3 if train else 1)}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_norm(s):
    x, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
    C = x.shape[1]
    mu = torch.einsum("rc->r", x) / C
    var = torch.einsum("rc,rc->r", x, x) / C - mu ** 2
    sigma = torch.sqrt(var + EPS)
    n = (x - mu[:, None]) / sigma[:, None]
    res = {"y": n * w + b}
    if s["dy"] is not None:
        dy = s["dy"].double()
        m1 = torch.einsum("rc,c->r", dy, w) / C
        m2 = torch.einsum("rc,rc,c->r", dy, n, w) / C
        res["dx"] = (dy * w - m1[:, None] - n * m2[:, None]) / sigma[:, None]
        res["dw"] = torch.einsum("rc,rc->c", dy, n)
        res["db"] = torch.einsum("rc->c", dy)
    return res


def _exact_scan(s):
    import numpy as np

    def host(t):  # time first, in the order of the recurrence
        t = t.detach().double().transpose(0, 1).cpu().numpy()
        return t[::-1] if s["case"]["reverse"] else t

    def back(t):
        t = t[::-1] if s["case"]["reverse"] else t
        return torch.from_numpy(np.ascontiguousarray(t)).transpose(0, 1).cuda()

    x, gate = host(s["x"]), host(s["gate"])
    T = x.shape[0]
    with np.errstate(over="ignore"):
        a, keep = 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))
    first = np.zeros_like(x[0]) if s["state"] is None else s["state"].detach().double().cpu().numpy()
    h = np.empty((T + 1,) + x.shape[1:])
    h[0] = first
    for t in range(T):
        h[t + 1] = a[t] * h[t] + keep[t] * x[t]
    res = {"h": back(h[1:]), "last": torch.from_numpy(h[T].copy()).cuda()}
    if s["dh"] is not None:
        dh = host(s["dh"])
        q = np.empty_like(x)
        c = s["dlast"].double().cpu().numpy()
        for t in range(T - 1, -1, -1):
            q[t] = dh[t] + c
            c = a[t] * q[t]
        res["dx"] = back(keep * q)
        res["dgate"] = back(q * (h[:-1] - x) * (a * keep))
        if s["state"] is not None:
            res["dstate"] = torch.from_numpy(c).cuda()
    return res


def _exact_ffn(s):
    x, wg, wu, wd = (s[n].detach().double() for n in ("x", "wg", "wu", "wd"))
    g, u = torch.einsum("mk,fk->mf", x, wg), torch.einsum("mk,fk->mf", x, wu)
    if s["case"]["act"] == "relu":
        a, slope = g.clamp(min=0), (g > 0).double()
    elif s["case"]["act"] == "silu":
        e = 1 / (1 + torch.exp(-g))
        a, slope = g * e, e + g * e * (1 - e)
    else:
        e = 0.5 * torch.erfc(-g / math.sqrt(2))
        a, slope = g * e, e + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    res = {"y": torch.einsum("mf,nf->mn", a * u, wd)}
    if s["dy"] is not None:
        dy = s["dy"].double()
        dh = torch.einsum("mn,nf->mf", dy, wd)
        dg, du = dh * u * slope, dh * a
        res["dx"] = torch.einsum("mf,fk->mk", dg, wg) + torch.einsum("mf,fk->mk", du, wu)
        res["dwg"] = torch.einsum("mf,mk->fk", dg, x)
        res["dwu"] = torch.einsum("mf,mk->fk", du, x)
        res["dwd"] = torch.einsum("mn,mf->nf", dy, a * u)
    return res


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "scan": _exact_scan, "ffn": _exact_ffn}[case["op"]](s)
