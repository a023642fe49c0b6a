"""GPU: layer norm, the gated linear recurrence and the gated feed-forward block against the 64-bit oracle.

Tolerances. u32 = 2^-24 and u of the result's type (2^-24, 2^-8, 2^-11) are the relative errors of one rounding. The
oracle gives beside each result the size of what was summed up to it; a result may be off by its own rounding (u), by
`steps` roundings of fp32 of that size, and by half the smallest subnormal of its type. steps counts the roundings on
the longest path: layer norm, sums of 16 in a thread and 5 to 10 in a tree, forward twice (64), backward on top (128), column
sums over at most 300 rows in a row (400); the recurrence, the gate's two roundings of exp and three more, a step and its
composition (16 a step; 16-bit types use the fast exponential, whose error grows by one u32 for each unit of the
gate, |gate| < 24 here where it is not infinite: 40).
The feed-forward block rounds h, dg and du to 16 bits for 16-bit types: with its own rounding a result has two independent
relative errors of at most u and under u/2 in the mean, u of the norm; for fp32 the products carry 24 bits and sums of up to
1100 terms, which wander by some sqrt(1100) u32: 64 u32. A single element may be off by 12 times the root mean square that this gives.
"""
import pytest
import torch

import fused_lncc
from oracle import token_blocks as ob

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}
U32 = 2.0 ** -24


def _rand(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _close(got, ref, name, steps):
    want, size = ref[name], ref["scale_" + name]
    assert got.shape == want.shape, name
    tol = U[got.dtype] * want.abs() + steps * U32 * size + TINY[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= tol * (1 + 2 * U[got.dtype]))
    assert not bad.any(), (name, int(bad.sum()), off.max().item(), (off / tol.clamp(min=1e-300)).max().item())


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------
def _norm_case(rows, width, dtype, wdtype, seed=0, x=None):
    if x is None:
        x = _rand(seed, rows, width, dtype=dtype) * 2 + _rand(seed + 1, rows, 1, dtype=dtype)
    w = _rand(seed + 2, width, dtype=wdtype, scale=0.3, shift=1.0)
    b = _rand(seed + 3, width, dtype=wdtype, scale=0.3)
    dy = _rand(seed + 4, rows, width, dtype=dtype)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = fused_lncc.fused_layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (dtype, dtype, wdtype, wdtype)
    ref = ob.layer_norm(x, w, b, 1e-5, dy)
    _close(y.detach(), ref, "y", 64)
    _close(dx, ref, "dx", 128)
    _close(dw, ref, "dw", 400)
    _close(db, ref, "db", 400)


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 17), (1000, 32), (777, 64), (129, 97), (64, 128), (301, 384),
                                        (33, 513), (70, 768), (9, 1000), (40, 1024), (20, 2048), (7, 3001), (5, 4104),
                                        (6, 8192), (3, 12345), (2, 16384), (4, 16385), (3, 20000)])
def test_norm(rows, width, dtype, wdtype):
    _norm_case(rows, width, dtype, wdtype, seed=rows + width)


def test_norm_many_rows():
    _norm_case(20011, 96, BF16, F32)
    _norm_case(30000, 40, F32, F32)


def test_norm_strides_and_views():
    big = _rand(1, 50, 3, 100, dtype=BF16)
    x = big[:, 1, 4:84]                       # rows 300 apart, not on a 16-byte boundary
    ref = ob.layer_norm(x)
    _close(fused_lncc.fused_layer_norm(x), ref, "y", 64)
    x = big[:, :, :80].transpose(0, 1)        # leading axes that no single stride describes
    y = fused_lncc.fused_layer_norm(x)
    assert y.shape == x.shape
    _close(y.reshape(-1, 80), ob.layer_norm(x.reshape(-1, 80)), "y", 64)
    x = _rand(2, 1, 64).expand(5, 64)         # one row, five times
    _close(fused_lncc.fused_layer_norm(x), ob.layer_norm(x), "y", 64)
    x = _rand(3, 64, 40, dtype=F16).t()       # columns are contiguous
    _close(fused_lncc.fused_layer_norm(x), ob.layer_norm(x), "y", 64)
    x = _rand(4, 12, 48).requires_grad_(True)
    y = fused_lncc.fused_layer_norm(x)
    (dx,) = torch.autograd.grad(y.sum(), x)   # an expanded upstream gradient
    _close(dx, ob.layer_norm(x, dy=torch.ones(12, 48, device="cuda")), "dx", 128)


def test_norm_hard_rows():
    x = _rand(5, 6, 200)
    x[0] = 3.25                               # no variance
    x[1] += 1e4                               # a mean that would cancel in a one-step variance
    x[2] *= 1e-20
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    y = fused_lncc.fused_layer_norm(x)
    ref = ob.layer_norm(x)
    fine = [0, 1, 2, 5]
    _close(y[fine], {k: v[fine] for k, v in ref.items()}, "y", 64)
    assert y[3].isnan().all() and y[4].isnan().all()


def test_norm_empty_and_missing_parts():
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = fused_lncc.fused_layer_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 8) and w.grad.abs().sum() == 0 and x.grad.shape == (0, 8)
    x, w = _rand(6, 10, 24), _rand(7, 24).requires_grad_(True)
    dy = _rand(8, 10, 24)
    ref = ob.layer_norm(x, w, None, 1e-5, dy)
    y = fused_lncc.fused_layer_norm(x, w)     # only the weight's gradient is wanted
    (dw,) = torch.autograd.grad(y, w, dy)
    _close(dw, ref, "dw", 400)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(fused_lncc.fused_layer_norm(x, w.detach()), x, dy)
    _close(dx, ref, "dx", 128)


def test_norm_same_bits_every_time():
    x, dy = _rand(9, 5000, 96, dtype=BF16), _rand(10, 5000, 96, dtype=BF16)
    w = _rand(11, 96).requires_grad_(True)
    runs = [torch.autograd.grad(fused_lncc.fused_layer_norm(x, w), w, dy)[0] for _ in range(4)]
    assert all(torch.equal(r, runs[0]) for r in runs)


def test_norm_past_32_bits():
    rows, width = 2 ** 31 // 1024 + 64, 1024
    x = torch.zeros(rows, width, dtype=F16, device="cuda")
    x[-3:] = _rand(12, 3, width, dtype=F16)
    y = fused_lncc.fused_layer_norm(x)
    _close(y[-3:], ob.layer_norm(x[-3:]), "y", 64)
    assert y[:-3].abs().max() == 0


# ---------------------------------------------------------------------------------------------------------------------
# gated scan
# ---------------------------------------------------------------------------------------------------------------------
STEPS = {F32: 16, BF16: 40, F16: 40}


def _scan_check(x, gate, state, reverse, dh, dlast):
    leaves = [t.requires_grad_(True) for t in (x, gate)] + ([state.requires_grad_(True)] if state is not None else [])
    h, last = fused_lncc.fused_gated_scan(x, gate, state, reverse)
    assert h.dtype == x.dtype and last.dtype == F32
    ref = ob.gated_scan(x, gate, state, reverse, dh, dlast)
    steps = STEPS[x.dtype]
    _close(h.detach(), ref, "h", steps)
    _close(last.detach(), ref, "last", steps)
    grads = torch.autograd.grad((h, last), leaves, (dh, dlast))
    for name, g in zip(("dx", "dgate", "dstate"), grads):
        _close(g, ref, name, steps)
    with torch.no_grad():
        h2, last2 = fused_lncc.fused_gated_scan(x, gate, state, reverse)
    assert torch.equal(h2, h) and torch.equal(last2, last)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (2, 1, 40), (3, 2, 33), (1, 15, 8), (2, 16, 3), (1, 17, 96), (2, 63, 130),
                                   (1, 64, 64), (3, 65, 31), (1, 127, 256), (2, 129, 16), (1, 1000, 24), (2, 1023, 7),
                                   (1, 4097, 66), (5, 300, 97), (1, 9001, 16), (40, 33, 1500),
                                   (2, 20, 80000)])
def test_scan(B, T, C, dtype):
    seed = B + T + C
    reverse = seed % 2 == 0
    state = _rand(seed + 2, B, C) if seed % 3 else None
    _scan_check(_rand(seed, B, T, C, dtype=dtype), _rand(seed + 1, B, T, C, dtype=dtype, scale=2.0, shift=1.5).clamp(-23, 23),
                state, reverse, _rand(seed + 3, B, T, C, dtype=dtype), _rand(seed + 4, B, C))


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_same_bits_every_time(reverse):
    x, gate, dh = (_rand(s, 2, 30000, 40) for s in (1, 2, 3))
    x.requires_grad_(True), gate.requires_grad_(True)

    def run():
        h, last = fused_lncc.fused_gated_scan(x, gate, reverse=reverse)
        return (h, last, *torch.autograd.grad(h, (x, gate), dh))
    first = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_strides(reverse):
    proj = _rand(1, 2, 200, 96, dtype=BF16)
    x, gate = (t.detach() for t in proj.chunk(2, -1))           # two halves of one projection
    dh = _rand(2, 2, 200, 96, dtype=BF16)[:, :, 3:51]
    _scan_check(x, gate, _rand(3, 2, 48), reverse, dh, _rand(4, 2, 48))
    x, gate = _rand(5, 200, 2, 31).transpose(0, 1), _rand(6, 31, 200, 2).permute(2, 1, 0)   # time first; channels strided
    _scan_check(x, gate, None, reverse, _rand(7, 1, 1, 31).expand(2, 200, 31), _rand(8, 2, 31))


def test_scan_extreme_gates():
    B, T, C = 2, 300, 37
    x, gate = _rand(1, B, T, C), _rand(2, B, T, C)
    gate[:, 10:150, ::3] = float("inf")       # padding: the state is kept
    gate[0, 170] = float("-inf")              # a cut: the state is dropped
    gate[1, 200:202] = torch.finfo(F32).min
    gate[1, 230:240] = torch.finfo(F32).max
    gate[0, 250] = -1e4
    _scan_check(x, gate, _rand(3, B, C), False, _rand(4, B, T, C), _rand(5, B, C))
    all_kept = torch.full((B, T, C), float("inf"), device="cuda")
    state = _rand(6, B, C)
    h, last = fused_lncc.fused_gated_scan(x.detach(), all_kept, state)
    assert torch.equal(last, state) and torch.equal(h, state[:, None].expand(B, T, C))
    all_cut = torch.full((B, T, C), float("-inf"), device="cuda")
    h, _ = fused_lncc.fused_gated_scan(x.detach(), all_cut, state)
    assert torch.equal(h, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_nan_stays_in_its_channel_and_after_its_step(dtype):
    x, gate = _rand(1, 1, 500, 40, dtype=dtype), _rand(2, 1, 500, 40, dtype=dtype)
    clean, _ = fused_lncc.fused_gated_scan(x, gate)
    x[0, 333, 5] = float("nan")
    gate[0, 123, 6] = float("nan")
    h, last = fused_lncc.fused_gated_scan(x, gate)
    hit = torch.zeros(500, 40, dtype=torch.bool, device="cuda")
    hit[333:, 5] = True
    hit[123:, 6] = True
    assert h[0][hit].isnan().all() and torch.equal(h[0][~hit], clean[0][~hit])
    assert last[0].isnan().sum() == 2


def test_scan_empty():
    state = _rand(1, 2, 5).requires_grad_(True)
    x = torch.empty(2, 0, 5, device="cuda")
    h, last = fused_lncc.fused_gated_scan(x, x, state)
    assert h.shape == (2, 0, 5) and torch.equal(last, state)
    g = _rand(2, 2, 5)
    assert torch.equal(torch.autograd.grad(last, state, g)[0], g)
    _, last = fused_lncc.fused_gated_scan(x, x)
    assert last.abs().sum() == 0
    h, last = fused_lncc.fused_gated_scan(torch.empty(0, 3, 5, device="cuda"), torch.empty(0, 3, 5, device="cuda"))
    assert h.shape == (0, 3, 5) and last.shape == (0, 5)


def test_scan_in_pieces_and_token_by_token():
    B, T, C = 2, 90, 24
    x, gate, state = _rand(1, B, T, C), _rand(2, B, T, C), _rand(3, B, C)
    ref = ob.gated_scan(x, gate, state)
    s, parts = state, []
    for a, b in ((0, 40), (40, 41), (41, 90)):
        h, s = fused_lncc.fused_gated_scan(x[:, a:b], gate[:, a:b], s)
        parts.append(h)
    _close(torch.cat(parts, 1), ref, "h", 16)
    s, parts = state, []
    for t in range(T):
        h, s = fused_lncc.fused_gated_scan(x[:, t:t + 1], gate[:, t:t + 1], s)
        parts.append(h)
    _close(torch.cat(parts, 1), ref, "h", 16)
    _close(s, ref, "last", 16)


def test_scan_gradient_of_last_only():
    B, T, C = 2, 77, 12
    x, gate, dlast = _rand(1, B, T, C).requires_grad_(True), _rand(2, B, T, C).requires_grad_(True), _rand(3, B, C)
    _, last = fused_lncc.fused_gated_scan(x, gate)
    dx, dgate = torch.autograd.grad(last, (x, gate), dlast)
    ref = ob.gated_scan(x, gate, dh=torch.zeros_like(x), dlast=dlast)
    _close(dx, ref, "dx", 16)
    _close(dgate, ref, "dgate", 16)


def test_scan_past_32_bits():
    B, T, C = 3, 1500, 2 ** 19
    x = torch.zeros(B, T, C, dtype=BF16, device="cuda")
    gate = torch.zeros(B, T, C, dtype=BF16, device="cuda")
    x[-1, -40:, -8:] = _rand(1, 40, 8, dtype=BF16)
    h, last = fused_lncc.fused_gated_scan(x, gate)
    ref = ob.gated_scan(x[-1:, -40:, -8:], gate[-1:, -40:, -8:])
    _close(h[-1:, -40:, -8:], ref, "h", 40)
    _close(last[-1:, -8:], ref, "last", 40)
    assert h[0].abs().max() == 0


def test_scan_past_32_bits_along_time():
    T, C = 2 ** 22, 520   # few channels: T is cut, and the last tiles lie past 2^31 elements
    x = torch.zeros(1, T, C, dtype=BF16, device="cuda")
    gate = torch.zeros(1, T, C, dtype=BF16, device="cuda")
    x[0, -40:, -8:] = _rand(1, 40, 8, dtype=BF16)
    h, last = fused_lncc.fused_gated_scan(x, gate)
    ref = ob.gated_scan(x[:, -40:, -8:], gate[:, -40:, -8:])
    _close(h[:, -40:, -8:], ref, "h", 40)
    _close(last[:, -8:], ref, "last", 40)
    assert h[0, :-40].abs().max() == 0
    h, last = fused_lncc.fused_gated_scan(x, gate, reverse=True)
    ref = ob.gated_scan(x[:, -40:, -8:], gate[:, -40:, -8:], reverse=True)
    _close(h[:, -40:, -8:], ref, "h", 40)


# ---------------------------------------------------------------------------------------------------------------------
# gated feed-forward
# ---------------------------------------------------------------------------------------------------------------------
def _near(got, want, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    off, tol = got.double() - want, 64 * U32 if dtype == F32 else U[dtype]
    rms = want.norm() / max(1, want.numel()) ** 0.5
    assert off.norm() <= tol * want.norm() + TINY[dtype] * want.numel() ** 0.5, (off.norm() / want.norm()).item()
    assert (off.abs() <= 12 * tol * torch.maximum(rms, want.abs()) + 12 * TINY[dtype]).all()


def _ffn_check(x, wg, wu, wd, act, dy):
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = fused_lncc.fused_gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = ob.gated_ffn(x, wg, wu, wd, act, dy)
    _near(y.detach(), ref["y"], x.dtype)
    for name, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), grads):
        _near(g, ref[name], x.dtype)
    with torch.no_grad():
        assert torch.equal(fused_lncc.fused_gated_ffn(*leaves, activation=act), y)


def _ffn_tensors(M, K, F, N, dtype, seed, act="silu"):
    if act == "relu":  # small whole numbers: g is exact in fp32, so its sign is the oracle's, zeros among them
        g = torch.Generator(device="cuda").manual_seed(seed)
        x, wg = (torch.randint(-2, 3, s, generator=g, device="cuda").to(dtype) for s in ((M, K), (F, K)))
    else:
        x, wg = _rand(seed, M, K, dtype=dtype), _rand(seed + 1, F, K, dtype=dtype, scale=K ** -0.5)
    return (x, wg, _rand(seed + 2, F, K, dtype=dtype, scale=K ** -0.5), _rand(seed + 3, N, F, dtype=dtype, scale=F ** -0.5),
            _rand(seed + 4, M, N, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,F,N,act", [
    (1, 64, 128, 64, "silu"), (1, 33, 51, 27, "gelu"), (2, 256, 512, 256, "relu"), (5, 96, 264, 96, "silu"),
    (8, 128, 384, 128, "gelu"), (4, 1024, 2816, 1024, "silu"), (3, 1000, 3001, 500, "silu"), (8, 2040, 1024, 96, "gelu"), (9, 200, 504, 200, "silu"), (16, 1024, 640, 72, "silu"), (17, 40, 1001, 8, "gelu"),
    (63, 96, 256, 96, "gelu"), (127, 64, 64, 64, "silu"), (128, 128, 128, 128, "relu"), (129, 136, 200, 136, "silu"),
    (300, 389, 1037, 389, "gelu"), (1000, 96, 256, 96, "gelu"), (513, 768, 1000, 768, "silu"), (700, 8, 16, 1000, "relu"),
    (2049, 72, 88, 104, "silu"), (260, 520, 260, 515, "silu")])
def test_ffn(M, K, F, N, act, dtype):
    x, wg, wu, wd, dy = _ffn_tensors(M, K, F, N, dtype, M + K + F, act)
    _ffn_check(x, wg, wu, wd, act, dy)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ffn_strides(dtype):
    _, wg, wu, wd, _ = _ffn_tensors(1, 72, 160, 80, dtype, 3)
    big, up = _rand(1, 140, 200, dtype=dtype), _rand(2, 140, 3, 81, dtype=dtype)
    _ffn_check(big[:, 5:77], wg, wu, wd, "silu", up[:, 1, :80])          # rows off the 16-byte boundary
    _ffn_check(big[:, 8:80], wg, wu, wd, "silu", up[:, 1, 1:])
    packed = _rand(4, 320, 72, dtype=dtype)
    _ffn_check(big.t()[:140, :72], *(w.detach() for w in packed.chunk(2)), wd.t().contiguous().t(), "gelu",
               _rand(5, 1, 80, dtype=dtype).expand(140, 80))
    x = _rand(6, 4, 5, 7, 72, dtype=dtype)
    y = fused_lncc.fused_gated_ffn(x, wg, wu, wd)
    assert y.shape == (4, 5, 7, 80)
    _near(y.reshape(-1, 80).detach(), ob.gated_ffn(x.reshape(-1, 72), wg, wu, wd, "silu")["y"], dtype)


@pytest.mark.parametrize("M", [4, 200])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_ffn_nan_stays_in_its_token(M, dtype):
    x, wg, wu, wd, _ = _ffn_tensors(M, 64, 96, 64, dtype, 9)
    clean = fused_lncc.fused_gated_ffn(x, wg, wu, wd)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = fused_lncc.fused_gated_ffn(x, wg, wu, wd)
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    assert torch.equal(y[keep], clean[keep]) and y[1].isnan().all() and not y[2].isfinite().any()


def test_ffn_large_activations():
    # gates of some hundreds: silu's exponential overflows on one side and vanishes on the other
    x, wg, wu, wd, dy = _ffn_tensors(200, 64, 96, 64, F32, 11)
    for act in ("silu", "gelu"):
        _ffn_check((x.detach() * 300), wg.detach(), wu.detach(), wd.detach(), act, dy)


def test_ffn_empty_and_some_gradients():
    x, wg, wu, wd, dy = _ffn_tensors(0, 16, 24, 16, BF16, 1)
    for t in (x, wg, wu, wd):
        t.requires_grad_(True)
    y = fused_lncc.fused_gated_ffn(x, wg, wu, wd)
    y.sum().backward()
    assert y.shape == (0, 16) and all(t.grad.abs().sum() == 0 for t in (wg, wu, wd))
    x, wg, wu, wd, dy = _ffn_tensors(150, 64, 96, 64, BF16, 2)
    ref = ob.gated_ffn(x, wg, wu, wd, "silu", dy)
    for i, name in enumerate(("dx", "dw_gate", "dw_up", "dw_down")):
        args = [t.detach().clone() for t in (x, wg, wu, wd)]
        args[i].requires_grad_(True)
        (g,) = torch.autograd.grad(fused_lncc.fused_gated_ffn(*args), args[i], dy)
        _near(g, ref[name], BF16)


def test_ffn_past_32_bits():
    M, K, F, N = 2 ** 31 // 2048 + 300, 16, 2048, 24   # the hidden matrices pass 2^31 elements
    x, dy = torch.zeros(M, K, dtype=BF16, device="cuda"), torch.zeros(M, N, dtype=BF16, device="cuda")
    x[-200:], dy[-200:] = _rand(1, 200, K, dtype=BF16), _rand(2, 200, N, dtype=BF16)
    _, wg, wu, wd, _ = _ffn_tensors(1, K, F, N, BF16, 3)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = fused_lncc.fused_gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = ob.gated_ffn(x[-200:], wg, wu, wd, "silu", dy[-200:])
    _near(y[-200:].detach(), ref["y"], BF16)
    _near(grads[0][-200:], ref["dx"], BF16)
    for name, g in zip(("dw_gate", "dw_up", "dw_down"), grads[1:]):
        _near(g, ref[name], BF16)
    assert y[:-200].abs().max() == 0 and grads[0][:-200].abs().max() == 0


def test_ffn_one_matrix_for_gate_and_up():
    x, wg, _, wd, dy = _ffn_tensors(140, 64, 96, 64, F32, 21)
    wg.requires_grad_(True)
    (g,) = torch.autograd.grad(fused_lncc.fused_gated_ffn(x, wg, wg, wd), wg, dy)
    ref = ob.gated_ffn(x, wg, wg, wd, "silu", dy)
    _near(g, ref["dw_gate"] + ref["dw_up"], F32)


def test_ffn_relu_gates_at_zero():
    """fp32 gates that are exactly 0, or closer to 0 than any order of summation can tell: the derivative there is that of the
    plain sum in the order of k, and an exact 0 has derivative 0."""
    M, K, F = 130, 300, 72
    x, wg = _rand(1, M, K), _rand(2, F, K)
    x[:, K // 2:], wg[:, K // 2:] = x[:, :K // 2], -wg[:, :K // 2]      # every gate is 0 up to rounding
    x[5] = 0
    _, _, wu, wd, dy = _ffn_tensors(M, K, F, 64, F32, 4)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(fused_lncc.fused_gated_ffn(x, wg, wu, wd, "relu"), x, dy)
    xs, ws = x.detach().cpu(), wg.cpu()
    # a multiply-add rounds once: the sum of products in 64 bits, rounded to fp32 after each (their products are exact there)
    g = torch.zeros(M, F, dtype=torch.float64)
    for k in range(K):
        g = (g + xs[:, k, None].double() * ws[None, :, k].double()).float().double()
    on = (g > 0).double().cuda()
    assert 0 < on.mean() < 1
    x64, g64 = x.detach().double(), g.cuda()
    dh = dy.double() @ wd.double()
    want = (dh * (x64 @ wu.double().T) * on) @ wg.double() + (dh * g64.clamp(min=0)) @ wu.double()
    _near(dx, want, F32)
    assert dx[5].isfinite().all()


def test_ffn_same_bits_every_time():
    x, wg, wu, wd, dy = _ffn_tensors(3000, 96, 160, 96, BF16, 5)
    wg.requires_grad_(True), wd.requires_grad_(True)
    runs = [torch.autograd.grad(fused_lncc.fused_gated_ffn(x, wg, wu, wd), (wg, wd), dy) for _ in range(4)]
    assert all(torch.equal(a, b) for r in runs for a, b in zip(r, runs[0]))


# ---------------------------------------------------------------------------------------------------------------------
# all of them
# ---------------------------------------------------------------------------------------------------------------------
def test_gradients_against_differences():
    """fp32 forward passes a step of 2^-6 apart against <gradient, direction>: the differences' own error is step^2 of
    the third derivative and u32 / step of the values' sum, together below 1e-3 of the sums' norms."""
    eps = 2.0 ** -6

    def check(f, args, dy):
        args = [a.requires_grad_(True) for a in args]
        grads = torch.autograd.grad(f(*args), args, dy)
        for i, g in enumerate(grads):
            v = _rand(50 + i, *args[i].shape) / args[i].numel() ** 0.5
            with torch.no_grad():
                up, down = list(args), list(args)
                up[i], down[i] = args[i] + eps * v, args[i] - eps * v
                diff = ((f(*up).double() - f(*down).double()) * dy.double()).sum() / (2 * eps)
            assert abs(diff - (g.double() * v.double()).sum()) <= 1e-3 * g.double().norm(), i

    check(lambda x, w, b: fused_lncc.fused_layer_norm(x, w, b), [_rand(1, 40, 96), _rand(2, 96), _rand(3, 96)], _rand(4, 40, 96))
    check(lambda x, g, s: fused_lncc.fused_gated_scan(x, g, s)[0], [_rand(1, 2, 200, 24), _rand(2, 2, 200, 24), _rand(3, 2, 24)],
          _rand(4, 2, 200, 24))
    for act in ("silu", "gelu"):
        check(lambda *a: fused_lncc.fused_gated_ffn(*a, activation=act),
              [_rand(1, 150, 64), _rand(2, 96, 64, scale=0.125), _rand(3, 96, 64, scale=0.125), _rand(4, 64, 96, scale=0.1)],
              _rand(5, 150, 64))


def _block(x, w, b, gates, wg, wu, wd):
    n = fused_lncc.fused_layer_norm(x, w, b)
    h, _ = fused_lncc.fused_gated_scan(n, gates)
    return x + h + fused_lncc.fused_gated_ffn(h, wg, wu, wd)


def _block_args(dtype=BF16):
    return (_rand(1, 2, 300, 96, dtype=dtype), _rand(2, 96, dtype=dtype), _rand(3, 96, dtype=dtype),
            _rand(4, 2, 300, 96, dtype=dtype), _rand(5, 256, 96, dtype=dtype, scale=0.1),
            _rand(6, 256, 96, dtype=dtype, scale=0.1), _rand(7, 96, 256, dtype=dtype, scale=0.06))


def test_other_stream():
    want = _block(*_block_args())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        args = _block_args()
        for a in args:
            a.requires_grad_(True)
        got = _block(*args)
        grads = torch.autograd.grad(got.float().square().sum(), args)
    s.synchronize()
    assert torch.equal(got, want)
    args2 = [a.detach().clone().requires_grad_(True) for a in args]
    for g, w in zip(grads, torch.autograd.grad(_block(*args2).float().square().sum(), args2)):
        assert torch.equal(g, w)


def test_graph_replay():
    args = _block_args()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            _block(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _block(*args)
    fresh = _rand(99, 2, 300, 96, dtype=BF16)
    args[0].copy_(fresh)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, _block(fresh, *args[1:]))


def test_compile_fullgraph():
    args = [a.requires_grad_(True) for a in _block_args(F32)]
    want = _block(*args)
    want_grads = torch.autograd.grad(want.square().sum(), args)
    got = torch.compile(_block, fullgraph=True)(*args)
    grads = torch.autograd.grad(got.square().sum(), args)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
    for g, w in zip(grads, want_grads):
        assert (g - w).norm() <= 1e-5 * w.norm()


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(16, 8, device="cuda")
    d = torch.zeros(8, 16, device="cuda")
    ln, scan, ffn = fused_lncc.fused_layer_norm, fused_lncc.fused_gated_scan, fused_lncc.fused_gated_ffn
    for call in (lambda: ln(x.double()), lambda: ln(x, torch.zeros(7, device="cuda")), lambda: ln(x, torch.zeros(8)),
                 lambda: ln(x, torch.zeros(8, device="cuda", dtype=BF16)), lambda: ln(torch.zeros(3, 0, device="cuda")),
                 lambda: ln(x.half(), torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda", dtype=F16)),
                 lambda: scan(x, x), lambda: scan(x[None], x[None].half()), lambda: scan(x[None], x[None, :3]),
                 lambda: scan(x[None], x[None], torch.zeros(2, 8, device="cuda")), lambda: scan(x[None], x[None].cpu()),
                 lambda: ffn(x, w, w, w), lambda: ffn(x, w, w[:8], d), lambda: ffn(x.half(), w, w, d),
                 lambda: ffn(x, w, w, d.cpu()), lambda: ffn(x[:, :4], w, w, d), lambda: ffn(x, w[0], w, d)):
        with pytest.raises(RuntimeError, match="fused_lncc"):
            call()
