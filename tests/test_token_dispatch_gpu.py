"""GPU: whatever stands between an argument of a token-block operator and its memory is honoured, whichever argument it is:
the negative bit, subclasses without memory of their own, vmap, the profiler's records."""
import pytest
import torch
from torch.utils._pytree import tree_map

import fused_lncc

pytestmark = pytest.mark.gpu
ln, scan, ffn = fused_lncc.fused_layer_norm, fused_lncc.fused_gated_scan, fused_lncc.fused_gated_ffn


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


# (function, arguments): results and gradients of each have to be the same however an argument's values are held
CALLS = {
    "norm": (lambda x, w, b: ln(x, w, b), lambda: [_rand(1, 6, 40), _rand(2, 40), _rand(3, 40)]),
    "scan": (lambda x, g, s: scan(x, g, s), lambda: [_rand(1, 2, 30, 24), _rand(2, 2, 30, 24), _rand(3, 2, 24)]),
    "few": (lambda *a: ffn(*a), lambda: [_rand(1, 3, 40), _rand(2, 56, 40), _rand(3, 56, 40), _rand(4, 24, 56)]),
    "ffn": (lambda *a: ffn(*a), lambda: [_rand(1, 30, 40), _rand(2, 56, 40), _rand(3, 56, 40), _rand(4, 24, 56)]),
}
EACH = [(name, i) for name, (_, make) in CALLS.items() for i in range(3 if name in ("norm", "scan") else 4)]


def _outs(r):
    return list(r) if isinstance(r, tuple) else [r]


@pytest.mark.parametrize("name,i", EACH)
def test_negative_bit_of_an_argument(name, i):
    f, make = CALLS[name]
    args = make()
    want = _outs(f(*args))
    args[i] = torch._neg_view(-args[i])
    assert args[i].is_neg()
    for a, b in zip(_outs(f(*args)), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", list(CALLS))
def test_negative_bit_of_upstream_gradients_and_saved_tensors(name):
    f, make = CALLS[name]
    args = [a.requires_grad_(True) for a in make()]
    outs = _outs(f(*args))
    ups = [_rand(9 + i, *o.shape) for i, o in enumerate(outs)]
    want = torch.autograd.grad(outs, args, ups, retain_graph=True)
    for i in range(len(ups)):
        mixed = [torch._neg_view(-u) if i == j else u for j, u in enumerate(ups)]
        for a, b in zip(torch.autograd.grad(outs, args, mixed, retain_graph=True), want):
            assert torch.equal(a, b)
    for i in range(len(args)):  # saved as it was given
        held = [torch._neg_view(-a.detach()).requires_grad_(True) if i == j else a for j, a in enumerate(args)]
        for a, b in zip(torch.autograd.grad(_outs(f(*held)), held, ups), want):
            assert torch.equal(a, b)


class Wrapped(torch.Tensor):
    """A tensor without memory of its own that holds another."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device,
                                                   strides=inner.stride())

    def __init__(self, inner):
        self.inner = inner

    __torch_function__ = torch._C._disabled_torch_function_impl

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        def bare(t):
            return t.inner if isinstance(t, Wrapped) else t
        return func(*tree_map(bare, args), **tree_map(bare, kwargs or {}))


@pytest.mark.parametrize("name,i", EACH)
def test_subclass_without_memory(name, i):
    f, make = CALLS[name]
    args = make()
    want = _outs(f(*args))
    args[i] = Wrapped(args[i])
    for a, b in zip(_outs(f(*args)), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["norm", "scan", "ffn"])
def test_vmap(name):
    f, make = CALLS[name]
    args = make()
    many = [torch.stack([args[0] * k for k in (1, 2, 3)]), *args[1:]]
    got = _outs(torch.vmap(f, in_dims=(0,) + (None,) * (len(args) - 1))(*many))
    for k in range(3):
        for a, b in zip(got, _outs(f(many[0][k], *args[1:]))):
            assert torch.equal(a[k], b)


def test_profiler_sees_the_operators():
    from torch.profiler import ProfilerActivity, profile
    args = CALLS["norm"][1]()
    with profile(activities=[ProfilerActivity.CPU]) as p:
        ln(*args)
    assert any(e.key == "fused_lncc::layer_norm" for e in p.key_averages())


@pytest.mark.parametrize("name", list(CALLS))
def test_under_a_function_mode(name):
    """torch.device as a context is one; gradients come through it as without."""
    f, make = CALLS[name]
    args = [a.requires_grad_(True) for a in make()]
    want = _outs(f(*args))
    want_grads = torch.autograd.grad([o.sum() for o in want], args)
    with torch.device("cuda"):
        got = _outs(f(*args))
        grads = torch.autograd.grad([o.sum() for o in got], args)
    for a, b in zip((*got, *grads), (*want, *want_grads)):
        assert torch.equal(a, b)


def test_torch_func_grad_is_refused():
    x = CALLS["norm"][1]()[0]
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda t: ln(t).sum())(x)
