"""CPU: the token-block functions hand tensor subclasses with __torch_function__ to them, as torch's own functions do, and
refuse forward-mode derivatives (on fake tensors that say they are on a GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

import fused_lncc


class Seen(torch.Tensor):
    calls = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.calls.append(str(func))
        return "seen"


@pytest.mark.parametrize("call", [
    lambda x, s: fused_lncc.fused_layer_norm(s), lambda x, s: fused_lncc.fused_layer_norm(x, bias=s),
    lambda x, s: fused_lncc.fused_gated_scan(x, s), lambda x, s: fused_lncc.fused_gated_scan(x, x, s),
    lambda x, s: fused_lncc.fused_gated_ffn(x, x, x, s)])
def test_torch_function_of_any_argument(call):
    x = torch.zeros(2, 8)
    assert call(x, x.clone().as_subclass(Seen)) == "seen"
    assert "fused_lncc" in Seen.calls[-1]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("i", range(10))
def test_tangent_of_any_argument_is_refused(i, requires_grad):
    """A result without a tangent would be taken for one whose tangent is zero."""
    with FakeTensorMode(), fwd.dual_level():
        def tensors(*shapes):
            ts = [torch.zeros(s, device="cuda") for s in shapes]
            ts[0].requires_grad_(requires_grad)
            return ts
        calls = [(fused_lncc.fused_layer_norm, tensors((4, 8), (8,), (8,)))] * 3 \
            + [(fused_lncc.fused_gated_scan, tensors((2, 3, 8), (2, 3, 8), (2, 8)))] * 3 \
            + [(fused_lncc.fused_gated_ffn, tensors((4, 8), (16, 8), (16, 8), (8, 16)))] * 4
        f, args = calls[i]
        args = list(args)
        k = i % 3 if i < 6 else i - 6
        args[k] = fwd.make_dual(args[k], torch.ones_like(args[k]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*args)
