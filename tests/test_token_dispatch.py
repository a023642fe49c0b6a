"""CPU: the token-block functions hand tensor subclasses with __torch_function__ to them, as torch's own functions do."""
import pytest
import torch

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
