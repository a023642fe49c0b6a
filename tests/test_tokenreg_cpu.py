"""CPU: what a token block starts training from."""
import pytest
import torch

from fused_lncc import tokenreg


@pytest.mark.parametrize("width", [8, 9, 96])
def test_both_directions_start_with_the_same_span_of_memories(width):
    """forward() gives the first half of the channels to the scan ahead and the others to the scan back; each has gates from
    sigmoid(1) (memories of 4 tokens) to sigmoid(6) (400)."""
    block = tokenreg.TokenBlock(width, 16)
    gates = block.mix_in.bias.detach()[width:]
    for half in (gates[:width // 2], gates[width // 2:]):
        assert half[0] == 1 and half[-1] == 6 and (half[1:] > half[:-1]).all()
    assert torch.equal(gates[:width // 2], gates[width // 2:]) or width % 2
