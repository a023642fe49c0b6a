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


def test_main_trains_with_one_optimiser(monkeypatch, capsys):
    """The steps that warm up and those that are timed are one run: Adam's state goes on."""
    seen = []
    monkeypatch.setattr(tokenreg, "make_pair", lambda size, seed: (None, None, None))
    monkeypatch.setattr(tokenreg, "identity_grid", lambda *a: None)
    monkeypatch.setattr(torch.nn.Module, "cuda", lambda self: self)

    class Event:
        def __init__(self, **k):
            pass

        def record(self):
            pass

        def elapsed_time(self, other):
            return 1.0
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    monkeypatch.setattr(tokenreg, "train", lambda net, pairs, base, iters, opt=None: seen.append(opt) or [0.5] * iters)
    tokenreg.main(["--size", "8", "--iters", "4"])
    assert len(seen) == 2 and seen[0] is not None and seen[0] is seen[1]
