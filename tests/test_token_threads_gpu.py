"""GPU: a token-block call that is the first use of the device by its thread, with all memory from torch's cache."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import fused_lncc

pytestmark = pytest.mark.gpu
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fused-lncc_b200")


def _args(M, dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    return [torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((M, 64), (128, 64), (128, 64), (128, 128))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M", [4, 8, 200])
def test_first_call_of_a_thread(M, dtype):
    args = _args(M, dtype)
    want = fused_lncc.fused_gated_ffn(*args)
    spare = [torch.empty(1 << 20, device="cuda") for _ in range(8)]  # memory for the thread, in the cache
    torch.cuda.synchronize()
    del spare
    got = []

    def work():
        try:
            got.append(fused_lncc.fused_gated_ffn(*args))
        except RuntimeError as e:
            got.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert torch.is_tensor(got[0]), got[0]
    assert torch.equal(got[0], want)


def test_first_backward_of_a_process():
    """Autograd's thread makes its first call on the device in the feed-forward block's backward pass."""
    code = f"""
import sys, torch
sys.path.insert(0, {PKG!r})
from fused_lncc import fused_gated_ffn
args = [torch.randn(*s, device="cuda").half().requires_grad_(True) for s in ((8, 64), (128, 64), (128, 64), (128, 128))]
y = fused_gated_ffn(*args)
up = torch.ones_like(y)
spare = [torch.empty(1 << 20, device="cuda") for _ in range(8)]
torch.cuda.synchronize()
del spare
g = torch.autograd.grad(y, args, up)
torch.cuda.synchronize()
assert all(t.isfinite().all() for t in g)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_first_calls_of_many_threads_at_once():
    """The library's marks of what a device was asked for are set by any thread, here by sixteen that start together, each on a
    stream of its own, with kernels that no other test has to have run before."""
    def work(i):
        g = torch.Generator(device="cuda").manual_seed(i % 4)
        x = torch.randn(33 + i % 4, 1000 + 8 * (i % 4), generator=g, device="cuda").half()
        w = [torch.randn(*s, generator=g, device="cuda").half() * 0.03 for s in ((96, x.shape[1]), (96, x.shape[1]), (64, 96))]
        y = fused_lncc.fused_layer_norm(x)
        return fused_lncc.fused_gated_ffn(y, *w, activation=("silu", "gelu", "relu")[i % 3])
    got, start = [None] * 16, threading.Barrier(16)

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            got[i] = work(i)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(16)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(16):
        assert torch.equal(got[i], work(i)), i
