"""GPU: 16-bit feed-forward sums over many tokens that do not cancel. The tensor cores cut what they add to an accumulator: with
two units of its last bit, 2^-23, lost at each addition of 16 products, n tokens in one accumulator come out n / 16 x 2^-23 too
small: 9.8e-4 for 131072 tokens, twice fp16's own rounding. An accumulator takes 2048, 1.5e-5, and the hidden values, sums of
1024, bring 0.8e-5 each: below 6.2e-5 with two of them. Roundings of the hidden values and of the results go either way and vanish
in the mean over a hundred thousand results and more: 1e-6."""
import pytest
import torch

import fused_lncc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_weight_gradients_over_many_tokens(dtype):
    M, K, F, N = 131072, 1024, 2048, 1024     # as many tiles as pairs of SMs: nothing else asks for splits
    g = torch.Generator(device="cuda").manual_seed(0)

    def positive(*shape, low, high):
        return (torch.rand(*shape, generator=g, device="cuda") * (high - low) + low).to(dtype)
    x, dy = positive(M, K, low=0.5, high=1.5), positive(M, N, low=0.5 / 64, high=1.5 / 64)
    wg, wu = positive(F, K, low=0.5 / K, high=1.5 / K), positive(F, K, low=0.5 / K, high=1.5 / K)
    wd = positive(N, F, low=0.5 / N, high=1.5 / N)
    # factors of 1 to 2 for each channel spread the results over octaves, so that their roundings are independent
    for t, axis in ((x, 1), (dy, 1), (wu, 0), (wd, 1)):
        t *= positive(*(n if i == axis else 1 for i, n in enumerate(t.shape)), low=1, high=2)
    leaves = [t.requires_grad_(True) for t in (wg, wu, wd)]
    grads = torch.autograd.grad(fused_lncc.fused_gated_ffn(x, *leaves, activation="relu"), leaves, dy)
    want = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in leaves]
    for i in range(0, M, 16384):
        x64, dy64 = x[i:i + 16384].double(), dy[i:i + 16384].double()
        g64, u64, dh = x64 @ wg.double().T, x64 @ wu.double().T, dy64 @ wd.double()
        want[0] += (dh * u64).T @ x64
        want[1] += (dh * g64).T @ x64
        want[2] += dy64.T @ (g64 * u64)
    for got, w in zip(grads, want):
        bias = (got.double() / w - 1).mean().item()
        assert got.isfinite().all() and abs(bias) <= 6.2e-5, bias
