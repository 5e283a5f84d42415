"""The gated delta rule over many chunks against the 64-bit recurrence: ragged tails, two blocks of value
channels a head, and decays so slow that a state's errors stay for the whole sequence.

The tolerances are those of the shorter sequences (they grow with the square root of the chunks)."""
import pytest
import torch

from oracle.delta import gated_delta, gated_delta_grads
from test_gpu_delta import check_grads, make, off, tol

dev = "cuda"


def slow(a, seed):
    """Log-decays of 0.05 per 64 tokens on average: 0.145 (the mean dt) x 64 x A."""
    g = torch.Generator().manual_seed(seed)
    a["A_log"] = torch.log(1e-3 + 9e-3 * torch.rand(a["A_log"].shape, generator=g))
    return a


def both_ways(ts, a, h0, dtype, L, scale=0.3):
    Bt, _, H, P = a["u"].shape
    N = a["B"].shape[3]
    d, h0d = {k: v.to(dev) for k, v in a.items()}, h0.to(dev)
    args = (d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"])
    ry, rh = gated_delta(**d, scale=scale, h0=h0d)
    ry, rh = ry.cpu(), rh.cpu()
    alone = ts.gated_delta_rule(*args, scale=scale, h0=h0d)
    assert off(alone.view(Bt, L, H, P), ry) < tol(dtype, L)
    y, h, saved = ts.gated_delta_rule(*args, scale=scale, h0=h0d, return_state=True, save=True)
    assert torch.equal(y, alone)
    assert off(h, rh) < tol(torch.float32, L)
    g = torch.Generator().manual_seed(L)
    dy, dh = torch.randn(Bt, L, H, P, generator=g).to(dtype), 0.3 * torch.randn(Bt, H, P, N, generator=g)
    grads = ts.gated_delta_rule_bwd(*args, dy.flatten(2).to(dev), saved, scale=scale, dh_last=dh.to(dev))
    ref = gated_delta_grads(*d.values(), dy.to(dev), scale=scale, h0=h0d, dh_last=dh.to(dev))
    check_grads(grads, [r.cpu() for r in ref], a, dtype, L)


@pytest.mark.gpu
@pytest.mark.parametrize("decay", ["fast", "slow"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,H,G,N,P", [(2, 600, 4, 2, 128, 128), (2, 641, 3, 1, 64, 64), (1, 700, 2, 2, 128, 192),
                                          (1, 577, 2, 1, 64, 192), (1, 590, 2, 2, 48, 80)])
def test_ten_chunks_and_a_tail(cuda_ops, Bt, L, H, G, N, P, dtype, decay):
    a, h0 = make(Bt, L, H, G, N, P, dtype, seed=81)
    both_ways(cuda_ops, slow(a, 82) if decay == "slow" else a, h0, dtype, L)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,P", [(128, 128), (64, 64)])
def test_sixty_four_chunks_that_forget_slowly(cuda_ops, N, P, dtype):
    a, h0 = make(1, 4113, 2, 1, N, P, dtype, seed=83)
    both_ways(cuda_ops, slow(a, 84), h0, dtype, 4113)
