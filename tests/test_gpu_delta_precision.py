"""The gated delta rule's bf16 results: their one rounding, and the same bits whatever else the call returns."""
import pytest
import torch

from test_gpu_delta import make

dev = "cuda"


def on(a):
    d = {k: v.to(dev) for k, v in a.items()}
    return d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,H,G,N,P", [(2, 300, 4, 2, 128, 128), (3, 130, 2, 2, 64, 192), (2, 200, 3, 1, 40, 24)])
def test_y_does_not_depend_on_what_else_is_asked_for(cuda_ops, Bt, L, H, G, N, P, dtype):
    a, h0 = make(Bt, L, H, G, N, P, dtype, seed=61)
    args, h0 = on(a), h0.to(dev)
    y = cuda_ops.gated_delta_rule(*args, h0=h0)
    assert torch.equal(cuda_ops.gated_delta_rule(*args, h0=h0, return_state=True)[0], y)
    assert torch.equal(cuda_ops.gated_delta_rule(*args, h0=h0, save=True)[0], y)
