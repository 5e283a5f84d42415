"""Group norm where a call has nothing to normalise."""
import pytest
import torch

dev = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 4, 0), (5, 0), (2, 0, 0)])
def test_statistics_of_no_channels(cuda_ops, shape):
    """A group without values has mean 0 and variance 0, whatever its buffers held."""
    keep = [torch.full((1 << 10,), 7.0, device=dev) for _ in range(64)]
    del keep
    x, w = torch.empty(shape, device=dev), torch.empty(0, device=dev)
    y, mean, rstd = cuda_ops.group_norm_act(x, w, w, 2, eps=0.25, return_stats=True)
    assert y.shape == x.shape and mean.shape == (shape[0], 2)
    assert not mean.any() and bool((rstd == 2.0).all())
    dx, dw, db = cuda_ops.group_norm_act_bwd(x, x, w, w, mean, rstd)
    assert dx.shape == x.shape and dw.numel() == 0 and db.numel() == 0
