"""Group norm with an activation, channels last, in 64 bits."""
import torch

__all__ = ["group_norm_act"]


def group_norm_act(x, weight, bias, groups, eps=1e-5, act="silu"):
    """x [Bt,L,C]; weight, bias [C].  Returns y [Bt,L,C] in f64; differentiable."""
    Bt, L, C = x.shape
    xg = x.double().reshape(Bt, L, groups, C // groups)
    mean = xg.mean((1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((xg - mean) / torch.sqrt(var + eps)).reshape(Bt, L, C) * weight.double() + bias.double()
    return z * torch.sigmoid(z) if act == "silu" else z
