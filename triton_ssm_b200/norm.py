"""Group norm with an activation, channels last (forward and backward).

It normalises the channels-last outputs of the scans: per token and head
(a [rows, C] tensor, ``groups`` = heads), or over a whole feature map
([Bt, L, C]).  Same conventions as ``ops.py``: bad arguments raise
``ValueError``, outputs are new tensors, the kernel runs on the current stream
of the inputs' device.
"""
import torch

from . import _lib
from ._lib import addr, call, dtype_code, on_device, raw_stream, same_device
from .ops import _need

__all__ = ["group_norm_act", "group_norm_act_bwd"]

_ACT = {"none": 0, "silu": 1}


def _norm_args(name, x, weight, bias, groups, act):
    _need(x, (torch.float32, torch.bfloat16), "x")
    _need(weight, (torch.float32,), "weight")
    _need(bias, (torch.float32,), "bias")
    if x.dim() not in (2, 3):
        raise ValueError("%s: expected x [Bt,L,C] or [rows,C]" % name)
    C = x.shape[-1]
    if weight.shape != (C,) or bias.shape != (C,):
        raise ValueError("%s: weight and bias must be [C]" % name)
    if groups < 1 or C % groups:
        raise ValueError("%s: C (%d) must be a multiple of groups (%d)" % (name, C, groups))
    if act not in _ACT:
        raise ValueError("%s: act must be 'silu' or 'none' (got %r)" % (name, act))
    return x.shape[0], (x.shape[1] if x.dim() == 3 else 1), C


def _workspace(x, Bt, L, C, groups, backward):
    need = int(_lib.load_library().tssm_group_norm_workspace_size(Bt, L, C, groups, dtype_code(x), int(backward)))
    return torch.empty(need, dtype=torch.uint8, device=x.device) if need else None, need


def group_norm_act(x, weight, bias, groups, eps=1e-5, act="silu", return_stats=False, y=None):
    """Group norm over channels-last x, then the activation:
    y = act((x - mean) / sqrt(var + eps) * weight + bias).

    x [Bt,L,C] (mean and variance per batch row and group, over L and the
    C/groups channels) or [rows,C] (per row and group, the head norm of single
    tokens); f32 or bf16.  weight, bias [C] f32; act "silu" or "none".
    Returns y in x's dtype, or (y, mean, rstd) with the statistics
    [Bt,groups] f32 when ``return_stats`` (the backward takes them).
    """
    dev = same_device(x, weight, bias, y)
    groups, eps = int(groups), float(eps)
    if not eps >= 0:
        raise ValueError("group_norm_act: eps must not be negative (got %r)" % eps)
    Bt, L, C = _norm_args("group_norm_act", x, weight, bias, groups, act)
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    if y is None:
        y = torch.empty_like(x)
    elif y.shape != x.shape or y.dtype != x.dtype or not y.is_contiguous():
        raise ValueError("group_norm_act: y must be contiguous and match x")
    mean = rstd = ws = None
    need = 0
    narrow = L == 1 and C // groups <= 128   # needs neither statistics nor workspace
    if return_stats or not narrow:
        mean, rstd = torch.empty(2, Bt, groups, device=x.device, dtype=torch.float32)
        if L == 0 or C == 0:
            mean.zero_()
            rstd.fill_(eps ** -0.5 if eps else float("inf"))
    if not narrow:
        ws, need = _workspace(x, Bt, L, C, groups, False)
    with on_device(dev):
        call("tssm_group_norm_act", addr(x), addr(weight), addr(bias), addr(y), addr(mean), addr(rstd), addr(ws), need, Bt, L,
             C, groups, eps, _ACT[act], dtype_code(x), raw_stream(dev))
    return (y, mean, rstd) if return_stats else y


def group_norm_act_bwd(dy, x, weight, bias, mean, rstd, act="silu"):
    """Backward of ``group_norm_act``.

    dy, x [Bt,L,C] or [rows,C] (one dtype); weight, bias [C] f32; mean, rstd
    [Bt,groups] f32 from the forward.  Returns (dx in x's dtype, dweight [C],
    dbias [C] f32); the sums over rows run in a fixed order.
    """
    dev = same_device(x, dy, weight, bias, mean, rstd)
    if mean.dim() != 2 or mean.shape != rstd.shape or mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        raise ValueError("group_norm_act_bwd: mean and rstd must be [Bt,groups] f32")
    groups = mean.shape[1]
    Bt, L, C = _norm_args("group_norm_act_bwd", x, weight, bias, groups, act)
    if dy.shape != x.shape or dy.dtype != x.dtype or mean.shape[0] != Bt:
        raise ValueError("group_norm_act_bwd: dy must match x, and mean and rstd its batch rows")
    dy, x, weight, bias, mean, rstd = (t.contiguous() for t in (dy, x, weight, bias, mean, rstd))
    dx = torch.empty_like(x)
    dw, db = torch.empty(2, C, device=x.device, dtype=torch.float32)
    ws, need = _workspace(x, Bt, L, C, groups, True)
    with on_device(dev):
        call("tssm_group_norm_act_bwd", addr(dy), addr(x), addr(weight), addr(bias), addr(mean), addr(rstd), addr(dx),
             addr(dw), addr(db), addr(ws), need, Bt, L, C, groups, _ACT[act], dtype_code(x), raw_stream(dev))
    return dx, dw, db
