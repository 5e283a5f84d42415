"""The gated delta rule: whole sequences, their backward, and single tokens.

Per head, with state h [P,N], value u_t [P], key B_t [N], query C_t [N], step
dt_t and write strength beta_t:

    hd  = exp(-exp(A_log) dt_t) h_{t-1}
    h_t = hd + beta_t (u_t - hd B_t) B_t^T ,   y_t = scale * h_t C_t

the scan of ``multihead_ssm`` (same decay, state layout and argument names)
with a write that corrects what the state already predicts.  Keys are usually
unit vectors and beta in [0, 1], which keeps the state bounded; neither is
required.  A token with dt = 0 and beta = 0 leaves the state as it was
(padding).  B and C may have fewer heads than u: G key heads, head i reading
key head i // (H // G).
"""
import torch

from ._lib import call, device_of, dtype_code, ptr, stream_of
from .ops import _cuda, _need

__all__ = ["gated_delta_step"]


def gated_delta_step(x, dt, h, A_log, B, C, beta, scale=1.0, y=None):
    """One token of every stream; the state is updated in place.

    x [S,H,P] f32 or bf16; dt, beta [S,H] f32; h [S,H,P,N] f32; A_log [H] f32;
    B, C [S,G,N] in x's dtype, H a multiple of G, N <= 256.  Returns y [S,H,P]
    in x's dtype.
    """
    _cuda(x, dt, h, A_log, B, C, beta, y)
    _need(x, (torch.float32, torch.bfloat16), "x")
    _need(h, (torch.float32,), "h")
    if x.dim() != 3 or h.dim() != 4 or B.dim() != 3:
        raise ValueError("gated_delta_step: expected x [S,H,P], h [S,H,P,N], B, C [S,G,N]")
    S, H, P = x.shape
    G, N = B.shape[1], h.shape[3]
    if tuple(h.shape) != (S, H, P, N) or tuple(B.shape) != (S, G, N) or C.shape != B.shape or \
            tuple(dt.shape) != (S, H) or tuple(beta.shape) != (S, H) or tuple(A_log.shape) != (H,):
        raise ValueError("gated_delta_step: shape mismatch")
    if B.dtype != x.dtype or C.dtype != x.dtype:
        raise ValueError("gated_delta_step: B and C must have x's dtype")
    if not h.is_contiguous():
        raise ValueError("gated_delta_step: the state must be contiguous (it is updated in place)")
    x, B, C = x.contiguous(), B.contiguous(), C.contiguous()
    dt, beta, A_log = (t.float().contiguous() for t in (dt, beta, A_log))
    if y is None:
        y = torch.empty_like(x)
    elif y.shape != x.shape or y.dtype != x.dtype or not y.is_contiguous():
        raise ValueError("gated_delta_step: y must be contiguous and match x")
    with device_of(x):
        call("tssm_gated_delta_step", ptr(x), ptr(dt), ptr(h), ptr(A_log), ptr(B), ptr(C), ptr(beta), ptr(y), S, H, G,
             P, N, float(scale), dtype_code(x), stream_of(x))
    return y
