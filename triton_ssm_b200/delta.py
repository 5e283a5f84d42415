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

from . import _lib
from ._lib import addr, call, dtype_code, on_device, raw_stream, same_device
from .ops import _need

__all__ = ["gated_delta_rule", "gated_delta_rule_bwd", "gated_delta_step"]

CHUNK = 64


_IO = (torch.float32, torch.bfloat16)


def _dense(t):
    """t contiguous and on a 16-byte boundary (a view at an odd offset is copied: the copies
    that the kernels make by hardware start there)."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _f32(t):
    """t as a contiguous f32 tensor."""
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _rule_args(name, u, A_log, B, C, dt, beta, h0):
    _need(u, _IO, "u")
    if u.dim() != 3 or B.dim() != 4 or dt.dim() != 3:
        raise ValueError("%s: expected u [Bt,L,H*P], B, C [Bt,L,G,N], dt [Bt,L,H]" % name)
    Bt, L, HP = u.shape
    G, N = B.shape[2:]
    H = dt.shape[2]
    if H < 1 or G < 1 or HP % H or H % G:
        raise ValueError("%s: u's last dim (%d) must be H*P and H (%d) a multiple of G (%d)" % (name, HP, H, G))
    P = HP // H
    if B.shape != (Bt, L, G, N) or C.shape != B.shape or dt.shape != (Bt, L, H) or beta.shape != dt.shape or \
            A_log.shape != (H,) or (h0 is not None and h0.shape != (Bt, H, P, N)):
        raise ValueError("%s: shape mismatch" % name)
    if B.dtype != u.dtype or C.dtype != u.dtype:
        raise ValueError("%s: B and C must have u's dtype" % name)
    return Bt, L, H, G, P, N


def gated_delta_rule(u, A_log, B, C, dt, beta, scale=1.0, h0=None, return_state=False, save=False, y=None,
                     h_last=None):
    """The gated delta rule over whole sequences.

    u [Bt,L,H*P] f32 or bf16; A_log [H] f32 (log(-A_h)); B, C [Bt,L,G,N] in
    u's dtype, H a multiple of G, N <= 128; dt, beta [Bt,L,H] f32; h0
    [Bt,H,P,N] f32 or None.  Values must be finite (a chunk of 64 tokens is one
    matrix problem); pad with zeros, dt = 0 and beta = 0.
    Returns y [Bt,L,H*P] in u's dtype, or a tuple: y, then h_last [Bt,H,P,N]
    f32 when ``return_state`` (written to the given ``h_last``, which may be
    h0 itself: the state is then updated in place), then, when ``save``, what
    ``gated_delta_rule_bwd`` reads: (the state before every chunk of 64 tokens
    [Bt,H,ceil(L/64),ceil(N/4),P,4], the prediction errors u_t - hd B_t
    [Bt,H,ceil(L/4),P,4]), f32.
    """
    dev = same_device(u, A_log, B, C, dt, beta, h0, y, h_last)
    Bt, L, H, G, P, N = _rule_args("gated_delta_rule", u, A_log, B, C, dt, beta, h0)
    u, B, C = _dense(u), _dense(B), _dense(C)
    A_log, dt, beta = _f32(A_log), _f32(dt), _f32(beta)
    h0 = _dense(h0.float()) if h0 is not None else None
    if y is None:
        y = torch.empty_like(u)
    elif y.shape != u.shape or y.dtype != u.dtype or not y.is_contiguous():
        raise ValueError("gated_delta_rule: y must be contiguous and match u")
    f32 = dict(device=u.device, dtype=torch.float32)
    hl = h_last
    if hl is None:
        hl = torch.empty(Bt, H, P, N, **f32) if return_state else None
    elif not return_state or hl.shape != (Bt, H, P, N) or hl.dtype != torch.float32 or not hl.is_contiguous():
        raise ValueError("gated_delta_rule: h_last must be contiguous f32 [Bt,H,P,N], with return_state=True")
    states = torch.empty(Bt, H, -(-L // CHUNK), -(-N // 4), P, 4, **f32) if save else None
    errors = torch.empty(Bt, H, -(-L // 4), P, 4, **f32) if save else None
    need = int(_lib.load_library().tssm_gated_delta_rule_workspace_size(Bt, L, H, G, P, N, dtype_code(u)))
    ws = torch.empty(need, dtype=torch.uint8, device=u.device) if need else None
    with on_device(dev):
        call("tssm_gated_delta_rule", addr(u), addr(A_log), addr(B), addr(C), addr(dt), addr(beta), addr(h0), addr(y), addr(hl),
             addr(states), addr(errors), addr(ws), need, Bt, L, H, G, P, N, float(scale), dtype_code(u), raw_stream(dev))
    out = [y]
    if return_state:
        out.append(hl)
    if save:
        out.append((states, errors))
    return out[0] if len(out) == 1 else tuple(out)


def gated_delta_rule_bwd(u, A_log, B, C, dt, beta, dy, saved, scale=1.0, dh_last=None):
    """Backward of ``gated_delta_rule``.

    The forward's inputs, dy [Bt,L,H*P] in u's dtype, ``saved`` from a forward
    with ``save=True`` (and the same ``scale``), dh_last [Bt,H,P,N] f32 or None
    (the gradient of the final state).  Returns (du, dA_log, dB, dC, ddt,
    dbeta, dh0): du, dB, dC in u's dtype, the others f32; dB and dC are summed
    over the heads that share a key head.  Every sum runs in a fixed order.
    """
    states, errors = saved
    dev = same_device(u, A_log, B, C, dt, beta, dy, states, errors, dh_last)
    Bt, L, H, G, P, N = _rule_args("gated_delta_rule_bwd", u, A_log, B, C, dt, beta, dh_last)
    if dy.shape != u.shape or dy.dtype != u.dtype:
        raise ValueError("gated_delta_rule_bwd: dy must match u")
    for t, shape in ((states, (Bt, H, -(-L // CHUNK), -(-N // 4), P, 4)), (errors, (Bt, H, -(-L // 4), P, 4))):
        if tuple(t.shape) != shape or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("gated_delta_rule_bwd: saved must be what gated_delta_rule(..., save=True) returned")
    u, B, C, dy = _dense(u), _dense(B), _dense(C), _dense(dy)
    A_log, dt, beta = _f32(A_log), _f32(dt), _f32(beta)
    dh_last = _dense(dh_last.float()) if dh_last is not None else None
    f32 = dict(device=u.device, dtype=torch.float32)
    du, dB, dC, dA_log = torch.empty_like(u), torch.empty_like(B), torch.empty_like(C), torch.empty_like(A_log)
    ddt, dbeta, dh0 = torch.empty_like(dt), torch.empty_like(beta), torch.empty(Bt, H, P, N, **f32)
    need = int(_lib.load_library().tssm_gated_delta_rule_bwd_workspace_size_dtype(Bt, L, H, G, P, N, dtype_code(u)))
    ws = torch.empty(need, dtype=torch.uint8, device=u.device) if need else None
    with on_device(dev):
        call("tssm_gated_delta_rule_bwd", addr(u), addr(A_log), addr(B), addr(C), addr(dt), addr(beta), addr(dy), addr(states),
             addr(errors), addr(dh_last), addr(du), addr(dA_log), addr(dB), addr(dC), addr(ddt), addr(dbeta), addr(dh0), addr(ws),
             need, Bt, L, H, G, P, N, float(scale), dtype_code(u), raw_stream(dev))
    return du, dA_log, dB, dC, ddt, dbeta, dh0


def gated_delta_step(x, dt, h, A_log, B, C, beta, scale=1.0, y=None):
    """One token of every stream; the state is updated in place.

    x [S,H,P] f32 or bf16; dt, beta [S,H] f32; h [S,H,P,N] f32; A_log [H] f32;
    B, C [S,G,N] in x's dtype, H a multiple of G, N <= 256.  Returns y [S,H,P]
    in x's dtype.
    """
    dev = same_device(x, dt, h, A_log, B, C, beta, y)
    _need(x, _IO, "x")
    _need(h, (torch.float32,), "h")
    if x.dim() != 3 or h.dim() != 4 or B.dim() != 3:
        raise ValueError("gated_delta_step: expected x [S,H,P], h [S,H,P,N], B, C [S,G,N]")
    S, H, P = x.shape
    G, N = B.shape[1], h.shape[3]
    if h.shape != (S, H, P, N) or B.shape != (S, G, N) or C.shape != B.shape or dt.shape != (S, H) or \
            beta.shape != (S, H) or A_log.shape != (H,):
        raise ValueError("gated_delta_step: shape mismatch")
    if B.dtype != x.dtype or C.dtype != x.dtype:
        raise ValueError("gated_delta_step: B and C must have x's dtype")
    if not h.is_contiguous():
        raise ValueError("gated_delta_step: the state must be contiguous (it is updated in place)")
    x, B, C = x.contiguous(), B.contiguous(), C.contiguous()
    dt, beta, A_log = _f32(dt), _f32(beta), _f32(A_log)
    if y is None:
        y = torch.empty_like(x)
    elif y.shape != x.shape or y.dtype != x.dtype or not y.is_contiguous():
        raise ValueError("gated_delta_step: y must be contiguous and match x")
    with on_device(dev):
        call("tssm_gated_delta_step", x.data_ptr(), dt.data_ptr(), h.data_ptr(), A_log.data_ptr(), B.data_ptr(),
             C.data_ptr(), beta.data_ptr(), y.data_ptr(), S, H, G, P, N, float(scale), dtype_code(x), raw_stream(dev))
    return y
