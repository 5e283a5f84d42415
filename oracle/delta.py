"""The gated delta rule in 64 bits, token by token (no chunks)."""
import torch

__all__ = ["gated_delta", "gated_delta_grads"]


def gated_delta(u, A_log, B, C, dt, beta, scale=1.0, h0=None):
    """u [Bt,L,H,P]; A_log [H]; B, C [Bt,L,G,N]; dt, beta [Bt,L,H]; h0 [Bt,H,P,N] or None.
    Returns (y [Bt,L,H,P], h_last [Bt,H,P,N]) in f64; differentiable."""
    u, A_log, B, C, dt, beta = (t.double() for t in (u, A_log, B, C, dt, beta))
    Bt, L, H, P = u.shape
    B, C = (t.repeat_interleave(H // t.shape[2], 2) for t in (B, C))
    h = h0.double() if h0 is not None else u.new_zeros(Bt, H, P, B.shape[3])
    alpha = torch.exp(-torch.exp(A_log) * dt)
    ys = []
    for t in range(L):
        h = alpha[:, t, :, None, None] * h
        e = u[:, t] - (h * B[:, t, :, None, :]).sum(-1)
        h = h + (beta[:, t, :, None] * e)[..., None] * B[:, t, :, None, :]
        ys.append(scale * (h * C[:, t, :, None, :]).sum(-1))
    return (torch.stack(ys, 1) if ys else u.clone()), h


def gated_delta_grads(u, A_log, B, C, dt, beta, dy, scale=1.0, h0=None, dh_last=None):
    """Gradients of <y, dy> + <h_last, dh_last> by autograd through gated_delta, in f64:
    (du, dA_log, dB, dC, ddt, dbeta, dh0)."""
    h0 = h0 if h0 is not None else u.new_zeros(u.shape[0], u.shape[2], u.shape[3], B.shape[3])
    leaves = [t.double().clone().requires_grad_(True) for t in (u, A_log, B, C, dt, beta, h0)]
    y, h = gated_delta(*leaves[:6], scale=scale, h0=leaves[6])
    f = (y * dy.double()).sum() + ((h * dh_last.double()).sum() if dh_last is not None else 0.0)
    return torch.autograd.grad(f, leaves)
