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


def half_step(ref):
    """Half of bf16's step at each value."""
    return torch.exp2(torch.floor(torch.log2(ref.abs().clamp_min(1e-30)))) * 2.0 ** -8


def one_hot(*shape, at, value):
    x = torch.zeros(*shape)
    x[..., at] = value
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("N,P", [(128, 128), (64, 64), (128, 192), (24, 40)])
@pytest.mark.parametrize("part", ["state", "write", "both"])
def test_y_is_rounded_once(cuda_ops, part, N, P):
    """One token on one coordinate n: y_p = scale (a S_pn q + beta (u_p - a S_pn k) k q) with a = exp(0) = 1.
    Every sum has a few terms, so that y before its rounding is off by f32 roundings alone: about 16 of them, of
    2^-24 (2^-23 where the tensor core cuts instead), one after the other: 2^-19 of the magnitudes that enter.
    Operands held to 16 bits would be off by up to 2^-17."""
    Bt, H, n = 96, 8, N - 5
    g = torch.Generator().manual_seed(N + P)
    u = torch.randn(Bt, 1, H, P, generator=g).bfloat16()
    h0 = torch.randn(Bt, H, P, N, generator=g) if part != "write" else torch.zeros(Bt, H, P, N)
    beta = torch.rand(Bt, 1, H, generator=g) if part != "state" else torch.zeros(Bt, 1, H)
    k, q = torch.rand(2, Bt, 1, H, 1, generator=g).add(0.5).bfloat16().unbind(0)
    B, C = (one_hot(Bt, 1, H, N, at=n, value=0).bfloat16() for _ in range(2))
    B[..., n:n + 1], C[..., n:n + 1] = k, q
    scale = 0.7
    y = cuda_ops.gated_delta_rule(u.flatten(2).to(dev), torch.zeros(H, device=dev), B.to(dev), C.to(dev),
                                  torch.zeros(Bt, 1, H, device=dev), beta.to(dev), scale=scale, h0=h0.to(dev))
    s, b, v = h0[..., n].double(), beta[:, 0, :, None].double(), u[:, 0].double()
    k, q = k[:, 0].double(), q[:, 0].double()
    ref = scale * q * (s + b * (v - s * k) * k)
    mag = scale * q * (s.abs() + b * (v.abs() + s.abs() * k) * k)
    d = (y.double().cpu().view_as(ref) - ref).abs() - half_step(ref)
    assert bool((d <= 2.0 ** -19 * mag).all()), "%d of %d values beyond" % (int((d > 2.0 ** -19 * mag).sum()), d.numel())
