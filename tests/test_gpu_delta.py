"""The gated delta rule against the 64-bit token-by-token oracle."""
import pytest
import torch

from oracle.delta import gated_delta, gated_delta_grads

dev = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(Bt, L, H, G, N, P, dtype, seed=0, decay=1.0):
    """Unit keys, beta in (0, 1), irregular steps; h0 and gradients of both outputs."""
    g = torch.Generator().manual_seed(seed)

    def n(*s):
        return torch.randn(*s, generator=g)

    B = n(Bt, L, G, N)
    return dict(u=n(Bt, L, H, P).to(dtype), A_log=torch.log(0.5 + 15.5 * torch.rand(H, generator=g)),
                B=(B / B.norm(dim=-1, keepdim=True)).to(dtype), C=n(Bt, L, G, N).to(dtype),
                dt=decay * torch.exp(-6.9 * torch.rand(Bt, L, H, generator=g)),
                beta=torch.sigmoid(n(Bt, L, H))), 0.3 * n(Bt, H, P, N)


# ------------------------------------------------------------------ single tokens
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,H,G,N,P", [(1, 1, 1, 64, 64), (3, 4, 2, 128, 128), (2, 3, 3, 20, 7), (5, 2, 1, 33, 130),
                                       (2, 2, 2, 256, 48), (1, 6, 3, 1, 1), (40, 16, 8, 128, 128), (2, 1, 1, 128, 513)])
def test_step(cuda_ops, S, H, G, N, P, dtype):
    a, h0 = make(S, 1, H, G, N, P, dtype, seed=N + P)
    h = h0.to(dev)
    y = cuda_ops.gated_delta_step(a["u"][:, 0].to(dev), a["dt"][:, 0].to(dev), h, a["A_log"].to(dev),
                                  a["B"][:, 0].to(dev), a["C"][:, 0].to(dev), a["beta"][:, 0].to(dev), scale=0.7)
    ry, rh = gated_delta(**a, scale=0.7, h0=h0)
    # the decay's argument (up to 16) rounds three times, the exponential twice: 50 steps of alpha;
    # a row's dot product rounds N / 8 + 3 times in a row
    k = (60 + N / 8) * 2.0 ** -24
    B, C = (a[m][:, 0].double().repeat_interleave(H // G, 1).abs() for m in ("B", "C"))
    al = torch.exp(-torch.exp(a["A_log"].double()) * a["dt"][:, 0].double())
    hd = al[..., None, None] * h0.double().abs()
    e = a["beta"][:, 0, :, None] * (a["u"][:, 0].double().abs() + (hd * B[:, :, None]).sum(-1))
    mag = hd + e[..., None] * B[:, :, None]
    assert bool(((h.double().cpu() - rh).abs() <= k * mag).all())
    tol = HALF[dtype] * 1.01 * ry[:, 0].abs() + 0.7 * 2 * k * (mag * C[:, :, None]).sum(-1)
    assert y.dtype == dtype and bool(((y.double().cpu() - ry[:, 0]).abs() <= tol).all())


@pytest.mark.gpu
def test_step_padding_reset_and_reuse(cuda_ops):
    """dt = 0 with beta = 0 keeps the state's bits; an infinite dt forgets it; y may be given."""
    a, h0 = make(4, 1, 2, 2, 64, 64, torch.bfloat16, seed=1)
    t = {k: (v if k == "A_log" else v[:, 0]).to(dev) for k, v in a.items()}
    t["dt"][0], t["beta"][0] = 0.0, 0.0
    t["dt"][1] = float("inf")
    h, y = h0.to(dev), torch.empty(4, 2, 64, device=dev, dtype=torch.bfloat16)
    out = cuda_ops.gated_delta_step(t["u"], t["dt"], h, t["A_log"], t["B"], t["C"], t["beta"], y=y)
    assert out is y
    assert torch.equal(h[0].cpu(), h0[0])
    ref = a["beta"][1, 0, :, None, None] * a["u"][1, 0].float()[:, :, None] * a["B"][1, 0].float()[:, None]
    assert (h[1].cpu() - ref).abs().max() <= 4 * 2.0 ** -24 * ref.abs().max()


@pytest.mark.gpu
def test_step_unaligned(cuda_ops):
    a, h0 = make(2, 1, 2, 2, 64, 32, torch.bfloat16, seed=2)
    t = {k: (v if k == "A_log" else v[:, 0]).to(dev) for k, v in a.items()}
    buf = torch.zeros(t["B"].numel() + 1, device=dev, dtype=torch.bfloat16)
    buf[1:] = t["B"].flatten()
    h, h2 = h0.to(dev), h0.to(dev)
    y = cuda_ops.gated_delta_step(t["u"], t["dt"], h, t["A_log"], t["B"], t["C"], t["beta"])
    y2 = cuda_ops.gated_delta_step(t["u"], t["dt"], h2, t["A_log"], buf[1:].view_as(t["B"]), t["C"], t["beta"])
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_step_refusals_without_gpu():
    import triton_ssm_b200 as ts
    from triton_ssm_b200 import _lib
    a, h0 = make(2, 1, 2, 2, 64, 32, torch.float32)
    t = {k: (v if k == "A_log" else v[:, 0]) for k, v in a.items()}
    with pytest.raises(ValueError, match="CUDA"):
        ts.gated_delta_step(t["u"], t["dt"], h0, t["A_log"], t["B"], t["C"], t["beta"])
    lib = _lib.load_library()
    one = 4096   # a non-null address that nothing reads

    def step(S=2, H=4, G=2, P=8, N=16, dtype=0, x=one):
        return lib.tssm_gated_delta_step(x, one, one, one, one, one, one, one, S, H, G, P, N, 1.0, dtype, 0)

    for kw in (dict(S=-1), dict(G=3), dict(G=0), dict(N=0), dict(N=257), dict(dtype=2), dict(x=0), dict(S=1 << 40)):
        assert step(**kw) == 1, kw
    assert step(S=0) == 0
