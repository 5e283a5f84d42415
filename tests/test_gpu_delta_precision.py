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


@pytest.mark.gpu
@pytest.mark.parametrize("N,P", [(128, 128), (64, 64), (24, 40)])
def test_key_and_query_gradients_are_rounded_once(cuda_ops, N, P):
    """Two tokens, k_0 on the first half of the coordinates, k_1 and q_1 on one of the second half, dy only for
    token 1 and channel p, no decay: on the first half dC_1 = scale beta_0 dy u_0p k_0 and
    dB_1 = -beta_0 beta_1 scale (q_1 k_1) dy u_0p k_0.  Every product on the way has one term, so that the values
    before their rounding are off by about 30 f32 roundings of 2^-24: 2^-19.  Factors held to 16 bits would be off
    by up to 2^-18."""
    Bt, H, n, p, scale = 512, 8, N - 3, P - 7, 0.75
    g = torch.Generator().manual_seed(N)

    def rand(*shape):
        return torch.rand(*shape, generator=g).add(0.5).bfloat16()

    u, dy = torch.randn(Bt, 2, H, P, generator=g).bfloat16(), torch.zeros(Bt, 2, H, P).bfloat16()
    dy[:, 1, :, p] = rand(Bt, H)
    B, C = torch.zeros(Bt, 2, H, N).bfloat16(), torch.zeros(Bt, 2, H, N).bfloat16()
    B[:, 0, :, :N // 2] = rand(Bt, H, N // 2)
    B[:, 1, :, n], C[:, 1, :, n] = rand(Bt, H), rand(Bt, H)
    beta = torch.rand(Bt, 2, H, generator=g)
    args = (u.flatten(2).to(dev), torch.zeros(H, device=dev), B.to(dev), C.to(dev), torch.zeros(Bt, 2, H, device=dev),
            beta.to(dev))
    _, saved = cuda_ops.gated_delta_rule(*args, scale=scale, save=True)
    grads = cuda_ops.gated_delta_rule_bwd(*args, dy.flatten(2).to(dev), saved, scale=scale)
    b = beta.double()
    m1 = scale * b[:, 0] * dy[:, 1, :, p].double() * u[:, 0, :, p].double()
    m2 = m1 * b[:, 1] * B[:, 1, :, n].double() * C[:, 1, :, n].double()
    k0 = B[:, 0, :, :N // 2].double()
    for name, x, ref in (("dC", grads[3], m1[..., None] * k0), ("dB", grads[2], -m2[..., None] * k0)):
        d = (x[:, 1, :, :N // 2].double().cpu() - ref).abs() - half_step(ref)
        bad = d > 2.0 ** -19 * ref.abs()
        assert not bool(bad.any()), "%s: %d of %d values beyond" % (name, int(bad.sum()), d.numel())


@pytest.mark.gpu
def test_f32_sums_over_the_width_of_the_state(cuda_ops):
    """Sums of 128 positive terms in f32: y = scale sum_n q_n S_pn, the error u - sum_n k_n S_pn with u = 0, and
    dC_n = scale sum_p S_pn dy_p (one token, beta = 0).  A piece of 16 terms is cut once at its full size (2 steps
    of 2^-24) and five times at 2^-8 of it; eight pieces are added with one rounding each, onto 9/16 of the sum on
    average (4.5 steps); the factors scale and exp(l) round twice and u - x once: 10 steps of 2^-24."""
    Bt, H, N, P, scale = 4, 2, 128, 128, 0.3
    g = torch.Generator().manual_seed(5)
    S, k, q, dy = (torch.rand(*s, generator=g) + 0.5 for s in ((Bt, H, P, N), (Bt, 1, H, N), (Bt, 1, H, N), (Bt, 1, H, P)))
    zero = torch.zeros(Bt, 1, H, device=dev)
    args = (torch.zeros(Bt, 1, H * P, device=dev), torch.zeros(H, device=dev), k.to(dev), q.to(dev), zero, zero)
    y, saved = cuda_ops.gated_delta_rule(*args, scale=scale, h0=S.to(dev), save=True)
    dC = cuda_ops.gated_delta_rule_bwd(*args, dy.flatten(2).to(dev), saved, scale=scale)[3]
    S, k, q, dy = (t.double() for t in (S, k[:, 0], q[:, 0], dy[:, 0]))
    e = saved[1][:, :, 0, :, 0]
    for name, x, ref in (("y", y.view(Bt, H, P), scale * (S * q[:, :, None]).sum(-1)), ("error", e, -(S * k[:, :, None]).sum(-1)),
                         ("dC", dC.view(Bt, H, N), scale * (S * dy[..., None]).sum(2))):
        d = ((x.double().cpu() - ref) / ref).abs().max().item() * 2.0 ** 24
        assert d <= 10, "%s: off by %.1f steps of 2^-24" % (name, d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,P", [(128, 128), (64, 64), (48, 80)])
def test_state_under_many_small_writes(cuda_ops, N, P, dtype):
    """1024 tokens whose writes take 2^-20 of one column of the state each: it is written four times a chunk, half a
    step off at most each time; e and the decay's product add one step a chunk: 6 steps of 2^-24 a chunk.  So is the
    state's gradient, with the signs of the backward's."""
    Bt, L, H, n = 2, 1024, 2, N - 2
    S = torch.rand(Bt, H, P, N, generator=torch.Generator().manual_seed(6)) + 0.5
    k = one_hot(Bt, L, H, N, at=n, value=2.0 ** -10).to(dev).to(dtype)
    u, zero = torch.zeros(Bt, L, H * P, device=dev, dtype=dtype), torch.zeros(Bt, L, H, device=dev)
    args = (u, torch.zeros(H, device=dev), k, k, zero, torch.ones(Bt, L, H, device=dev))
    _, h, saved = cuda_ops.gated_delta_rule(*args, h0=S.to(dev), return_state=True, save=True)
    dh0 = cuda_ops.gated_delta_rule_bwd(*args, u, saved, dh_last=S.to(dev))[6]
    other = [i for i in range(N) if i != n]
    ref = S[..., n].double() * (1 - 2.0 ** -20) ** L
    for x in (h.cpu(), dh0.cpu()):
        assert torch.equal(x[..., other], S[..., other])
        d = ((x[..., n].double() - ref) / ref).abs().max().item() * 2.0 ** 24
        assert d <= 6 * L / 64, "off by %.1f steps of 2^-24" % d
