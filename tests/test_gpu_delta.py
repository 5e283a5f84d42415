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


# ------------------------------------------------------------------ whole sequences
def off(out, ref):
    """2-norm of the difference over the 2-norm of the result."""
    return ((out.double().cpu() - ref).norm() / ref.norm().clamp_min(1e-300)).item()


# Relative 2-norm tolerances.  A bf16 result: its own rounding is uniform within half a step of
# 2^-9 to 2^-8 of the value, 2-norm 2^-8 / sqrt(3) at most, and y has two planes (2^-16) of slack:
# 2^-8.  An f32 result goes through at most L / 64 + 1 chunks, each a chain of five products of
# f32-exact operands whose sums round once per 16 terms (N / 16 + 2 roundings of 2^-24, at most 10),
# and an inverse whose entries round 64 times: (5 * 10 + 64) * 2^-24 a chunk; errors decay or stay
# bounded with the state, so chunks add at most like their number's square root: 2^-17 sqrt(chunks).
def tol(dtype, L):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -17 * max(1.0, (L / 64) ** 0.5)


SHAPES = [(2, 1, 2, 1, 64, 64), (1, 63, 1, 1, 64, 64), (2, 64, 2, 2, 128, 128), (1, 65, 4, 2, 128, 64),
          (2, 200, 3, 1, 64, 128), (1, 150, 2, 2, 40, 24), (1, 129, 2, 1, 17, 5), (2, 333, 4, 2, 128, 130),
          (3, 70, 60, 30, 64, 128), (1, 100, 1, 1, 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,H,G,N,P", SHAPES)
def test_rule(cuda_ops, Bt, L, H, G, N, P, dtype):
    a, h0 = make(Bt, L, H, G, N, P, dtype, seed=L)
    d = {k: v.to(dev) for k, v in a.items()}
    d["u"] = d["u"].reshape(Bt, L, H * P)
    y, h, (states, errors) = cuda_ops.gated_delta_rule(**d, scale=0.3, h0=h0.to(dev), return_state=True, save=True)
    ry, rh = gated_delta(**a, scale=0.3, h0=h0)
    assert y.dtype == dtype and y.shape == (Bt, L, H * P)
    assert off(y.view(Bt, L, H, P), ry) < tol(dtype, L)
    assert off(h, rh) < tol(torch.float32, L)
    states = states.transpose(3, 4).flatten(4)[..., :N]
    assert torch.equal(states[:, :, 0].cpu(), h0)
    if L > 64:
        cut = {k: (v if k == "A_log" else v[:, :64]) for k, v in a.items()}
        assert off(states[:, :, 1], gated_delta(**cut, h0=h0)[1]) < tol(torch.float32, 64)
    # without a state, y comes from two planes
    y2 = cuda_ops.gated_delta_rule(**d, scale=0.3)
    assert off(y2.view(Bt, L, H, P), gated_delta(**a, scale=0.3)[0]) < tol(dtype, L)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rule_same_key_again_and_again(cuda_ops, dtype):
    """One key for every token, beta 1, next to no decay: A is all ones below the diagonal, where the
    powers of A overflow any expansion; each write replaces the value before it."""
    a, h0 = make(1, 130, 1, 1, 64, 64, dtype, seed=7)
    a["B"][:] = 0
    a["B"][..., 3] = 1
    a["beta"][:] = 1
    a["dt"][:] = 1e-6
    d = {k: v.to(dev) for k, v in a.items()}
    y, h = cuda_ops.gated_delta_rule(d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"], h0=h0.to(dev),
                                     return_state=True)
    ry, rh = gated_delta(**a, h0=h0)
    assert off(y.view_as(ry), ry) < tol(dtype, 130) and off(h, rh) < tol(torch.float32, 130)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rule_resets_strong_decay_and_padding(cuda_ops, dtype):
    """Infinite and large steps forget the state; padded tokens (zeros) leave it; what follows still fits."""
    a, h0 = make(2, 200, 2, 1, 64, 64, dtype, seed=9, decay=20.0)
    a["dt"][0, 70], a["dt"][1, 3] = float("inf"), 1e30
    for k in ("u", "B", "C", "dt", "beta"):
        a[k][0, 150:] = 0
    d = {k: v.to(dev) for k, v in a.items()}
    y, h = cuda_ops.gated_delta_rule(d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"], h0=h0.to(dev),
                                     return_state=True)
    ry, rh = gated_delta(**a, h0=h0)
    assert off(y.view_as(ry), ry) < tol(dtype, 200) and off(h, rh) < tol(torch.float32, 200)
    cut = cuda_ops.gated_delta_rule(d["u"][:1, :150].flatten(2), d["A_log"], d["B"][:1, :150], d["C"][:1, :150],
                                    d["dt"][:1, :150], d["beta"][:1, :150], h0=h0[:1].to(dev), return_state=True)[1]
    assert off(h[:1], cut.double().cpu()) < 2.0 ** -22


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rule_meets_step(cuda_ops, dtype):
    """A prompt in one call, then tokens one by one, is the whole sequence; two calls are one."""
    a, h0 = make(2, 100, 4, 2, 128, 64, dtype, seed=11)
    d = {k: v.to(dev) for k, v in a.items()}
    ry, rh = gated_delta(**a)
    part = lambda s: (d["u"][:, s].flatten(2), d["A_log"], d["B"][:, s], d["C"][:, s], d["dt"][:, s], d["beta"][:, s])  # noqa: E731
    y, h = cuda_ops.gated_delta_rule(*part(slice(0, 90)), return_state=True)
    h2 = h.clone()
    outs = [y.view(2, 90, 4, 64)]
    for t in range(90, 100):
        outs.append(cuda_ops.gated_delta_step(d["u"][:, t], d["dt"][:, t], h, d["A_log"], d["B"][:, t], d["C"][:, t],
                                              d["beta"][:, t])[:, None])
    assert off(torch.cat(outs, 1), ry) < tol(dtype, 100) and off(h, rh) < tol(torch.float32, 100)
    y2, h2 = cuda_ops.gated_delta_rule(*part(slice(90, 100)), h0=h2, return_state=True)
    assert off(y2.view(2, 10, 4, 64), ry[:, 90:]) < tol(dtype, 100) and off(h2, rh) < tol(torch.float32, 100)


@pytest.mark.gpu
def test_rule_empty_strided_stream_and_graph(cuda_ops):
    a, h0 = make(2, 77, 2, 2, 64, 64, torch.bfloat16, seed=13)
    d = {k: v.to(dev) for k, v in a.items()}
    args = (d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"])
    y, h = cuda_ops.gated_delta_rule(*args, h0=h0.to(dev), return_state=True)
    # no tokens: the state passes through
    none = cuda_ops.gated_delta_rule(*(t if t.dim() == 1 else t[:, :0] for t in args), h0=h0.to(dev), return_state=True)
    assert none[0].shape == (2, 0, 128) and torch.equal(none[1].cpu(), h0)
    # a transposed view and an odd offset
    wide = torch.zeros(2, 77, 2, 80, device=dev, dtype=torch.bfloat16)
    wide[..., 16:] = d["B"]
    buf = torch.zeros(args[0].numel() + 1, device=dev, dtype=torch.bfloat16)
    buf[1:] = args[0].flatten()
    y2 = cuda_ops.gated_delta_rule(buf[1:].view_as(args[0]), d["A_log"], wide[..., 16:], *args[3:], h0=h0.to(dev), return_state=True)
    assert torch.equal(y2[0], y) and torch.equal(y2[1], h)
    # another stream, and a captured call replayed on new inputs
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y3 = cuda_ops.gated_delta_rule(*args, h0=h0.to(dev), return_state=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y3[0], y) and torch.equal(y3[1], h)
    graph, u = torch.cuda.CUDAGraph(), torch.zeros_like(args[0])
    with torch.cuda.graph(graph):
        y4, h4 = cuda_ops.gated_delta_rule(u, *args[1:], h0=None, return_state=True)
    u.copy_(args[0])
    graph.replay()
    torch.cuda.synchronize()
    y5, h5 = cuda_ops.gated_delta_rule(*args, return_state=True)
    assert torch.equal(y4, y5) and torch.equal(h4, h5)


def test_rule_refusals_without_gpu():
    import triton_ssm_b200 as ts
    from triton_ssm_b200 import _lib
    from triton_ssm_b200.delta import _rule_args
    a, h0 = make(2, 5, 4, 2, 16, 8, torch.float32)
    a["u"] = a["u"].flatten(2)
    with pytest.raises(ValueError, match="CUDA"):
        ts.gated_delta_rule(**a)
    order = ("u", "A_log", "B", "C", "dt", "beta")
    for bad in (dict(u=a["u"].double()), dict(u=a["u"][..., :-1]), dict(B=a["B"][:, :, :1]), dict(C=a["C"].bfloat16()),
                dict(beta=a["beta"][:, :4]), dict(A_log=a["A_log"][:3]), dict(h0=h0[:, :, :4]), dict(dt=a["dt"][0]),
                dict(B=a["B"][:, :, [0, 1, 1]], C=a["C"][:, :, [0, 1, 1]])):
        kw = dict(a, h0=h0, **{}) | bad
        with pytest.raises(ValueError):
            _rule_args("gated_delta_rule", *(kw[k] for k in order), kw["h0"])
    lib = _lib.load_library()
    one = 4096   # a non-null address that nothing reads

    def rule(Bt=2, L=3, H=4, G=2, P=8, N=16, dtype=0, u=one, states=0, errors=0, ws=0, nbytes=0):
        return lib.tssm_gated_delta_rule(u, one, one, one, one, one, 0, one, 0, states, errors, ws, nbytes, Bt, L, H, G,
                                         P, N, 1.0, dtype, 0)

    for kw in (dict(Bt=-1), dict(G=3), dict(G=0), dict(N=0), dict(N=129), dict(dtype=2), dict(u=0), dict(L=1 << 31),
               dict(states=one), dict(errors=one), dict(dtype=1, P=64, N=64),
               dict(dtype=1, P=64, N=64, ws=one, nbytes=1000), dict(dtype=1, P=64, N=64, ws=one + 4, nbytes=1 << 30)):
        assert rule(**kw) == 1, kw
    assert rule(Bt=0) == 0


# ------------------------------------------------------------------ backward
NAMES = ("du", "dA_log", "dB", "dC", "ddt", "dbeta", "dh0")


def run_bwd(ts, a, h0, dy, dh, scale):
    d = {k: v.to(dev) for k, v in a.items()}
    args = (d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"])
    _, saved = ts.gated_delta_rule(*args, scale=scale, h0=None if h0 is None else h0.to(dev), save=True)
    return ts.gated_delta_rule_bwd(*args, dy.to(dev).flatten(2), saved, scale=scale,
                                   dh_last=None if dh is None else dh.to(dev))


def check_grads(grads, ref, a, dtype, L):
    """The forward's chain and the backward's: twice the forward's f32 tolerance.  A dt's gradient is a sum of
    up to 64 x 64 paths within a chunk, 16 more roundings.  dA_log sums ddt dt over all tokens with either sign:
    its tolerance is of the sum of magnitudes."""
    f32 = 4 * tol(torch.float32, L)
    for name, x, r in zip(NAMES, grads, ref):
        r = r.reshape(x.shape)
        if name == "dA_log":
            size = (ref[4].abs() * a["dt"].double().clamp(max=1e6)).sum((0, 1))
            assert bool(((x.double().cpu() - r).abs() <= f32 * size).all()), name
        else:
            t = f32 if x.dtype == torch.float32 else tol(dtype, L)
            assert off(x, r) < t, "%s: %.3g, tolerance %.3g" % (name, off(x, r), t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,H,G,N,P", SHAPES)
def test_backward(cuda_ops, Bt, L, H, G, N, P, dtype):
    a, h0 = make(Bt, L, H, G, N, P, dtype, seed=L + 1)
    g = torch.Generator().manual_seed(L)
    dy, dh = torch.randn(Bt, L, H, P, generator=g).to(dtype), 0.3 * torch.randn(Bt, H, P, N, generator=g)
    grads = run_bwd(cuda_ops, a, h0, dy, dh, 0.3)
    check_grads(grads, gated_delta_grads(*a.values(), dy, scale=0.3, h0=h0, dh_last=dh), a, dtype, L)
    for x, like in zip(grads, (a["u"], a["A_log"], a["B"], a["C"], a["dt"], a["beta"], h0)):
        assert x.dtype == like.dtype and x.numel() == like.numel()


@pytest.mark.gpu
def test_backward_without_states(cuda_ops):
    """No h0, no gradient of the final state."""
    a, _ = make(2, 130, 2, 2, 64, 64, torch.float32, seed=21)
    dy = torch.randn(2, 130, 2, 64, generator=torch.Generator().manual_seed(1))
    check_grads(run_bwd(cuda_ops, a, None, dy, None, 1.0), gated_delta_grads(*a.values(), dy), a, torch.float32, 130)


@pytest.mark.gpu
def test_backward_same_key_resets_and_zero_beta(cuda_ops):
    """One key again and again, beta 0 and 1, infinite steps and padding."""
    a, h0 = make(2, 140, 1, 1, 64, 64, torch.float32, seed=22)
    a["B"][0] = 0
    a["B"][0, ..., 3] = 1
    a["beta"][0], a["dt"][0] = 1, 1e-6
    a["beta"][1, ::3] = 0
    a["dt"][1, 50] = 1e4    # exp(-5000) is 0 in both precisions
    for k in ("u", "B", "C", "dt", "beta"):
        a[k][1, 120:] = 0
    g = torch.Generator().manual_seed(2)
    dy, dh = torch.randn(2, 140, 1, 64, generator=g), torch.randn(2, 1, 64, 64, generator=g)
    grads = run_bwd(cuda_ops, a, h0, dy, dh, 1.0)
    check_grads(grads, gated_delta_grads(*a.values(), dy, h0=h0, dh_last=dh), a, torch.float32, 140)
    a["dt"][1, 50] = float("inf")
    again = run_bwd(cuda_ops, a, h0, dy, dh, 1.0)
    for x, y in zip(grads, again):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_backward_against_differences(cuda_ops):
    a, h0 = make(1, 70, 2, 1, 32, 16, torch.float32, seed=23)
    g = torch.Generator().manual_seed(3)
    dy, dh = torch.randn(1, 70, 2, 16, generator=g).double(), torch.randn(1, 2, 16, 32, generator=g).double()
    grads = run_bwd(cuda_ops, a, h0, dy.float(), dh.float(), 0.5)
    dy, dh = dy.float().double(), dh.float().double()
    leaves = [t.double() for t in (*a.values(), h0)]
    e = 1e-5
    for i, gr in enumerate(grads):
        d = torch.randn(leaves[i].shape, generator=g).double()
        f = []
        for s in (e, -e):
            x = list(leaves)
            x[i] = x[i] + s * d
            y, h = gated_delta(*x[:6], scale=0.5, h0=x[6])
            f.append(((y * dy).sum() + (h * dh).sum()).item())
        got = (gr.double().cpu().reshape(d.shape) * d).sum().item()
        size = (gr.double().cpu().reshape(d.shape) * d).abs().sum().item()
        assert abs((f[0] - f[1]) / (2 * e) - got) < 1e-5 * size + 1e-6, NAMES[i]


@pytest.mark.gpu
def test_backward_graph_repeats_and_empty(cuda_ops):
    a, h0 = make(2, 100, 4, 2, 128, 64, torch.bfloat16, seed=24)
    g = torch.Generator().manual_seed(4)
    dy, dh = torch.randn(2, 100, 4, 64, generator=g).bfloat16(), torch.randn(2, 4, 64, 128, generator=g)
    first = run_bwd(cuda_ops, a, h0, dy, dh, 1.0)
    d = {k: v.to(dev) for k, v in a.items()}
    args = (d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"])
    hd, dyd, dhd = h0.to(dev), dy.to(dev).flatten(2), dh.to(dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _, saved = cuda_ops.gated_delta_rule(*args, h0=hd, save=True)
        again = cuda_ops.gated_delta_rule_bwd(*args, dyd, saved, dh_last=dhd)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(first, again):
        assert torch.equal(x, y)
    none = tuple(t if t.dim() == 1 else t[:, :0] for t in args)
    _, saved = cuda_ops.gated_delta_rule(*none, h0=hd, save=True)
    out = cuda_ops.gated_delta_rule_bwd(*none, dyd[:, :0], saved, dh_last=dhd)
    assert torch.equal(out[6], dhd) and not out[1].any()


@pytest.mark.gpu
def test_many_streams_go_through_in_segments(cuda_ops):
    """So many streams that the sequence is cut into segments of single chunks: a row's results are
    those of the row alone."""
    Bt, L = 3300, 150
    a, h0 = make(2, L, 2, 1, 64, 64, torch.bfloat16, seed=27)
    d = {k: v.to(dev) for k, v in a.items()}
    g = torch.Generator().manual_seed(7)
    dy, dh = torch.randn(2, L, 128, generator=g).bfloat16().to(dev), torch.randn(2, 2, 64, 64, generator=g).to(dev)
    many = {k: (v if k == "A_log" else v.repeat(Bt // 2, *[1] * (v.dim() - 1))) for k, v in d.items()}

    def run(x, h, dy, dh):
        args = (x["u"].flatten(2), x["A_log"], x["B"], x["C"], x["dt"], x["beta"])
        y, hl, saved = cuda_ops.gated_delta_rule(*args, h0=h, return_state=True, save=True)
        grads = cuda_ops.gated_delta_rule_bwd(*args, dy, saved, dh_last=dh)
        return [y, hl] + [g for n, g in zip(NAMES, grads) if n != "dA_log"]

    few = run(d, h0.to(dev), dy, dh)
    out = run(many, h0.to(dev).repeat(Bt // 2, 1, 1, 1), dy.repeat(Bt // 2, 1, 1), dh.repeat(Bt // 2, 1, 1, 1))
    for x, y in zip(few, out):
        assert torch.equal(y[:2], x) and torch.equal(y[-2:], x)


def test_backward_refusals_without_gpu():
    from triton_ssm_b200 import _lib
    lib = _lib.load_library()
    one = 4096   # a non-null address that nothing reads

    def bwd(Bt=2, L=3, H=4, G=2, P=8, N=16, dtype=0, dy=one, ws=one, nbytes=1 << 30):
        return lib.tssm_gated_delta_rule_bwd(one, one, one, one, one, one, dy, one, one, 0, one, one, one, one, one, one,
                                             one, ws, nbytes, Bt, L, H, G, P, N, 1.0, dtype, 0)

    for kw in (dict(Bt=-1), dict(G=3), dict(G=0), dict(N=0), dict(N=129), dict(dtype=2), dict(dy=0), dict(ws=0),
               dict(nbytes=100), dict(ws=one + 4), dict(L=1 << 31)):
        assert bwd(**kw) == 1, kw
