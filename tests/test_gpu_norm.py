"""Group norm with an activation (channels last) against the 64-bit oracle.

Tolerances: an output is off by the rounding to its type (half a step, u times
its value) plus f32 arithmetic: K * 2^-24 times the sum of magnitudes that
enter it, K counting the roundings in a row on its way (a thread's share of a
sum, the tree that joins the threads, and about 60 for the rest)."""
import pytest
import torch

from oracle.norm import group_norm_act as oracle_norm

dev = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(Bt, L, C, dtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(Bt, L, C, generator=g) + offset * torch.randn(Bt, 1, C, generator=g)).to(dtype)
    w = 1.0 + 0.3 * torch.randn(C, generator=g)
    b = 0.3 * torch.randn(C, generator=g)
    return x, w, b, torch.randn(Bt, L, C, generator=g).to(dtype)


def terms(L, C, groups):
    return 80 + L * C // groups / 64


def scales(x, w, b, groups):
    """Per element: the magnitudes that enter z, and rstd (broadcast)."""
    Bt, L, C = x.shape
    xg = x.double().reshape(Bt, L, groups, -1)
    r = 1.0 / torch.sqrt(xg.var((1, 3), correction=0, keepdim=True) + 1e-5)
    big = (xg.abs() + xg.abs().mean((1, 3), keepdim=True)) * r
    return big.reshape(Bt, L, C) * w.abs() + b.abs(), r


def check(out, ref, tol, what):
    d = (out.double().cpu() - ref).abs()
    assert bool((d <= tol).all()), "%s: off by up to %.3g times its tolerance" % (what, (d / tol).max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,C,groups", [
    (5, 1, 32, 8),        # 4 channels a group
    (3, 1, 96, 2),        # 48 channels: idle lanes
    (2, 1, 21, 7),        # 3 channels: no wide access
    (70, 1, 4096, 32),    # full token rows
    (9, 1, 1030, 2),      # a group wider than a warp's registers hold: the map passes with L = 1
    (2, 1, 5, 1), (3, 7, 8, 8),   # one channel a group
    (2, 2, 64, 4), (3, 333, 48, 3), (1, 5000, 16, 2), (2, 130, 2560, 5), (4, 3, 35, 5),
])
def test_forward(cuda_ops, Bt, L, C, groups, dtype, act):
    x, w, b, _ = make(Bt, L, C, dtype, seed=Bt * 100 + L)
    y, mean, rstd = cuda_ops.group_norm_act(x.to(dev), w.to(dev), b.to(dev), groups, act=act, return_stats=True)
    ref = oracle_norm(x, w, b, groups, act=act)
    big, r = scales(x, w, b, groups)
    k = terms(L, C, groups) * 2.0 ** -24
    # SiLU: |act'| <= 1.1, and the bf16 form's exponential is off by up to 2^-21 (2 + |z|) of its value
    fast = 2.0 ** -21 * (2 + big) if act == "silu" and dtype == torch.bfloat16 else 0.0
    check(y, ref, HALF[dtype] * ref.abs() * 1.01 + (1.1 * k + fast) * big, "y")
    assert y.dtype == dtype and mean.shape == (Bt, groups)
    xg = x.double().reshape(Bt, L, groups, -1)
    check(mean, xg.mean((1, 3)), k * xg.abs().mean((1, 3)), "mean")
    check(rstd, r.reshape(Bt, groups), k * r.reshape(Bt, groups), "rstd")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,C,groups", [
    (5, 1, 32, 8), (3, 1, 96, 2), (2, 1, 21, 7), (300, 1, 2048, 32), (9, 1, 1030, 2), (3, 7, 8, 8), (2, 2, 64, 4),
    (3, 333, 48, 3), (1, 3000, 16, 2), (2, 130, 2560, 5), (4, 3, 35, 5),
])
def test_backward(cuda_ops, Bt, L, C, groups, dtype, act):
    x, w, b, dy = make(Bt, L, C, dtype, seed=Bt * 100 + L + 1)
    xd, wd, bd = (t.to(dev) for t in (x, w, b))
    _, mean, rstd = cuda_ops.group_norm_act(xd, wd, bd, groups, act=act, return_stats=True)
    dx, dw, db = cuda_ops.group_norm_act_bwd(dy.to(dev), xd, wd, bd, mean, rstd, act=act)
    leaves = [t.double().requires_grad_(True) for t in (x, w, b)]
    rx, rw, rb = torch.autograd.grad((oracle_norm(*leaves, groups, act=act) * dy.double()).sum(), leaves)
    big, r = scales(x, w, b, groups)
    fast = 2.0 ** -21 if act == "silu" and dtype == torch.bfloat16 else 0.0
    k = terms(L, C, groups) * 2.0 ** -24
    # dz = dy act'(z): |act'| <= 1.1, |act''| <= 0.5 carries z's own error
    dz = dy.double().abs()
    ez = dz * (1.1 * k + 0.5 * k * big + fast * (4 + 2 * big))
    n = (big / w.abs().clamp_min(1e-3)).clamp_max(1e6)
    gz = (dz * w.abs()).reshape(Bt, L, groups, -1)
    ng = n.reshape(Bt, L, groups, -1)
    # each of gr, mean(gr), n mean(gr n) with the error of its parts
    eg = (ez * w.abs()).reshape(Bt, L, groups, -1) + k * gz
    en = eg + eg.mean((1, 3), keepdim=True) + ng * ((eg * ng).mean((1, 3), keepdim=True) + 3 * k * (gz * ng).mean((1, 3), keepdim=True))
    check(dx, rx, HALF[dtype] * rx.abs() * 1.01 + (r * en * 1.5).reshape(Bt, L, C), "dx")
    kr = (80 + Bt * L / 8) * 2.0 ** -24
    check(dw, rw, ((ez + kr * dz) * n).sum((0, 1)) + 2.0 ** -24 * rw.abs(), "dweight")
    check(db, rb, (ez + kr * dz).sum((0, 1)) + 2.0 ** -24 * rb.abs(), "dbias")


@pytest.mark.gpu
def test_backward_against_differences(cuda_ops):
    x, w, b, dy = make(2, 37, 24, torch.float32, seed=3)
    xd, wd, bd = (t.to(dev) for t in (x, w, b))
    _, mean, rstd = cuda_ops.group_norm_act(xd, wd, bd, 3, return_stats=True)
    grads = cuda_ops.group_norm_act_bwd(dy.to(dev), xd, wd, bd, mean, rstd)
    g = torch.Generator().manual_seed(4)
    e = 1e-4   # central differences in f64: off by e^2 f''' / 6 and 1e-16 |f| / e
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=g).double()
        a = [t.double() for t in (x, w, b)]
        f = []
        for s in (e, -e):
            a2 = list(a)
            a2[i] = a[i] + s * d
            f.append((oracle_norm(*a2, 3) * dy.double()).sum())
        assert abs((f[0] - f[1]) / (2 * e) - (gr.double().cpu() * d).sum()) < 1e-5 * gr.double().cpu().abs().sum()


@pytest.mark.gpu
def test_large_mean_small_spread(cuda_ops):
    """Values around 1000 with a spread of 0.1: E[x^2] - E[x]^2 would keep nothing of the variance."""
    g = torch.Generator().manual_seed(8)
    x = 1000.0 + 0.1 * torch.randn(2, 400, 64, generator=g)
    w, b = torch.ones(64), torch.zeros(64)
    for t in (x, x[:, :1]):
        y = cuda_ops.group_norm_act(t.to(dev), w.to(dev), b.to(dev), 4, act="none")
        ref = oracle_norm(t, w, b, 4, act="none")
        # the mean is off by a few steps of 1000, 2^-14 each way, over a spread of 0.1
        assert (y.double().cpu() - ref).abs().max() < 4 * 2.0 ** -14 / 0.08


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3, 8), (2, 0, 8), (0, 8)])
def test_empty(cuda_ops, shape):
    x = torch.empty(shape, device=dev)
    w, b = torch.ones(8, device=dev), torch.zeros(8, device=dev)
    y, mean, rstd = cuda_ops.group_norm_act(x, w, b, 2, return_stats=True)
    dx, dw, db = cuda_ops.group_norm_act_bwd(x, x, w, b, mean, rstd)
    assert y.shape == x.shape and dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 50])
def test_strided_unaligned_and_repeated(cuda_ops, L):
    """A view at an odd offset takes the narrow accesses; results repeat bit for bit, also from a graph."""
    x, w, b, dy = make(6, L, 64, torch.bfloat16, seed=6)
    buf = torch.zeros(6 * L * 64 + 1, device=dev, dtype=torch.bfloat16)
    buf[1:] = x.to(dev).flatten()
    xo, wd, bd, dyd = buf[1:].view(6, L, 64), w.to(dev), b.to(dev), dy.to(dev)
    ref = cuda_ops.group_norm_act(x.to(dev), wd, bd, 4, return_stats=True)
    out = cuda_ops.group_norm_act(xo, wd, bd, 4, return_stats=True)
    assert (out[0].float() - ref[0].float()).abs().max() <= 2 ** -7 * ref[0].float().abs().max()
    first = cuda_ops.group_norm_act_bwd(dyd, xo, wd, bd, *out[1:])
    wide = torch.zeros(6, L, 128, device=dev, dtype=torch.bfloat16)
    wide[..., :64] = x.to(dev)
    assert torch.equal(cuda_ops.group_norm_act(wide[..., :64], wd, bd, 4), ref[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cuda_ops.group_norm_act_bwd(dyd, xo, wd, bd, *out[1:])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = cuda_ops.group_norm_act_bwd(dyd, xo, wd, bd, *out[1:])
    graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(first, again):
        assert torch.equal(a, c)


def test_refusals_without_gpu():
    import triton_ssm_b200 as ts
    x, w, b, dy = make(2, 3, 8, torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        ts.group_norm_act(x, w, b, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ts.group_norm_act_bwd(dy, x, w, b, torch.zeros(2, 2), torch.zeros(2, 2))
    from triton_ssm_b200.norm import _norm_args
    for bad in (dict(x=x.double()), dict(weight=w[:4]), dict(groups=3), dict(groups=0), dict(act="relu"),
                dict(x=x[0, 0]), dict(weight=w.bfloat16())):
        kw = dict(dict(x=x, weight=w, bias=b, groups=2, act="silu"), **bad)
        with pytest.raises(ValueError):
            _norm_args("group_norm_act", **kw)


def test_entry_point_refusals_without_gpu():
    """The C entry points check before they launch, so this runs without a device."""
    from triton_ssm_b200 import _lib
    lib = _lib.load_library()
    one = 4096   # a non-null address that nothing reads
    def fwd(Bt=2, L=3, C=8, groups=2, act=1, dtype=0, mean=one, rstd=one, ws=one, nbytes=1 << 20, x=one):
        return lib.tssm_group_norm_act(x, one, one, one, mean, rstd, ws, nbytes, Bt, L, C, groups, 1e-5, act, dtype, 0)
    for kw in (dict(Bt=-1), dict(groups=3), dict(groups=0), dict(act=2), dict(dtype=3), dict(x=0), dict(mean=0),
               dict(mean=0, rstd=0), dict(ws=0), dict(nbytes=1), dict(ws=one + 4), dict(C=1 << 24)):
        assert fwd(**kw) == 1, kw
        assert lib.tssm_last_error()
    assert fwd(Bt=0) == 0
    bwd = lib.tssm_group_norm_act_bwd
    assert bwd(one, one, one, one, one, one, one, one, one, one, 1, 2, 3, 8, 2, 1, 0, 0) == 1
    assert bwd(one, one, one, one, 0, one, one, one, one, one, 1 << 20, 2, 3, 8, 2, 1, 0, 0) == 1


def test_negative_eps_is_refused_without_gpu():
    from triton_ssm_b200 import _lib
    lib, one = _lib.load_library(), 4096   # a non-null address that nothing reads
    for eps in (-1e-5, float("nan")):
        assert lib.tssm_group_norm_act(one, one, one, one, one, one, one, 1 << 20, 2, 3, 8, 2, eps, 1, 0, 0) == 1


@pytest.mark.gpu
def test_eps_zero_negative_and_empty_maps(cuda_ops):
    x, w, b, _ = (t.to(dev) for t in make(2, 0, 8, torch.float32))
    _, mean, rstd = cuda_ops.group_norm_act(x, w, b, 2, eps=0, return_stats=True)
    assert not mean.any() and bool(rstd.isinf().all())
    with pytest.raises(ValueError, match="eps"):
        cuda_ops.group_norm_act(x, w, b, 2, eps=-1.0)
