"""The gated delta rule and the group norm together: streams that are prefilled,
stepped, checkpointed and resumed, and a layer's gradients through both."""
import pytest
import torch

from oracle.delta import gated_delta
from oracle.norm import group_norm_act as oracle_norm
from test_gpu_delta import make

dev = "cuda"


def layer(a, h0, w, b, scale, H):
    """Delta rule, then the norm per token and head, in 64 bits."""
    y, h = gated_delta(**a, scale=scale, h0=h0)
    Bt, L = y.shape[:2]
    return oracle_norm(y.reshape(Bt * L, 1, -1), w, b, H).reshape(Bt, L, -1), h


def off(out, ref):
    return ((out.double().cpu() - ref).norm() / ref.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_steps_checkpoint(cuda_ops, tmp_path, dtype):
    S, L, H, G, P, N, n = 3, 90, 4, 2, 64, 128, 80
    a, h0 = make(S, L, H, G, N, P, dtype, seed=31)
    g = torch.Generator().manual_seed(5)
    w, b = 1 + 0.2 * torch.randn(H * P, generator=g), 0.2 * torch.randn(H * P, generator=g)
    # the streams end at different lengths: the second prompt is padded from token 50 on
    for k in ("u", "B", "C", "dt", "beta"):
        a[k][1, 50:n] = 0
    ref, rh = layer(a, h0, w, b, N ** -0.5, H)
    d = {k: v.to(dev) for k, v in a.items()}
    st = cuda_ops.DeltaStream(S, H, P, N, d["A_log"], weight=w, bias=b, h0=h0.to(dev))

    def part(s):
        return [d["u"][:, s].flatten(2)] + [d[k][:, s] for k in ("B", "C", "dt", "beta")]

    outs = [st.prefill(*part(slice(0, n)))]
    st.save(tmp_path / "streams.pt")
    tail = [[t[:, 0] for t in part(slice(i, i + 1))] for i in range(n, L)]
    for x in tail:
        outs.append(st.step(*x)[:, None])
    out = torch.cat(outs, 1)
    live = torch.ones(S, L, dtype=torch.bool)
    live[1, 50:n] = False   # a padded token's output is the norm of zeros: the bias
    # y enters the norm with its own rounding (bf16: up to 2^-8), which the norm keeps relative to a
    # head's size; the norm's output rounds once more, and SiLU grows relative errors by 1.1 at most
    tol = (2.2 * 2.0 ** -8) if dtype == torch.bfloat16 else 2.0 ** -16
    assert off(out[live.to(dev)], ref[live]) < tol
    assert off(st.h, rh) < 2.0 ** -16 and st.tokens == L
    again = cuda_ops.DeltaStream.load(tmp_path / "streams.pt")
    assert again.tokens == n
    for i, x in enumerate(tail):
        assert torch.equal(again.step(*x), outs[1 + i][:, 0])
    assert torch.equal(again.h, st.h)


@pytest.mark.gpu
def test_two_streams_objects_on_two_cuda_streams(cuda_ops):
    """Two sets of streams advanced at once: workspaces are each call's own."""
    a, h0 = make(2, 200, 2, 2, 64, 64, torch.bfloat16, seed=33)
    d = {k: v.to(dev) for k, v in a.items()}
    args = [d["u"].flatten(2)] + [d[k] for k in ("B", "C", "dt", "beta")]
    want = cuda_ops.DeltaStream(2, 2, 64, 64, d["A_log"], h0=h0).prefill(*args)
    objs = [cuda_ops.DeltaStream(2, 2, 64, 64, d["A_log"], h0=h0) for _ in range(2)]
    cs = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for o, c in zip(objs, cs):
        with torch.cuda.stream(c):
            got.append(o.prefill(*args))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


@pytest.mark.gpu
def test_layer_gradients(cuda_ops):
    """Training through both operators in f32, against autograd in 64 bits."""
    Bt, L, H, G, P, N = 2, 100, 4, 2, 32, 64
    a, _ = make(Bt, L, H, G, N, P, torch.float32, seed=35)
    g = torch.Generator().manual_seed(6)
    w, b = 1 + 0.2 * torch.randn(H * P, generator=g), 0.2 * torch.randn(H * P, generator=g)
    dz = torch.randn(Bt, L, H * P, generator=g)
    d = {k: v.to(dev) for k, v in a.items()}
    args = (d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"])
    wd, bd = w.to(dev), b.to(dev)
    y, saved = cuda_ops.gated_delta_rule(*args, save=True)
    rows = y.view(Bt * L, H * P)
    _, mean, rstd = cuda_ops.group_norm_act(rows, wd, bd, H, return_stats=True)
    dy, dw, db = cuda_ops.group_norm_act_bwd(dz.to(dev).view(Bt * L, H * P), rows, wd, bd, mean, rstd)
    grads = cuda_ops.gated_delta_rule_bwd(*args, dy.view_as(y), saved)
    leaves = [t.double().requires_grad_(True) for t in (*a.values(), w, b)]
    out, _ = layer(dict(zip(a, leaves)), None, leaves[6], leaves[7], 1.0, H)
    ref = torch.autograd.grad((out * dz.double()).sum(), leaves)
    for name, x, r in zip(("u", "A_log", "B", "C", "dt", "beta", "w", "b"), (*grads[:6], dw, db), ref):
        # y's f32 error (2^-17 of a head's size) times rstd enters the norm's gradient, which divides
        # by the spread of a head of 32 values: a few times the delta rule's own 2^-15
        tol = 2.0 ** -12 if name == "A_log" else 2.0 ** -14
        assert off(x.reshape(r.shape), r) < tol, name


def test_refuses_cpu():
    import triton_ssm_b200 as ts
    with pytest.raises(ValueError, match="CUDA"):
        ts.DeltaStream(2, 2, 8, 8, torch.zeros(2))
