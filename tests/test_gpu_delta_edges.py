"""The gated delta rule and the group norm where their calls meet memory: states updated in place
and by captured steps, uninitialised buffers, many streams in f32, offsets behind 2^31."""
import pytest
import torch

from oracle.delta import gated_delta_grads
from test_gpu_delta import NAMES, check_grads, make, run_bwd
from test_gpu_norm import make as make_norm

dev = "cuda"


def on(a):
    d = {k: v.to(dev) for k, v in a.items()}
    return d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"]


@pytest.mark.gpu
def test_captured_step_sees_a_later_prefill(cuda_ops):
    """A step captured before a prefill replays on the state that the prefill left."""
    S, H, G, N, P = 3, 4, 2, 64, 64
    a, h0 = make(S, 71, H, G, N, P, torch.bfloat16, seed=41)
    u, A, B, C, dt, beta = on(a)
    st, eager = (cuda_ops.DeltaStream(S, H, P, N, A, h0=h0.to(dev)) for _ in range(2))
    first = [t[:, 0].contiguous() for t in (u, B, C, dt, beta)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        st.step(*first)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = st.step(*first)
    st.h.copy_(h0)
    for i in (0, 1):
        want = eager.step(*(t[:, i * 40] for t in (u, B, C, dt, beta)))
        for t, src in zip(first, (u, B, C, dt, beta)):
            t.copy_(src[:, i * 40])
        graph.replay()
        assert torch.equal(y, want) and torch.equal(st.h, eager.h)
        part = [t[:, 1:40] for t in (u, B, C, dt, beta)]
        assert torch.equal(st.prefill(*part), eager.prefill(*part)) and torch.equal(st.h, eager.h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,P,L", [(torch.bfloat16, 128, 128, 130), (torch.bfloat16, 24, 40, 70),
                                         (torch.float32, 64, 64, 130), (torch.float32, 16, 24, 0)])
def test_state_in_place(cuda_ops, dtype, N, P, L):
    a, h0 = make(2, L, 4, 2, N, P, dtype, seed=42)
    args, h = on(a), h0.to(dev)
    y, want = cuda_ops.gated_delta_rule(*args, h0=h, return_state=True)
    again, out = cuda_ops.gated_delta_rule(*args, h0=h, return_state=True, h_last=h)
    assert out is h and torch.equal(h, want) and torch.equal(again, y)
    for bad in (h[:1], h.double(), h.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(ValueError):
            cuda_ops.gated_delta_rule(*args, return_state=True, h_last=bad)
    with pytest.raises(ValueError):
        cuda_ops.gated_delta_rule(*args, h_last=h)


def soil(value):
    """Give the allocator free blocks that hold a value, large and small ones."""
    torch.cuda.empty_cache()
    keep = [torch.full((1 << 27,), value, device=dev)] + [torch.full((1 << 17,), value, device=dev) for _ in range(64)]
    torch.cuda.synchronize()
    del keep


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,H,G,N,P", [(2, 141, 4, 2, 128, 128), (2, 66, 2, 2, 18, 7), (1, 130, 2, 1, 64, 192)])
def test_rule_ignores_what_buffers_held(cuda_ops, Bt, L, H, G, N, P, dtype):
    a, h0 = make(Bt, L, H, G, N, P, dtype, seed=43)
    args, h = on(a), h0.to(dev)
    dy, dh = torch.randn(Bt, L, H * P, device=dev).to(dtype), torch.randn(Bt, H, P, N, device=dev)
    outs = []
    for value in (0.0, float("nan")):
        soil(value)
        y, hl, saved = cuda_ops.gated_delta_rule(*args, h0=h, return_state=True, save=True)
        soil(value)
        outs.append((y, hl) + tuple(cuda_ops.gated_delta_rule_bwd(*args, dy, saved, dh_last=dh)))
        assert all(bool(t.isfinite().all()) for t in outs[-1])
    assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.gpu
@pytest.mark.parametrize("Bt,L,C,groups", [(9, 1, 96, 4), (3, 77, 40, 5), (2, 1, 1030, 2), (3, 1000, 256, 4)])
def test_norm_ignores_what_buffers_held(cuda_ops, Bt, L, C, groups):
    x, w, b, dy = (t.to(dev) for t in make_norm(Bt, L, C, torch.float32, seed=44))
    outs = []
    for value in (0.0, float("nan")):
        soil(value)
        y, mean, rstd = cuda_ops.group_norm_act(x, w, b, groups, return_stats=True)
        soil(value)
        outs.append((y, mean, rstd) + tuple(cuda_ops.group_norm_act_bwd(dy, x, w, b, mean, rstd)))
        assert all(bool(t.isfinite().all()) for t in outs[-1])
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    again = x.clone()   # y may be x itself
    assert cuda_ops.group_norm_act(again, w, b, groups, y=again) is again and torch.equal(again, outs[0][0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,P", [(torch.float32, 8, 8), (torch.bfloat16, 12, 8)])
def test_many_narrow_streams_go_through_in_segments(cuda_ops, dtype, N, P):
    """As for the wide bf16 heads: segments of single chunks, and a row's results are the row's alone."""
    Bt, L, H = 2000, 130, 4
    a, h0 = make(2, L, H, 2, N, P, dtype, seed=45)
    dy, dh = torch.randn(2, L, H * P, device=dev).to(dtype), torch.randn(2, H, P, N, device=dev)

    def run(n):
        u, A, B, C, dt, beta = on(a)
        u, B, C, dt, beta, h, y, d = (t.repeat(n, *[1] * (t.dim() - 1)) for t in (u, B, C, dt, beta, h0.to(dev), dy, dh))
        args = (u, A, B, C, dt, beta)
        out, hl, saved = cuda_ops.gated_delta_rule(*args, h0=h, return_state=True, save=True)
        grads = cuda_ops.gated_delta_rule_bwd(*args, y, saved, dh_last=d)
        return [out, hl] + [g for n, g in zip(NAMES, grads) if n != "dA_log"]

    for x, y in zip(run(1), run(Bt // 2)):
        assert torch.equal(y[:2], x) and torch.equal(y[-2:], x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Bt,L,H,G,P", [(2, 70, 6, 2, 64), (1, 129, 16, 2, 128), (3, 65, 32, 2, 64), (2, 64, 7, 1, 192)])
def test_backward_of_shared_key_heads(cuda_ops, Bt, L, H, G, P, dtype):
    """Key heads with 3, 7, 8 and 16 value heads each: their gradients are summed in different ways."""
    N = 128
    a, h0 = make(Bt, L, H, G, N, P, dtype, seed=L + H)
    g = torch.Generator().manual_seed(H)
    dy, dh = torch.randn(Bt, L, H, P, generator=g).to(dtype), 0.3 * torch.randn(Bt, H, P, N, generator=g)
    grads = run_bwd(cuda_ops, a, h0, dy, dh, 0.3)
    check_grads(grads, gated_delta_grads(*a.values(), dy, scale=0.3, h0=h0, dh_last=dh), a, dtype, L)
    for x, y in zip(grads, run_bwd(cuda_ops, a, h0, dy, dh, 0.3)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_two_backwards_at_once_and_captured(cuda_ops):
    """Two calls on two streams, and both replayed from one graph, give what each gives alone."""
    work = []
    for seed, (Bt, L, H, G, P) in ((47, (4, 260, 8, 2, 128)), (48, (3, 200, 6, 6, 64))):
        a, h0 = make(Bt, L, H, G, 128, P, torch.bfloat16, seed=seed)
        args, h = on(a), h0.to(dev)
        dy = torch.randn(Bt, L, H * P, device=dev).bfloat16()
        _, saved = cuda_ops.gated_delta_rule(*args, h0=h, save=True)
        work.append((args, dy, saved))
    alone = [cuda_ops.gated_delta_rule_bwd(*w[0], w[1], w[2]) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]

    def both():
        out = []
        for s, (args, dy, saved) in zip(streams, work):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                out.append(cuda_ops.gated_delta_rule_bwd(*args, dy, saved))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        return out

    got = both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = both()
    for _ in range(2):
        for t in (t for o in again for t in o):
            t.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for one, x, y in zip(alone, got, again):
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(one, x, y))


def rand(*shape, dtype=torch.float32):
    return torch.randn(*shape, device=dev, dtype=dtype)


@pytest.mark.gpu
def test_step_behind_offset_2_31(cuda_ops):
    S, H, N, P = 8200, 16, 128, 128   # 2.15e9 state values
    h = torch.empty(S, H, P, N, device=dev).normal_()
    x, dt, beta = rand(S, H, P, dtype=torch.bfloat16), torch.rand(S, H, device=dev), torch.rand(S, H, device=dev)
    B, C, A = rand(S, 4, N, dtype=torch.bfloat16), rand(S, 4, N, dtype=torch.bfloat16), torch.zeros(H, device=dev)
    t = slice(S - 5, S)
    few = h[t].clone()
    y = cuda_ops.gated_delta_step(x, dt, h, A, B, C, beta)
    assert torch.equal(cuda_ops.gated_delta_step(x[t], dt[t], few, A, B[t], C[t], beta[t]), y[t])
    assert torch.equal(few, h[t])
    del h
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("Bt,L,C,groups", [(524400, 1, 4096, 32), (3, 175000, 4096, 16)])
def test_norm_behind_offset_2_31(cuda_ops, Bt, L, C, groups):
    x, dy = rand(Bt, L, C, dtype=torch.bfloat16), rand(Bt, L, C, dtype=torch.bfloat16)
    w, b = rand(C), rand(C)
    y, mean, rstd = cuda_ops.group_norm_act(x, w, b, groups, return_stats=True)
    dx = cuda_ops.group_norm_act_bwd(dy, x, w, b, mean, rstd)[0]
    y1, m1, r1 = cuda_ops.group_norm_act(x[-1:], w, b, groups, return_stats=True)
    assert torch.equal(y1, y[-1:]) and torch.equal(m1, mean[-1:]) and torch.equal(r1, rstd[-1:])
    assert torch.equal(cuda_ops.group_norm_act_bwd(dy[-1:], x[-1:], w, b, m1, r1)[0], dx[-1:])
    del x, dy, y, dx
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rule_behind_offset_2_31(cuda_ops, dtype):
    Bt, L, H, N, P = 8, 16400, 128, 64, 128   # 2.15e9 values, errors and saved states
    B, C = (rand(Bt, L, 1, N) for _ in range(2))
    B = torch.nn.functional.normalize(B, dim=-1)
    args = (rand(Bt, L, H * P, dtype=dtype), torch.zeros(H, device=dev), B.to(dtype), C.to(dtype),
            torch.rand(Bt, L, H, device=dev), torch.rand(Bt, L, H, device=dev))
    dy = rand(Bt, L, H * P, dtype=dtype)

    def run(s):
        part = tuple(t if t.dim() == 1 else t[s] for t in args)
        y, hl, saved = cuda_ops.gated_delta_rule(*part, return_state=True, save=True)
        grads = cuda_ops.gated_delta_rule_bwd(*part, dy[s], saved)
        return [t[-1:].clone() for t in [y, hl] + [g for n, g in zip(NAMES, grads) if n != "dA_log"]]

    for x, y in zip(run(slice(Bt - 1, Bt)), run(slice(0, Bt))):
        assert torch.equal(x, y)
    del args, dy
    torch.cuda.empty_cache()
