"""The delta rule's backward: its workspace holds per-head parts of dB and dC only where a kernel writes them."""
import pytest
import torch

F32, BF16 = 0, 1


def sizes(Bt, L, H, G, P, N, dtype):
    from triton_ssm_b200 import _lib
    lib = _lib.load_library()
    return (lib.tssm_gated_delta_rule_bwd_workspace_size(Bt, L, H, G, P, N),
            lib.tssm_gated_delta_rule_bwd_workspace_size_dtype(Bt, L, H, G, P, N, dtype))


@pytest.mark.parametrize("H,G,P,N,dtype,parts", [
    (16, 8, 128, 128, BF16, False), (8, 1, 64, 128, BF16, False),   # summed in a cluster
    (16, 1, 64, 128, BF16, True), (16, 8, 64, 64, BF16, True), (16, 8, 96, 128, BF16, True), (16, 8, 128, 128, F32, True),
    (8, 8, 128, 128, BF16, False), (8, 8, 128, 128, F32, False),    # no shared key heads
])
def test_parts_of_shared_key_heads(H, G, P, N, dtype, parts):
    Bt, L = 4, 2048
    every, one = sizes(Bt, L, H, G, P, N, dtype)
    alone = sizes(Bt, L, H, H, P, N, dtype)[1]
    assert one - alone == (8 * Bt * L * H * N if parts else 0)
    assert every - alone == (8 * Bt * L * H * N if H != G else 0)


@pytest.mark.parametrize("Bt,L", [(0, 5), (2, 0), (-1, 5)])
def test_nothing_for_empty_calls(Bt, L):
    assert sizes(Bt, L, 4, 2, 128, 128, BF16) == (0, 0)


def test_refusals_name_the_bytes():
    """The entry point checks before it launches, so this runs without a device."""
    from triton_ssm_b200 import _lib
    lib, one = _lib.load_library(), 4096   # a non-null, aligned address that nothing reads
    every, least = sizes(2, 70, 4, 2, 128, 128, BF16)

    def bwd(nbytes, B=one, Bt=2):
        return lib.tssm_gated_delta_rule_bwd(one, one, B, one, one, one, one, one, one, 0, one, one, one, one, one, one,
                                             one, one, nbytes, Bt, 70, 4, 2, 128, 128, 1.0, BF16, 0)

    assert bwd(least - 1) == 1 and str(least) in lib.tssm_last_error().decode()
    assert bwd(every - 1, B=one + 2) == 1 and str(every) in lib.tssm_last_error().decode()   # the unaligned fallback's


@pytest.mark.gpu
def test_misaligned_tensors_take_the_larger_workspace(cuda_ops):
    """The C entry point with B at an odd offset: its fallback sums key heads from parts."""
    from triton_ssm_b200 import _lib
    from test_gpu_delta import make
    Bt, L, H, G, P, N, dev = 2, 70, 4, 2, 128, 128, "cuda"
    a, h0 = make(Bt, L, H, G, N, P, torch.bfloat16, seed=71)
    d = {k: v.to(dev) for k, v in a.items()}
    args = [d["u"].flatten(2), d["A_log"], d["B"], d["C"], d["dt"], d["beta"]]
    dy = torch.randn(Bt, L, H * P, device=dev).bfloat16()
    _, (states, errors) = cuda_ops.gated_delta_rule(*args, h0=h0.to(dev), save=True)
    want = cuda_ops.gated_delta_rule_bwd(*args, dy, (states, errors))
    buf = torch.zeros(d["B"].numel() + 1, device=dev, dtype=torch.bfloat16)
    buf[1:] = d["B"].flatten()
    args[2] = buf[1:]
    out = [torch.empty_like(t) for t in want]
    every, _ = sizes(Bt, L, H, G, P, N, BF16)
    ws = torch.full((every,), 255, device=dev, dtype=torch.uint8)   # f32 NaN
    _lib.call("tssm_gated_delta_rule_bwd", *(t.data_ptr() for t in args + [dy, states, errors]), None,
              *(t.data_ptr() for t in out), ws.data_ptr(), every, Bt, L, H, G, P, N, 1.0, BF16, 0)
    torch.cuda.synchronize()
    for x, y in zip(out, want):   # two kernels of f32 accuracy; bf16 results round to neighbours at most
        assert (x.float() - y.float()).norm() <= (2.0 ** -7 if x.dtype == torch.bfloat16 else 2.0 ** -14) * y.float().norm()
