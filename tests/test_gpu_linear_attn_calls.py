"""Calls of linear attention at the edges of what it takes."""
import pytest
import torch

from conftest import announce
from test_gpu_linear_attn import BF16, F32, call, gradients_in, make, run_all

pytestmark = pytest.mark.gpu


def test_shared_rows_past_a_launch_of_2_32_threads(gpu, monkeypatch):
    """2^32 values of q and of k, each shared by two heads (104 GB in all): their
    gradients against a call on the first and the last group of the last sequence."""
    from mogt_amd import ops
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        pytest.skip("needs 130 GB of free memory")
    B, L, G, dk, segment = 4, 65536, 128, 128, 8192
    announce(f"linear_attention gradients of {B} x {L} x {G} x {dk} shared rows")
    monkeypatch.setattr(ops, "_linear_attn_segment", lambda *a: segment)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.empty(B, L, G, dk, device="cuda", dtype=BF16).normal_(generator=g) for _ in "qk")
    v, dout = (torch.empty(B, L, 2 * G, 1, device="cuda", dtype=BF16).normal_(generator=g) for _ in "vo")
    decay = torch.rand(B, L, 2 * G, generator=g, device="cuda") * -0.1

    def gradients(*t, dout):
        leaves = [x.detach().requires_grad_(True) for x in t[:2]]
        return torch.autograd.grad(ops.linear_attention(*leaves, *t[2:]), leaves, dout)

    got = gradients(q, k, v, decay, dout=dout)
    for at in (0, G - 1):
        heads = slice(2 * at, 2 * at + 2)
        want = gradients(q[3:, :, at:at + 1], k[3:, :, at:at + 1], v[3:, :, heads], decay[3:, :, heads], dout=dout[3:, :, heads])
        for a, b in zip(got, want):
            assert bool(b.any()) and torch.equal(a[3:, :, at:at + 1], b)
    del q, k, v, dout, decay, got, want
    torch.cuda.empty_cache()


def test_a_training_forward_keeps_its_states_once(gpu):
    from mogt_amd import ops
    announce("linear_attention memory of a training forward")
    t, kw = make(2, 4096, 8, 8, 128, 128, BF16, init=False)
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items() if x is not None}
    call(leaves, kw)
    torch.cuda.synchronize()
    segments = 4096 // ops._linear_attn_segment(2, 4096, 8, 128, 128, BF16)
    states = 2 * 8 * (segments + 1) * 128 * 128 * 4
    assert segments > 8 and states > 30 << 20
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call(leaves, kw)
    assert torch.cuda.max_memory_allocated() - before < states + out.numel() * 2 + (4 << 20)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_query_gradient_alone_forms_no_reverse_states(gpu, dtype):
    """Through the C entry, on a workspace whose first part takes the reverse states;
    dq is the one of all."""
    from mogt_amd import _lib, ops
    announce(f"linear_attention dq alone {dtype}")
    t, kw = make(2, 700, 2, 2, 32, 48, dtype, seed=3)
    dout, dstate = gradients_in(t)
    want = run_all(t, kw, dout, dstate)[2]
    segment = ops._linear_attn_segment(2, 700, 2, 32, 48, dtype)
    scale = 32 ** -0.5
    _, _, carries = ops._linear_attn_op(t["q"], t["k"], t["v"], t["log_decay"], t["initial_state"], None, scale, True, True)
    p, held = ops._linear_attn_problem(t["q"], t["k"], t["v"], t["log_decay"], t["initial_state"], None, scale, segment)
    lib = _lib.load()
    ws = torch.full((lib.mogt_linear_attn_bwd_workspace_bytes(p),), 0x5a, device="cuda", dtype=torch.uint8)
    dq = torch.empty_like(t["q"])
    rc = lib.mogt_linear_attn_bwd(p, dout.data_ptr(), dstate.data_ptr(), carries.data_ptr(),
                                  _lib.LINEAR_ATTN_GRADIENTS.pack(dq.data_ptr(), 0, 0, 0, 0), ws.data_ptr(), ws.numel(),
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(dq, want)
    assert bool((ws[:carries.numel() * 4] == 0x5a).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_stride_of_a_single_step_is_any_number(gpu, dtype):
    announce(f"linear_attention of one step at a stride of 2^40 {dtype}")
    t, kw = make(3, 1, 2, 1, 32, 48, dtype, seed=4)
    dout, dstate = gradients_in(t)
    far = {n: x if n == "initial_state" else x.as_strided(x.shape, (x.stride(0), 1 << 40, *x.stride()[2:])) for n, x in t.items()}
    for a, b in zip(run_all(far, kw, dout, dstate), run_all(t, kw, dout, dstate)):
        assert torch.equal(a, b)
