"""What linear attention, its step, the 8-bit norm, quantiser and product refuse:
the public functions on fake GPU tensors, the C entries before any device call
(CPU); and the public functions traced into one graph."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mogt_amd import _lib, ops

F8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def on(device):
    return lambda *s, dtype=torch.float32: torch.empty(*s, device=device, dtype=dtype)


def attn_args(**change):
    e = on(change.pop("device", "cuda"))
    a = dict(q=e(2, 5, 2, 8), k=e(2, 5, 2, 8), v=e(2, 5, 4, 12), log_decay=e(2, 5, 4), initial_state=e(2, 4, 8, 12),
             lengths=e(2, dtype=torch.int32))
    a.update({k: v(e) for k, v in change.items()})
    return a


ATTN = [
    (dict(q=lambda e: e(5, 2, 8)), r"\[B, L, G, dk\]"),
    (dict(q=lambda e: e(2, 5, 2, 8, dtype=torch.float16)), "dtype"),
    (dict(k=lambda e: e(2, 5, 2, 8, dtype=BF16)), "one dtype"),
    (dict(v=lambda e: e(2, 5, 4, 12, dtype=BF16)), "one dtype"),
    (dict(k=lambda e: e(2, 5, 2, 7)), "same shape"),
    (dict(k=lambda e: e(2, 5, 4, 8)), "same shape"),
    (dict(v=lambda e: e(2, 4, 4, 12)), "v must"),
    (dict(v=lambda e: e(2, 5, 12)), "v must"),
    (dict(v=lambda e: e(2, 5, 3, 12), log_decay=lambda e: e(3)), "groups"),
    (dict(q=lambda e: e(2, 5, 0, 8), k=lambda e: e(2, 5, 0, 8)), "groups"),
    (dict(q=lambda e: e(2, 5, 2, 129), k=lambda e: e(2, 5, 2, 129)), "widths 129"),
    (dict(v=lambda e: e(2, 5, 4, 0), initial_state=lambda e: e(2, 4, 8, 0)), "widths 8 and 0"),
    (dict(log_decay=lambda e: e(2, 5, 2)), "log_decay must"),
    (dict(log_decay=lambda e: e(5, 4)), "log_decay must"),
    (dict(log_decay=lambda e: e(2, 5, 4, dtype=torch.int32)), "log_decay must be real"),
    (dict(log_decay=lambda e: e(4, dtype=torch.complex64)), "log_decay must be real"),
    (dict(initial_state=lambda e: e(2, 4, 12, 8)), "state"),
    (dict(initial_state=lambda e: e(2, 4, 8, 12, dtype=BF16)), "float32"),
    (dict(lengths=lambda e: e(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=lambda e: e(2)), "lengths"),
    (dict(lengths=lambda e: torch.empty(2, dtype=torch.int32)), "one device"),
    (dict(log_decay=lambda e: torch.empty(4)), "one device"),
    (dict(device="cpu"), "CUDA"),
]


@pytest.mark.parametrize("change,word", ATTN)
def test_attention_refuses(change, word):
    with FakeTensorMode():
        a = attn_args(**change)
        args = [a.pop(n) for n in ("q", "k", "v", "log_decay")]
        with pytest.raises(ValueError, match=word):
            ops.linear_attention(*args, **a)


@pytest.mark.parametrize("change,word", [
    (dict(q=lambda e: e(2, 1, 2, 8)), r"\[B, G, dk\]"),
    (dict(state=lambda e: e(3, 4, 8, 12)), "state"),
    (dict(state=lambda e: e(2, 4, 8, 12, dtype=BF16)), "float32"),
    (dict(state=lambda e: e(2, 4, 12, 8).transpose(2, 3)), "contiguous"),
    (dict(log_decay=lambda e: e(2, 2)), "log_decay must"),
    (dict(v=lambda e: e(3, 4, 12)), "v must"),
])
def test_step_refuses(change, word):
    with FakeTensorMode():
        e = on("cuda")
        a = dict(q=e(2, 2, 8), k=e(2, 2, 8), v=e(2, 4, 12), state=e(2, 4, 8, 12), log_decay=e(4))
        a.update({k: v(e) for k, v in change.items()})
        with pytest.raises(ValueError, match=word):
            ops.linear_attention_step(**a)


@pytest.mark.parametrize("change,word", [
    (dict(x=lambda e: e(3, 256, dtype=BF16)), "float32"),
    (dict(z=lambda e: e(3, 128)), "same shape"),
    (dict(z=lambda e: e(3, 256, dtype=torch.float16)), "dtype"),
    (dict(weight=lambda e: e(128)), "weight"),
    (dict(weight=lambda e: e(256, dtype=torch.complex64)), "weight must be real"),
    (dict(x=lambda e: e(3, 6), z=lambda e: e(3, 6), weight=lambda e: e(6)), "rows of 6"),
    (dict(x=lambda e: e(3, 4100), z=lambda e: e(3, 4100), weight=lambda e: e(4100)), "rows of 4100"),
    (dict(z=lambda e: torch.empty(3, 256)), "one device"),
    (dict(x=lambda e: torch.empty(3, 256)), "CUDA"),
])
def test_norm_refuses(change, word):
    with FakeTensorMode():
        e = on("cuda")
        a = dict(x=e(3, 256), z=e(3, 256, dtype=BF16), weight=e(256))
        a.update({k: v(e) for k, v in change.items()})
        with pytest.raises(ValueError, match=word):
            ops.add_rmsnorm_fp8(a["x"], a["z"], 1.0, a["weight"])


@pytest.mark.parametrize("x,rows,word", [
    (lambda e: e(3, 6), 1, "rows of 6"), (lambda e: e(3, 0), 1, "rows of 0"), (lambda e: e(3, 8, dtype=F8), 1, "dtype"),
    (lambda e: e(3, 8), 64, "blocks of 64"), (lambda e: e(2, 3, 8), 128, r"\[N, D\]"), (lambda e: e(8).sum(), 1, r"\[N, D\]"),
    (lambda e: torch.empty(3, 8), 1, "CUDA"),
])
def test_quantiser_refuses(x, rows, word):
    with FakeTensorMode():
        with pytest.raises(ValueError, match=word):
            ops.quantize_fp8(x(on("cuda")), block_rows=rows)


@pytest.mark.parametrize("change,word", [
    (dict(x=lambda e: e(5, 272)), "must be torch.float8"),
    (dict(w=lambda e: e(130, 272, dtype=torch.float8_e5m2)), "must be torch.float8"),
    (dict(x=lambda e: e(5, 256, dtype=F8)), "w \\[N, K\\]"),
    (dict(w=lambda e: e(1, 130, 272, dtype=F8)), "w \\[N, K\\]"),
    (dict(x=lambda e: e(5, 264, dtype=F8), w=lambda e: e(130, 264, dtype=F8)), "rows of 264"),
    (dict(x_scale=lambda e: e(5, 2)), "x_scale"),
    (dict(x_scale=lambda e: e(5, 3, dtype=BF16)), "scales must be float32"),
    (dict(w_scale=lambda e: e(1, 3)), "w_scale"),
    (dict(out_dtype=lambda e: torch.float16), "dtype"),
    (dict(w_scale=lambda e: torch.empty(2, 3)), "one device"),
])
def test_product_refuses(change, word):
    with FakeTensorMode():
        e = on("cuda")
        a = dict(x=e(5, 272, dtype=F8), x_scale=e(5, 3), w=e(130, 272, dtype=F8), w_scale=e(2, 3))
        a.update({k: v(e) for k, v in change.items()})
        with pytest.raises(ValueError, match=word):
            ops.linear_fp8(**a)


def test_traced_into_one_graph():
    """Shapes and types of the outputs and gradients without running a kernel."""
    with FakeTensorMode():
        a = attn_args()
        inputs = [a[n] for n in ("q", "k", "v", "log_decay", "initial_state")]

        def layer(q, k, v, g, s, x, z, weight, w, w_scale):
            out, state = ops.linear_attention(q, k, v, g, initial_state=s, lengths=a["lengths"], return_state=True)
            o = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], state, g[:, 0])
            res, x8, xs = ops.add_rmsnorm_fp8(x, z, 0.5, weight)
            y = ops.linear_fp8(x8, xs, w, w_scale, out_dtype=torch.float32)
            return out, state, o, res, y, *ops.quantize_fp8(z, block_rows=128)

        e = on("cuda")
        more = [e(3, 256), e(3, 256, dtype=BF16), e(256), e(130, 256, dtype=F8), e(2, 2)]
        got = torch.compile(layer, fullgraph=True, backend="eager")(*inputs, *more)
        assert [tuple(t.shape) for t in got] == [(2, 5, 4, 12), (2, 4, 8, 12), (2, 4, 12), (3, 256), (3, 130), (3, 256),
                                                 (1, 2)]
        carries = torch.empty(2, 4, 2, 12, 8, device="cuda")
        grads = ops._linear_attn_grad_op(a["v"], None, *inputs, a["lengths"], carries, 1.0, [True] * 5)
        assert [tuple(g.shape) for g in grads] == [tuple(t.shape) for t in inputs]


def test_packed_layouts_are_the_structures():
    packed, struct = _lib.LINEAR_ATTN_PROBLEM, _lib.LinearAttnProblem
    assert packed.size == ctypes.sizeof(struct)
    assert _lib.LINEAR_ATTN_GRADIENTS.size == ctypes.sizeof(_lib.LinearAttnGradients)
    values = list(range(1, len(struct._fields_) + 1))
    read = struct.from_buffer_copy(packed.pack(*values))
    assert [getattr(read, name) for name, _ in struct._fields_] == values


def problem(**change):
    p = _lib.LinearAttnProblem(1, 8, 4, 2, 8, 12, 64, 0, 0, 0, 1.0, 64, 64, 64, 64, None, None, 16, 128, 8, 16, 128, 8,
                               48, 384, 12, 4, 32, 1)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,rc,word", [
    (dict(batch=-1), -1, b"batch"), (dict(groups=0), -1, b"groups"), (dict(groups=3), -1, b"groups"),
    (dict(key_dim=129), -1, b"width"), (dict(value_dim=0), -1, b"width"), (dict(io_dtype=2), -1, b"dtype"),
    (dict(segment=0), -1, b"segment"), (dict(segment=48), -1, b"segment"), (dict(io_dtype=1, segment=32), -1, b"segment"),
    (dict(batch=21846), -1, b"batch"), (dict(heads=65536), -1, b"heads"), (dict(length=(1 << 30) + 1), -1, b"length"),
    (dict(length=1 << 30), -1, b"segments"), (dict(q=None), -1, b"null"), (dict(log_decay=None), -1, b"null"),
    (dict(lengths=64, lengths_bytes=2), -1, b"lengths"), (dict(q_row=-16), -1, b"strides"),
    (dict(v_row=1 << 28), -1, b"2^31"), (dict(g_row=1 << 28), -1, b"2^31"), (dict(length=65), -2, b"workspace"),
    (dict(batch=0), 0, b""), (dict(heads=0), 0, b""),
])
def test_attention_entry_refuses(change, rc, word):
    lib = _lib.load()
    p = problem(**change)
    assert lib.mogt_linear_attn_fwd(ctypes.byref(p), 64, None, None, None, 0, None) == rc
    assert word in lib.mogt_last_error()


def test_entries_refuse_null_and_small():
    lib = _lib.load()
    p, g = problem(), _lib.LinearAttnGradients()
    ref = ctypes.byref
    assert lib.mogt_linear_attn_fwd(None, 64, None, None, None, 0, None) == -1
    assert lib.mogt_linear_attn_fwd(ref(p), None, None, None, None, 0, None) == -1
    assert lib.mogt_linear_attn_workspace_bytes(None) == 0
    assert lib.mogt_linear_attn_workspace_bytes(ref(p)) == 0 < lib.mogt_linear_attn_workspace_bytes(ref(problem(length=65)))
    n = lib.mogt_linear_attn_bwd_workspace_bytes(ref(p))
    assert n > 0 == lib.mogt_linear_attn_bwd_workspace_bytes(ref(problem(segment=1)))
    assert lib.mogt_linear_attn_bwd(ref(p), 64, None, 64, None, 64, n, None) == -1
    assert lib.mogt_linear_attn_bwd(ref(p), 64, None, None, ref(g), 64, n, None) == -1
    assert lib.mogt_linear_attn_bwd(ref(p), None, None, 64, ref(g), 64, n, None) == -1
    assert lib.mogt_linear_attn_bwd(ref(p), 64, None, 64, ref(g), 64, n - 1, None) == -2
    assert lib.mogt_linear_attn_step(ref(p), 64, 64, None) == -1   # length 8
    assert lib.mogt_linear_attn_step(ref(problem(length=1)), None, 64, None) == -1

    assert lib.mogt_add_rmsnorm_fp8_fwd(64, 64, 1.0, 64, 64, 64, 64, 2, 6, 1e-6, 0, None) == -1
    assert lib.mogt_add_rmsnorm_fp8_fwd(64, 64, 1.0, 64, 64, 64, 64, 2, 4100, 1e-6, 0, None) == -1
    assert lib.mogt_add_rmsnorm_fp8_fwd(64, 64, 1.0, 64, 64, 64, 64, 2, 8, 1e-6, 2, None) == -1
    assert lib.mogt_add_rmsnorm_fp8_fwd(68, 64, 1.0, 64, 64, 64, 64, 2, 8, 1e-6, 0, None) == -1
    assert lib.mogt_add_rmsnorm_fp8_fwd(64, None, 1.0, 64, 64, 64, 64, 2, 8, 1e-6, 0, None) == -1
    assert lib.mogt_add_rmsnorm_fp8_fwd(None, None, 1.0, None, None, None, None, 0, 8, 1e-6, 0, None) == 0
    assert lib.mogt_quantize_fp8(64, 8, 64, 64, 2, 6, 0, 1, None) == -1
    assert lib.mogt_quantize_fp8(64, 4, 64, 64, 2, 8, 0, 1, None) == -1
    assert lib.mogt_quantize_fp8(64, 10, 64, 64, 2, 8, 0, 1, None) == -1
    assert lib.mogt_quantize_fp8(64, 8, 64, 64, 2, 8, 0, 2, None) == -1
    assert lib.mogt_quantize_fp8(64, 8, 64, 64, 2, 8, 3, 1, None) == -1
    assert lib.mogt_quantize_fp8(None, 8, 64, 64, 2, 8, 0, 1, None) == -1
    assert lib.mogt_quantize_fp8(64, 8, 64, 64, 65536 * 128, 8, 0, 128, None) == -1
    for a, word in ((dict(width=24), b"16"), (dict(ldx=16), b"16"), (dict(ldx=40), b"16"), (dict(x=65), b"aligned"),
                    (dict(w=None), b"null"), (dict(out=3), b"dtype"), (dict(ldx=1 << 23), b"2^22"),
                    (dict(rows=1 << 36, n=1 << 20), b"tiles")):
        d = dict(x=64, ldx=32, w=64, rows=3, n=5, width=32, out=0)
        d.update(a)
        assert lib.mogt_linear_fp8(d["x"], d["ldx"], 64, d["w"], 64, 64, d["rows"], d["n"], d["width"], d["out"], None) == -1, a
        assert word in lib.mogt_last_error(), a
    assert lib.mogt_linear_fp8(None, 32, None, None, None, None, 0, 5, 32, 0, None) == 0


@pytest.mark.parametrize("B,L,H,dk,dv", [(1, 1, 1, 1, 1), (1, 200, 12, 64, 64), (1, 32768, 16, 128, 128), (2, 8192, 12, 64, 64),
                                         (21845, 5000, 2, 64, 64), (1, 1 << 30, 1, 64, 64), (1, 3000, 65535, 128, 128), (0, 0, 0, 4, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_segments_are_whole_chunks_that_the_entry_takes(B, L, H, dk, dv, dtype):
    s = ops._linear_attn_segment(B, L, H, dk, dv, dtype)
    chunk = ops.LINEAR_ATTN_CHUNK[dtype]
    assert s % chunk == 0 and s >= chunk and -(-L // s) <= 1 << 20
    p = problem(batch=B, length=L, heads=H, groups=1, key_dim=dk, value_dim=dv, segment=s, io_dtype=int(dtype == BF16),
                q_row=dk, k_row=dk, v_row=H * dv, g_row=H)
    # several segments take a workspace; a problem that is refused takes none
    assert (_lib.load().mogt_linear_attn_workspace_bytes(ctypes.byref(p)) > 0) == (L > s and B * H > 0)
    assert _lib.load().mogt_linear_attn_bwd_workspace_bytes(ctypes.byref(p)) > 0 or B * H == 0


@pytest.mark.parametrize("shape", [(1, 2, 4, 12, 8), (1, 2, 5, 12, 8), (0,), (1, 2, 6, 8, 12)])
def test_gradient_refuses_the_carries_of_other_segments(shape):
    """300 steps are five segments of 64 and a final state: the kernels would read
    past fewer."""
    e = torch.zeros
    assert ops._linear_attn_segment(1, 300, 2, 8, 12, torch.float32) == 64
    with pytest.raises(ValueError, match="carries"):
        ops._linear_attn_grad_op.impl(e(1, 300, 2, 12), None, e(1, 300, 2, 8), e(1, 300, 2, 8), e(1, 300, 2, 12), e(1, 300, 2),
                                      None, None, e(*shape), 1.0, [True] * 4 + [False])
