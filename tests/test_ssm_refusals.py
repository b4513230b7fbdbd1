"""What the selective scan, the short convolution and their steps refuse: the
public functions on fake GPU tensors, the C entries before any device call
(CPU); and the public functions traced into one graph."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mogt_amd import _lib, ops


def scan_args(**change):
    dev = change.pop("device", "cuda")
    e = lambda *s, dtype=torch.float32: torch.empty(*s, device=dev, dtype=dtype)  # noqa: E731
    a = dict(x=e(2, 5, 8), delta=e(2, 5, 8), A=e(8, 4), B=e(2, 5, 2, 4), C=e(2, 5, 2, 4), D=e(8), z=e(2, 5, 8),
             delta_bias=e(8), initial_state=e(2, 8, 4), lengths=e(2, dtype=torch.int32))
    a.update({k: v(e) for k, v in change.items()})
    return a


@pytest.mark.parametrize("change,word", [
    (dict(x=lambda e: e(5, 8)), r"\[B, L, D\]"),
    (dict(x=lambda e: e(2, 5, 8, dtype=torch.float16)), "dtype"),
    (dict(delta=lambda e: e(2, 5, 7)), "delta"),
    (dict(delta=lambda e: e(2, 5, 8, dtype=torch.bfloat16)), "delta"),
    (dict(z=lambda e: e(2, 4, 8)), "z must"),
    (dict(A=lambda e: e(7, 4)), "A must"),
    (dict(A=lambda e: e(8, 129)), "129 states"),
    (dict(A=lambda e: e(8, 0)), "0 states"),
    (dict(B=lambda e: e(2, 5, 4, 4)), "same shape"),
    (dict(B=lambda e: e(2, 5, 2, 3), C=lambda e: e(2, 5, 2, 3)), "B and C"),
    (dict(B=lambda e: e(2, 5, 3, 4), C=lambda e: e(2, 5, 3, 4)), "groups"),
    (dict(B=lambda e: e(2, 5, 0, 4), C=lambda e: e(2, 5, 0, 4)), "B and C"),
    (dict(B=lambda e: e(2, 5, 2, 4, dtype=torch.float64), C=lambda e: e(2, 5, 2, 4, dtype=torch.float64)), "dtype"),
    (dict(C=lambda e: e(2, 5, 2, 4, dtype=torch.bfloat16)), "dtype"),
    (dict(D=lambda e: e(9)), "D must"),
    (dict(delta_bias=lambda e: e(1)), "delta_bias"),
    (dict(initial_state=lambda e: e(2, 4, 8)), "state"),
    (dict(initial_state=lambda e: e(2, 8, 4, dtype=torch.bfloat16)), "float32"),
    (dict(lengths=lambda e: e(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=lambda e: e(2)), "lengths"),
    (dict(A=lambda e: torch.empty(8, 4)), "one device"),
    (dict(lengths=lambda e: torch.empty(2, dtype=torch.int32)), "one device"),
    (dict(device="cpu"), "CUDA"),
])
def test_scan_refuses(change, word):
    with FakeTensorMode():
        a = scan_args(**change)
        args = [a.pop(k) for k in ("x", "delta", "A", "B", "C")]
        with pytest.raises(ValueError, match=word):
            ops.ssm_scan(*args, **a)


@pytest.mark.parametrize("change,word", [
    (dict(x=lambda e: e(2, 1, 8)), r"\[B, D\]"),
    (dict(state=lambda e: e(3, 8, 4)), "state"),
    (dict(state=lambda e: e(2, 8, 4, dtype=torch.bfloat16)), "float32"),
    (dict(state=lambda e: e(2, 4, 8).transpose(1, 2)), "contiguous"),
    (dict(B=lambda e: e(2, 5), C=lambda e: e(2, 5)), "B and C"),
])
def test_step_refuses(change, word):
    with FakeTensorMode():
        e = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        a = dict(x=e(2, 8), state=e(2, 8, 4), delta=e(2, 8), A=e(8, 4), B=e(2, 4), C=e(2, 4))
        a.update({k: v(e) for k, v in change.items()})
        with pytest.raises(ValueError, match=word):
            ops.ssm_step(**a)


@pytest.mark.parametrize("change,word", [
    (dict(x=lambda e: e(5, 8)), r"\[B, L, D\]"),
    (dict(x=lambda e: e(2, 5, 8, dtype=torch.float16)), "dtype"),
    (dict(weight=lambda e: e(7, 4)), "weight"),
    (dict(weight=lambda e: e(8, 9)), "9 taps"),
    (dict(weight=lambda e: e(8, 0)), "0 taps"),
    (dict(bias=lambda e: e(7)), "bias"),
    (dict(activation=lambda e: "gelu"), "gelu"),
    (dict(initial_state=lambda e: e(2, 4, 8)), "state"),
    (dict(initial_state=lambda e: e(2, 3, 8, dtype=torch.bfloat16)), "dtype"),
    (dict(lengths=lambda e: e(1, dtype=torch.int64)), "lengths"),
    (dict(lengths=lambda e: e(2, dtype=torch.int16)), "lengths"),
    (dict(weight=lambda e: torch.empty(8, 4)), "one device"),
])
def test_conv_refuses(change, word):
    with FakeTensorMode():
        e = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        a = dict(x=e(2, 5, 8), weight=e(8, 4), bias=e(8), activation="silu", initial_state=e(2, 3, 8), lengths=None)
        a.update({k: v(e) for k, v in change.items()})
        args = [a.pop(k) for k in ("x", "weight", "bias")]
        with pytest.raises(ValueError, match=word):
            ops.short_conv(*args, **a)
        with pytest.raises(ValueError, match="contiguous"):
            ops.short_conv_step(e(2, 8), e(2, 8, 3).transpose(1, 2), e(8, 4))


class _Traced(Exception):
    pass


def test_traced_into_one_graph():
    """The public functions under a compiler: one graph, the ops in it; and
    the gradients' shapes on fake tensors."""
    with FakeTensorMode():
        a = scan_args()
        args = [a.pop(k).requires_grad_(True) for k in ("x", "delta", "A", "B", "C")]
        w = torch.empty(8, 4, device="cuda", requires_grad=True)

    def layer(x, delta, A, B, C, w):
        u = ops.short_conv(x, w, activation="silu")
        out, state = ops.ssm_scan(u, delta, A, B, C, **a, return_state=True)
        return out.sum() + state.sum()

    graphs = []

    def backend(gm, inputs):
        graphs.append(gm)

        def run(*_):
            raise _Traced

        return run

    torch._dynamo.reset()
    with pytest.raises(_Traced):
        torch.compile(layer, fullgraph=True, backend=backend)(*args, w)
    code = "".join(m.code for m in graphs[0].modules() if isinstance(m, torch.fx.GraphModule))
    assert len(graphs) == 1 and "mogt.ssm_scan" in code and "mogt.short_conv" in code
    with args[0].fake_mode, torch.no_grad():
        inputs = [*args, a["D"], a["z"], a["delta_bias"], a["initial_state"]]
        carries = torch.empty(2, 1, 4, 8, device="cuda")
        grads = ops._ssm_scan_grad_op(a["z"], None, *inputs[:8], a["lengths"], carries, True, [True] * 9)
        assert [tuple(g.shape) for g in grads] == [tuple(t.shape) for t in inputs]
        dx, dw, db, dinit = ops._short_conv_grad_op(a["z"], None, args[0], w, None, None, None, True, True, False)
        assert dx.shape == args[0].shape and dw.shape == w.shape and dinit.shape == (0,)


def test_packed_layouts_are_the_structures():
    assert _lib.SSM_PROBLEM.size == ctypes.sizeof(_lib.SsmProblem)
    assert _lib.SSM_GRADIENTS.size == ctypes.sizeof(_lib.SsmGradients)
    assert _lib.SHORT_CONV_PROBLEM.size == ctypes.sizeof(_lib.ShortConvProblem)
    for packed, struct in ((_lib.SSM_PROBLEM, _lib.SsmProblem), (_lib.SHORT_CONV_PROBLEM, _lib.ShortConvProblem)):
        values = list(range(1, len(struct._fields_) + 1))
        read = struct.from_buffer_copy(packed.pack(*values))
        assert [getattr(read, name) for name, _ in struct._fields_] == values


def scan_problem(**change):
    p = _lib.SsmProblem(1, 8, 8, 4, 1, 16, 0, 0, 0, 0, *[64] * 5, 64, None, None, None, None, 8, 64, 8, 64, 8, 64, 4,
                        32, 4, 32)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,rc,word", [
    (dict(states=0), -1, b"sizes"), (dict(states=129), -1, b"states"), (dict(batch=-1), -1, b"sizes"),
    (dict(groups=3), -1, b"groups"), (dict(io_dtype=2), -1, b"dtype"), (dict(bc_dtype=1), -1, b"dtype"),
    (dict(segment=12), -1, b"segment"), (dict(segment=0), -1, b"segment"), (dict(batch=65536), -1, b"batch"),
    (dict(length=1 << 31), -1, b"length"), (dict(x=None), -1, b"null"), (dict(lengths=64, lengths_bytes=2), -1, b"lengths"),
    (dict(io_dtype=0, bc_dtype=3), -1, b"dtype"), (dict(length=20), -2, b"workspace"),
    (dict(length=8 * 65536 * 2, segment=8), -1, b"segments"), (dict(batch=0), 0, b""),
])
def test_scan_entry_refuses(change, rc, word):
    lib = _lib.load()
    p = scan_problem(**change)
    assert lib.mogt_ssm_scan_fwd(ctypes.byref(p), 64, None, None, None, 0, None) == rc
    assert word in lib.mogt_last_error()


def test_entries_refuse_null_and_small():
    lib = _lib.load()
    p, g = scan_problem(), _lib.SsmGradients()
    assert lib.mogt_ssm_scan_fwd(None, 64, None, None, None, 0, None) == -1
    assert lib.mogt_ssm_scan_fwd(ctypes.byref(p), None, None, None, None, 0, None) == -1
    n = lib.mogt_ssm_scan_bwd_workspace_bytes(1, 8, 8, 4, 1, 16)
    assert n > 0 and lib.mogt_ssm_scan_bwd_workspace_bytes(1, 8, 8, 4, 3, 16) == 0
    assert lib.mogt_ssm_scan_bwd(ctypes.byref(p), 64, None, 64, None, 64, n, None) == -1
    assert lib.mogt_ssm_scan_bwd(ctypes.byref(p), 64, None, None, ctypes.byref(g), 64, n, None) == -1
    assert lib.mogt_ssm_scan_bwd(ctypes.byref(p), 64, None, 64, ctypes.byref(g), 64, n - 1, None) == -2
    g.dz, p.z = 64, None
    assert lib.mogt_ssm_scan_bwd(ctypes.byref(p), 64, None, 64, ctypes.byref(g), 64, n, None) == -1
    assert lib.mogt_ssm_step(ctypes.byref(p), 64, 64, None) == -1   # length 8
    assert lib.mogt_ssm_scan_workspace_bytes(1, 16, 8, 4, 16) == 0
    assert lib.mogt_ssm_scan_workspace_bytes(1, 17, 8, 4, 16) == 2 * 8 * 5 * 4

    c = _lib.ShortConvProblem(1, 8, 8, 4, 0, 1, 0, 64, 64, None, None, None, 8, 64)
    for k, v, word in (("taps", 9, b"taps"), ("taps", 0, b"taps"), ("io_dtype", 2, b"dtype"), ("length", -1, b"sizes"),
                       ("length", 1 << 27, b"length"), ("weight", None, b"null"), ("batch", 1 << 17, b"batch")):
        old = getattr(c, k)
        setattr(c, k, v)
        assert lib.mogt_short_conv_fwd(ctypes.byref(c), 64, None, None) == -1 and word in lib.mogt_last_error(), k
        setattr(c, k, old)
    assert lib.mogt_short_conv_fwd(ctypes.byref(c), None, None, None) == -1
    n = lib.mogt_short_conv_bwd_workspace_bytes(1, 8, 8, 4)
    assert lib.mogt_short_conv_bwd(ctypes.byref(c), 64, None, 64, 64, 64, None, 64, n - 1, None) == -2
    assert lib.mogt_short_conv_bwd(ctypes.byref(c), None, None, 64, 64, 64, None, 64, n, None) == -1
    assert lib.mogt_short_conv_step(ctypes.byref(c), 64, 64, None) == -1
    c.length = 1
    assert lib.mogt_short_conv_step(ctypes.byref(c), None, 64, None) == -1


@pytest.mark.parametrize("B,L,D,N,G", [(1, 1, 1, 1, 1), (1, 200, 1280, 16, 1), (1, 32768, 2048, 16, 1),
                                       (256, 4096, 2048, 64, 2), (3, 1001, 333, 24, 1), (1, 1 << 20, 64, 128, 1)])
def test_segments_are_whole_blocks_within_the_grid(B, L, D, N, G):
    s = ops._ssm_segment(B, L, D, N, G)
    assert s % 8 == 0 and s >= 8 and -(-L // s) <= max(1, ops.SSM_WAVES)


@pytest.mark.parametrize("L,D,N,word", [(1 << 25, 1, 64, "below 2\\^31"), (1, 1 << 22, 64, "below 2\\^28")])
def test_scan_refuses_what_its_backward_cannot_take(L, D, N, word):
    """Before the forward runs, and only where a gradient is recorded."""
    with FakeTensorMode():
        e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        a = [e(1, L, D), e(1, L, D), e(D, N), e(1, L, N), e(1, L, N)]
        assert ops.ssm_scan(*a).shape == (1, L, D)
        a[0].requires_grad_(True)
        with pytest.raises(ValueError, match=word):
            ops.ssm_scan(*a)
        with torch.no_grad():
            assert ops.ssm_scan(*a).shape == (1, L, D)


@pytest.mark.parametrize("B,L,D,N,G,segment", [(1, 2048, 2048, 16, 1, 24), (1, 2048, 2048, 16, 256, 24),
                                               (1, 2048, 2048, 16, 2048, 24), (2, 513, 768, 8, 1, 8),
                                               (3, 7, 70, 17, 7, 8), (1, 0, 5, 3, 1, 8)])
def test_gradient_workspace_goes_by_the_channels(B, L, D, N, G, segment):
    """As documented: the states by the channels, however few a group has; sums by
    the 64-channel blocks of the groups."""
    states = -(-L // 4) * N * 64 * -(-D // 64)
    sums = 2 * L * N * G * -(-(D // G) // 64)
    segments = max(1, -(-L // segment)) * D * (2 * N + 3)
    got = _lib.load().mogt_ssm_scan_bwd_workspace_bytes(B, L, D, N, G, segment)
    assert got == 4 * B * (states + sums + segments)


def test_scan_entry_refuses_more_blocks_than_a_launch_takes():
    lib = _lib.load()
    p = scan_problem(channels=(1 << 24) - 1, groups=(1 << 24) - 1, states=128)
    assert lib.mogt_ssm_scan_fwd(ctypes.byref(p), 64, None, None, None, 0, None) == -1
    assert b"launch" in lib.mogt_last_error()


@pytest.mark.parametrize("name", ["A", "D", "delta_bias"])
@pytest.mark.parametrize("dtype", [torch.complex64, torch.int32, torch.bool])
def test_scan_refuses_parameters_that_are_not_real(name, dtype):
    """A complex spectrum among them: a cast would run without its imaginary part."""
    with FakeTensorMode():
        shape = (8, 4) if name == "A" else (8,)
        a = scan_args(**{name: lambda e: e(*shape, dtype=dtype)})
        args = [a.pop(k) for k in ("x", "delta", "A", "B", "C")]
        with pytest.raises(ValueError, match=f"{name} must be real"):
            ops.ssm_scan(*args, **a)
        one = dict(x=args[0][:, 0], delta=args[1][:, 0], A=args[2], B=args[3][:, 0], C=args[4][:, 0], D=a["D"],
                   delta_bias=a["delta_bias"], state=a["initial_state"])
        with pytest.raises(ValueError, match=f"{name} must be real"):
            ops.ssm_step(**one)


@pytest.mark.parametrize("name", ["weight", "bias"])
def test_conv_refuses_parameters_that_are_not_real(name):
    with FakeTensorMode():
        e = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        p = dict(weight=e(8, 4), bias=e(8))
        p[name] = p[name].to(torch.complex64)
        with pytest.raises(ValueError, match=f"{name} must be real"):
            ops.short_conv(e(2, 5, 8), **p)
        with pytest.raises(ValueError, match=f"{name} must be real"):
            ops.short_conv_step(e(2, 8), e(2, 3, 8), **p)


@pytest.mark.parametrize("shape", [(1, 2, 4, 8), (1, 4, 4, 8), (0,), (1, 3, 8, 4)])
def test_gradient_refuses_the_carries_of_other_segments(shape):
    """17 steps are three segments of 8: the kernels would read past fewer."""
    e = torch.zeros
    assert ops._ssm_segment(1, 17, 8, 4, 1) == 8
    with pytest.raises(ValueError, match="carries"):
        ops._ssm_scan_grad_op.impl(e(1, 17, 8), None, e(1, 17, 8), e(1, 17, 8), e(8, 4), e(1, 17, 1, 4), e(1, 17, 1, 4),
                                   None, None, None, None, e(*shape), False, [True] * 5 + [False] * 3 + [True])
