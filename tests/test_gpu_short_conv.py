"""Short causal convolution and its step (``ops.short_conv``,
``ops.short_conv_step``) against ``oracle/ssm_oracle.py``, and the two operators
of a layer in a row with the scan.

Tolerances, derived: S is the oracle's sum of absolute values.  A sum of K + 1
products rounds at most K + 1 times, 2^-24 each; silu and its slope add 8 for
the exponential and reciprocal and pass on at most 1.1 of the sum's error; the
slope's own change with the sum is at most 0.5 per unit, so the sum's error
counts up to 0.5 S_max (sums here stay below 16) more in the gradients.  The
gradients of weight and bias add one rounding per step: bound
(32 (K + 1) + 8 + B L) 2^-24 S, and half a step of the output's type."""
import pytest
import torch

from conftest import announce
from oracle import ssm_oracle as so

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(B, L, D, K, dtype=F32, bias=True, init=True, lengths=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = dict(x=r(B, L, D).to(dtype), weight=r(D, K), bias=r(D) if bias else None,
             initial_state=r(B, K - 1, D).to(dtype) if init else None)
    return t, None if lengths is None else torch.tensor(lengths, device="cuda")


def call(t, lengths, silu, **more):
    from mogt_amd import ops
    return ops.short_conv(t["x"], t["weight"], t["bias"], activation="silu" if silu else None,
                          initial_state=t["initial_state"], lengths=lengths, **more)


def check(name, got, want, mag, tol):
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.detach().double().cpu() - want).abs()
    lim = tol * mag + half * (want.abs() + tol * mag) + 1e-30
    assert bool((err <= lim).all()), f"{name}: {float((err / lim).max()):.3g} of the bound"


def run_both(t, lengths, silu, seed=1):
    B, L, D = t["x"].shape
    K = t["weight"].shape[1]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = torch.randn(B, L, D, generator=g, device="cuda").to(t["x"].dtype)
    ds = torch.randn(B, K - 1, D, generator=g, device="cuda").to(t["x"].dtype)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    y, state = call({**t, **leaves}, lengths, silu, return_state=True)
    grads = dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [dy, ds], allow_unused=K == 1)))
    kw = dict(silu=silu, initial_state=t["initial_state"], lengths=lengths, dy=dy, dstate=ds)
    want, mag = (so.short_conv(t["x"], t["weight"], t["bias"], **kw, mag=m) for m in (False, True))
    tol = (32 * (K + 1) + 8 + B * L) * 2.0 ** -24
    check("y", y, want["y"], mag["y"], tol)
    assert torch.equal(state.double().cpu(), want["state"])
    for k, v in grads.items():
        if v is not None:
            check("d" + k, v, want["d" + k], mag["d" + k], tol)
    return y, state, grads


@pytest.mark.parametrize("B,L,D,K,dtype", [
    (1, 1, 1, 4, F32), (2, 1, 64, 4, BF16), (1, 2, 8, 4, F32), (1, 3, 65, 4, BF16), (2, 8, 256, 4, F32),
    (1, 9, 512, 4, BF16), (3, 33, 513, 3, BF16), (2, 40, 260, 2, F32), (1, 64, 24, 1, BF16), (2, 31, 72, 8, BF16),
    (1, 50, 12, 5, F32), (1, 37, 16, 6, BF16), (2, 5, 16, 8, F32), (1, 70, 520, 7, BF16), (1, 1000, 16, 4, F32)])
@pytest.mark.parametrize("silu", [True, False])
def test_forward_and_gradients(gpu, B, L, D, K, dtype, silu):
    announce(f"short_conv B={B} L={L} D={D} K={K} {dtype} silu={silu}")
    run_both(*make(B, L, D, K, dtype, seed=L + K), silu)


@pytest.mark.parametrize("opt", [dict(bias=False), dict(init=False), dict(bias=False, init=False)])
def test_options(gpu, opt):
    run_both(*make(2, 19, 40, 4, **opt), True)


@pytest.mark.parametrize("lengths", [[40, 0, 1, 39], [0, 0, 0, 0], [2, 3, 8, 32], [99, -1, 40, 33]])
@pytest.mark.parametrize("K,dtype", [(4, F32), (4, BF16), (7, F32)])
def test_lengths(gpu, lengths, K, dtype):
    announce(f"short_conv lengths {lengths} K={K} {dtype}")
    t, n = make(4, 40, 32, K, dtype, lengths=lengths, seed=3)
    y, state, grads = run_both(t, n, True)
    for i, k in enumerate(lengths):
        k = min(max(k, 0), 40)
        assert not y[i, k:].any() and not grads["x"][i, k:].any()


def test_padding_is_not_read(gpu):
    t, n = make(3, 40, 32, 4, lengths=[40, 13, 0], seed=4)
    y, state, grads = run_both(t, n, True)
    bad = {**t, "x": t["x"].clone()}
    bad["x"][1, 13:] = float("nan")
    bad["x"][2] = float("inf")
    y2, state2, grads2 = run_both_values(bad, n)
    assert torch.equal(y2, y) and torch.equal(state2, state)
    for k in grads:
        assert torch.equal(grads2[k], grads[k]), k


def run_both_values(t, lengths):
    g = torch.Generator(device="cuda").manual_seed(1)
    dy = torch.randn(t["x"].shape, generator=g, device="cuda").to(t["x"].dtype)
    ds = torch.randn(t["initial_state"].shape, generator=g, device="cuda").to(t["x"].dtype)
    dy[1, 13:] = float("nan")
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    y, state = call(leaves, lengths, True, return_state=True)
    return y, state, dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [dy, ds])))


@pytest.mark.parametrize("K", [2, 3, 4, 5])
def test_infinities_stay_in_their_window(gpu, K):
    """An infinity reaches the K outputs of its window and no other."""
    t, _ = make(1, 30, 8, K, seed=5, init=False)
    t["x"][0, 10] = float("inf")
    y = call(t, None, False)
    hit = ~torch.isfinite(y[0]).all(-1)
    assert hit.nonzero().flatten().tolist() == list(range(10, 10 + K))


def test_strided_rows(gpu):
    t, _ = make(2, 21, 64, 4, BF16, seed=6)
    want = call(t, None, True)
    for off, width in ((0, 128), (8, 80), (1, 65), (3, 70)):
        proj = torch.zeros(2, 21, width, dtype=BF16, device="cuda")
        proj[..., off:off + 64] = t["x"]
        assert torch.equal(call({**t, "x": proj[..., off:off + 64]}, None, True), want), (off, width)
    time_first = t["x"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(call({**t, "x": time_first}, None, True), want)
    channel_slow = t["x"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(call({**t, "x": channel_slow}, None, True), want)


@pytest.mark.parametrize("shape", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_empty(gpu, shape):
    t, _ = make(*shape, 4)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    y, state = call(leaves, None, True, return_state=True)
    assert y.shape == shape and state.shape == (shape[0], 3, shape[2])
    if shape[1] == 0:
        assert torch.equal(state, t["initial_state"])
    grads = torch.autograd.grad([y, state], list(leaves.values()), [torch.ones_like(y), torch.ones_like(state)])
    for (k, v), g in zip(leaves.items(), grads):
        assert g.shape == v.shape
        assert bool((g == (1.0 if k == "initial_state" and shape[1] == 0 else 0.0)).all()) or g.numel() == 0


@pytest.mark.parametrize("B,D,K,dtype", [(1, 1, 4, F32), (3, 65, 4, BF16), (2, 512, 2, F32), (2, 40, 8, BF16),
                                         (2, 40, 1, F32), (300, 64, 4, BF16)])
@pytest.mark.parametrize("silu", [True, False])
def test_step(gpu, B, D, K, dtype, silu):
    from mogt_amd import ops
    t, _ = make(B, 1, D, K, dtype, seed=K)
    state = t["initial_state"].clone()
    y = ops.short_conv_step(t["x"][:, 0], state, t["weight"], t["bias"], activation="silu" if silu else None)
    kw = dict(silu=silu, initial_state=t["initial_state"])
    want, mag = (so.short_conv(t["x"], t["weight"], t["bias"], **kw, mag=m) for m in (False, True))
    check("y", y[:, None], want["y"], mag["y"], (2 * K + 12) * 2.0 ** -24)
    assert torch.equal(state.double().cpu(), want["state"])


def test_large_offsets(gpu):
    """Rows past 2^31 elements of their tensor."""
    rows, D = (1 << 31) // 1024 + 70, 1024
    announce(f"short_conv rows of a tensor of {rows} x {D} bf16")
    wide = torch.zeros(1, rows, D, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    tail = torch.randn(1, 64, D, generator=g, device="cuda").to(BF16)
    wide[:, -64:] = tail
    w, b = torch.randn(D, 4, generator=g, device="cuda"), torch.zeros(D, device="cuda")
    from mogt_amd import ops
    y = ops.short_conv(wide, w, b)
    assert torch.equal(y[:, -64:], ops.short_conv(tail, w, b))
    assert not y[:, :-64].any()


def test_runs_repeat_and_replay(gpu):
    """Bit-equal from run to run, on another stream, and from a captured graph
    replayed between eager calls."""
    t, _ = make(2, 300, 64, 4, BF16, seed=9)

    def once():
        leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
        y = call(leaves, None, True)
        return [y, *torch.autograd.grad(y, list(leaves.values()), torch.ones_like(y))]

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = once()
    for _ in range(3):
        for k in kept:
            k.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c, d in zip(kept, want, other, once()):
            assert torch.equal(a, b) and torch.equal(c, b) and torch.equal(d, b)


def test_layer_for_prompts_and_tokens(gpu):
    """The operators as a layer uses them: projection, convolution, step size
    and rows from its output, scan with gate.  A ragged batch of prompts in one
    call, then token by token, against the whole sequences run at once."""
    from mogt_amd import ops
    g = torch.Generator(device="cuda").manual_seed(10)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    B, L, D, N, K, R, T = 3, 24, 64, 16, 4, 8, 5
    xz = r(B, L + T, 2 * D)
    w, bias, to_rows, to_dt = r(D, K) / 2, 0.1 * r(D), r(R + 2 * N, D) / 8, r(D, R) / 4
    A, skip, dt_bias = -torch.rand(D, N, generator=g, device="cuda") * 4, r(D), r(D) - 3
    prompt = [24, 7, 1]

    def rows(u):
        low, Bm, Cm = (u @ to_rows.t()).split([R, N, N], -1)
        return low @ to_dt.t(), Bm, Cm

    def whole(seq):   # one sequence [n, 2 D], no cache
        u = ops.short_conv(seq[None, :, :D], w, bias, activation="silu")
        return ops.ssm_scan(u, *scan_args(u), D=skip, z=seq[None, :, D:], delta_bias=dt_bias, delta_softplus=True)[0]

    def scan_args(u):
        dt, Bm, Cm = rows(u)
        return dt, A, Bm, Cm

    lengths = torch.tensor(prompt, device="cuda")
    u, cs = ops.short_conv(xz[:, :L, :D], w, bias, activation="silu", lengths=lengths, return_state=True)
    out, hs = ops.ssm_scan(u, *scan_args(u), D=skip, z=xz[:, :L, D:], delta_bias=dt_bias, delta_softplus=True,
                           lengths=lengths, return_state=True)
    got = [[out[i, :n]] for i, n in enumerate(prompt)]
    for k in range(T):
        tok = torch.stack([xz[i, n + k] for i, n in enumerate(prompt)])
        u = ops.short_conv_step(tok[:, :D], cs, w, bias, activation="silu")
        dt, Bm, Cm = rows(u)
        o = ops.ssm_step(u, hs, dt, A, Bm, Cm, D=skip, z=tok[:, D:], delta_bias=dt_bias, delta_softplus=True)
        for i in range(B):
            got[i].append(o[i][None])
    for i, n in enumerate(prompt):
        want = whole(xz[i, :n + T])
        # fp32 throughout: the library's products may sum in another order for
        # another row count, 64 roundings of 2^-24 each; passed on through two
        # more sums of up to 29 steps and 16 states
        err = (torch.cat(got[i]) - want).abs().max()
        assert float(err) <= 64 * 29 * 2.0 ** -24 * float(want.abs().max())


def test_negated_gradient_of_the_state(gpu):
    """A gradient of the final state that is a lazily negated view."""
    t, _ = make(2, 20, 64, 4, F32, seed=11)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    g = torch.Generator(device="cuda").manual_seed(4)
    dy, ds = torch.randn(2, 20, 64, generator=g, device="cuda"), torch.randn(2, 3, 64, generator=g, device="cuda")
    for a, b in ((dy, torch._neg_view(ds)), (torch._neg_view(dy), ds)):
        assert a.is_neg() or b.is_neg()
        got, want = (torch.autograd.grad(list(call(leaves, None, True, return_state=True)), list(leaves.values()),
                                         list(d)) for d in ((a, b), (a.resolve_neg(), b.resolve_neg())))
        for k, u, v in zip(leaves, got, want):
            assert torch.equal(u, v), k


def test_lengths_of_four_bytes(gpu):
    t, n = make(3, 40, 32, 4, lengths=[40, 13, 0], seed=12)
    assert n.dtype == torch.int64
    wide, narrow = run_both(t, n, True), run_both(t, n.int(), True)
    for a, b in zip((*wide[:2], *wide[2].values()), (*narrow[:2], *narrow[2].values())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("K", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("B,L,D,dtype", [(32, 347, 130, F32), (32, 701, 130, BF16), (32, 517, 260, F32),
                                         (16, 1029, 520, BF16)])
def test_walks_of_several_blocks(gpu, B, L, D, K, dtype):
    """Enough waves for walks of 16 and 32 steps (two and four blocks), of single
    channels and of 16-byte vectors, with a last vector block that is not full
    and sequences that end inside a walk; in the backward more than the 128
    steps of a work-group.  Bounds as above, with the steps' term for the sums
    over steps only."""
    announce(f"short_conv walks B={B} L={L} D={D} K={K} {dtype}")
    lengths = [L, 0, 1, K, 31, 33, 128, 129, L - 1] + [L - 7 * i for i in range(1, B - 8)]
    t, n = make(B, L, D, K, dtype, lengths=lengths, seed=K)
    g = torch.Generator(device="cuda").manual_seed(1)
    dy = torch.randn(B, L, D, generator=g, device="cuda").to(dtype)
    ds = torch.randn(B, K - 1, D, generator=g, device="cuda").to(dtype)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    y, state = call(leaves, n, True, return_state=True)
    grads = torch.autograd.grad([y, state], list(leaves.values()), [dy, ds])
    kw = dict(silu=True, initial_state=t["initial_state"], lengths=n, dy=dy, dstate=ds)
    want, mag = (so.short_conv(t["x"], t["weight"], t["bias"], **kw, mag=m) for m in (False, True))
    assert torch.equal(state.double().cpu(), want["state"])
    for k, v in {"y": y, **{"d" + k: v for k, v in zip(leaves, grads)}}.items():
        steps = B * L if k in ("dweight", "dbias") else 0
        check(k, v, want[k], mag[k], (32 * (K + 1) + 8 + steps) * 2.0 ** -24)
