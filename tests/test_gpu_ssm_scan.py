"""Selective state space scan and its step (``ops.ssm_scan``, ``ops.ssm_step``)
against the float64 loops of ``oracle/ssm_oracle.py``.

Tolerances, derived: every result is a sum of products, and its error is
measured against the same sum with absolute values (the oracle's ``mag``), S.
One rounding is 2^-24 of what it rounds.  The step size carries up to 24 of
them (its argument's, |raw| < 8 in the softplus's exponent, and the
exponential's, logarithm's and reciprocal's one or two ulp each); a decay takes
2 more and the product of t decays the sum of what they carry, at most
24 |A| sum(dt) exp(-|A| sum(dt)) < 9 for the step size's part plus 2 t <= 2 L.
The sums add at most one rounding per term in fp32: N states, L steps (dA, dD,
bias), D channels (dB, dC).  Each test's bound is (64 + 4 (L + N + D)) 2^-24 S.
With positive or no decay (A >= 0) the step size's part is not damped: 26 |A|
sum(dt) more.  bf16 outputs add half a step, 2^-8 of the value."""
import pytest
import torch

from conftest import announce
from oracle import ssm_oracle as so

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAMES = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state")


def make(B, L, D, N, G=1, dtype=torch.float32, z=True, softplus=True, skip=True, bias=True, init=True, lengths=None,
         seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    t = dict(x=r(B, L, D).to(dtype), delta=(0.7 * r(B, L, D)).to(dtype) if softplus else
             (0.1 * r(B, L, D).abs()).to(dtype), A=-torch.rand(D, N, generator=g, device=device) * 4,
             B=r(B, L, G, N).to(dtype), C=r(B, L, G, N).to(dtype))
    t["D"] = r(D) if skip else None
    t["z"] = r(B, L, D).to(dtype) if z else None
    t["delta_bias"] = (r(D) - 2 if softplus else 0.05 * r(D).abs()) if bias else None
    t["initial_state"] = r(B, D, N) if init else None
    kw = dict(delta_softplus=softplus, lengths=None if lengths is None else
              torch.tensor(lengths, device=device, dtype=torch.int32))
    return t, kw


def call(t, kw, **more):
    from mogt_amd import ops
    return ops.ssm_scan(t["x"], t["delta"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], delta_bias=t["delta_bias"],
                        initial_state=t["initial_state"], **kw, **more)


def bound(t, extra=0.0):
    B, L, D = t["x"].shape
    return (64 + 4 * (L + t["A"].shape[1] + D) + extra) * U


def check(name, got, want, mag, tol):
    got = got.detach()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.double().cpu() - want).abs()
    lim = tol * mag + half * (want.abs() + tol * mag) + 1e-30
    assert bool((err <= lim).all()), f"{name}: {float((err / lim).max()):.3g} of the bound"


def oracle(t, kw, **more):
    args = [t[k] for k in ("x", "delta", "A", "B", "C")]
    opt = {k: t[k] for k in ("D", "z", "delta_bias", "initial_state")}
    return [so.ssm_scan(*args, **opt, **kw, **more, mag=m) for m in (False, True)]


def run_both(t, kw, seed=1, tol=None):
    """Forward and all gradients, through both outputs, against the oracle."""
    B, L, D = t["x"].shape
    N = t["A"].shape[1]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dout = torch.randn(B, L, D, generator=g, device="cuda").to(t["x"].dtype)
    dstate = torch.randn(B, D, N, generator=g, device="cuda")
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    out, state = call({**{k: None for k in NAMES}, **leaves}, kw, return_state=True)
    grads = dict(zip(leaves, torch.autograd.grad([out, state], list(leaves.values()), [dout, dstate])))
    want, mag = oracle(t, kw, dout=dout, dstate=dstate)
    tol = bound(t) if tol is None else tol
    check("out", out, want["out"], mag["out"], tol)
    check("state", state, want["state"], mag["state"], tol)
    for k, v in grads.items():
        assert v.dtype == t[k].dtype
        check("d" + k, v, want["d" + k], mag["d" + k], tol)
    return out, state, grads


F32, BF16 = torch.float32, torch.bfloat16
SHAPES = [  # B, L, D, N, G, dtype: single tokens, edges of the 8-step blocks and of the segments, odd sizes
    (1, 1, 1, 1, 1, F32), (2, 1, 64, 16, 1, BF16), (1, 7, 65, 16, 1, F32), (1, 8, 64, 16, 1, BF16),
    (2, 9, 63, 3, 1, F32), (1, 16, 128, 16, 2, F32), (1, 17, 70, 8, 7, BF16), (3, 31, 130, 15, 1, BF16),
    (1, 33, 40, 16, 4, BF16), (1, 100, 64, 17, 1, F32), (2, 25, 66, 24, 2, BF16), (1, 40, 64, 64, 1, BF16),
    (1, 21, 64, 33, 1, F32), (1, 22, 33, 48, 1, BF16), (1, 26, 64, 56, 1, F32), (1, 13, 64, 60, 2, BF16),
    (1, 12, 64, 72, 1, F32), (1, 19, 65, 128, 1, F32), (1, 18, 10, 127, 5, BF16), (1, 300, 64, 16, 1, BF16), (2, 129, 192, 4, 3, F32),
]


@pytest.mark.parametrize("B,L,D,N,G,dtype", SHAPES)
def test_forward_and_gradients(gpu, B, L, D, N, G, dtype):
    announce(f"ssm_scan B={B} L={L} D={D} N={N} G={G} {dtype}")
    run_both(*make(B, L, D, N, G, dtype, seed=L))


@pytest.mark.parametrize("opt", [dict(z=False), dict(softplus=False), dict(skip=False), dict(bias=False),
                                 dict(init=False), dict(z=False, softplus=False, skip=False, bias=False, init=False)])
@pytest.mark.parametrize("dtype,N", [(F32, 16), (BF16, 40)])
def test_options(gpu, opt, dtype, N):
    announce(f"ssm_scan options {opt} {dtype}")
    run_both(*make(2, 37, 72, N, 1, dtype, seed=4, **opt))


@pytest.mark.parametrize("lengths", [[50, 0, 1, 49], [0, 0, 0, 0], [16, 17, 8, 9], [60, -3, 50, 32]])
@pytest.mark.parametrize("N", [16, 20])
def test_lengths(gpu, lengths, N):
    """Empty and single-token sequences, lengths at the edges of blocks and
    segments, and lengths outside the batch, which count as its ends."""
    announce(f"ssm_scan lengths {lengths} N={N}")
    t, kw = make(4, 50, 64, N, 2, F32, lengths=lengths, seed=2)
    out, state, grads = run_both(t, kw)
    for i, n in enumerate(lengths):
        n = min(max(n, 0), 50)
        for v in (out, grads["x"], grads["delta"], grads["z"], grads["B"], grads["C"]):
            assert not v[i, n:].any()
        if n == 0:
            assert torch.equal(state[i], t["initial_state"][i])


def test_padding_is_not_read(gpu):
    """NaN and infinities in the padded rows reach nothing."""
    t, kw = make(3, 40, 64, 16, 1, F32, lengths=[40, 13, 0], seed=3)
    clean = [o.clone() for o in call(t, kw, return_state=True)]
    bad = {k: v if v is None else v.clone() for k, v in t.items()}
    for k, v in (("x", float("nan")), ("delta", float("inf")), ("B", float("nan")), ("C", float("-inf")),
                 ("z", float("nan"))):
        bad[k][1, 13:] = v
        bad[k][2] = v
    for a, b in zip(call(bad, kw, return_state=True), clean):
        assert torch.equal(a, b)
    _, _, want = run_both(t, kw)
    leaves = {k: v.requires_grad_(True) for k, v in bad.items()}
    g = torch.Generator(device="cuda").manual_seed(1)
    dout = torch.randn(3, 40, 64, generator=g, device="cuda")
    dstate = torch.randn(3, 64, 16, generator=g, device="cuda")
    dout[1, 13:] = float("nan")
    got = torch.autograd.grad(list(call(leaves, kw, return_state=True)), list(leaves.values()), [dout, dstate])
    for k, v in zip(leaves, got):
        assert torch.equal(v, want[k]), k


def test_decays_of_zero_one_and_above(gpu):
    """A of 0 keeps the state for good, a large step size clears it, a positive A
    grows it."""
    t, kw = make(1, 60, 64, 16, seed=6)
    t["A"][:, 0] = 0.0
    t["A"][:, 1] = 0.05
    t["A"][:, 2] = -200.0
    t["delta"][0, 20] = 30.0
    run_both(t, kw, tol=bound(t, 26 * 0.05 * 40 + 26 * 4))


def test_long_sequence_in_many_segments(gpu):
    announce("ssm_scan 3000 steps")
    run_both(*make(1, 3000, 16, 16, 1, F32, seed=8))


def test_strided_rows(gpu):
    """Inputs as slices of wider projections, broadcast batches, transposed rows."""
    t, kw = make(2, 21, 64, 16, 2, BF16, seed=5)
    want = call(t, kw)
    proj = torch.zeros(2, 21, 3 * 64 + 2, dtype=BF16, device="cuda")
    proj[..., 1:65], proj[..., 66:130], proj[..., 130:194] = t["x"], t["z"], t["delta"]
    bc = torch.zeros(2, 21, 2 * 32 + 3, dtype=BF16, device="cuda")
    bc[..., 1:33], bc[..., 33:65] = t["B"].flatten(2), t["C"].flatten(2)
    s = {**t, "x": proj[..., 1:65], "z": proj[..., 66:130], "delta": proj[..., 130:194],
         "B": bc[..., 1:33].unflatten(-1, (2, 16)), "C": bc[..., 33:65].unflatten(-1, (2, 16))}
    assert torch.equal(call(s, kw), want)
    time_first = {k: v.transpose(0, 1).contiguous().transpose(0, 1) if k in ("x", "z", "delta", "B", "C") else v
                  for k, v in t.items()}
    assert torch.equal(call(time_first, kw), want)
    channel_slow = {**t, "x": t["x"].transpose(1, 2).contiguous().transpose(1, 2)}
    assert torch.equal(call(channel_slow, kw), want)
    one = {**t, "x": t["x"][:1].expand(2, -1, -1), "B": t["B"][:, :1].expand(-1, 21, -1, -1)}
    same = {k: v if v is None else v.contiguous() for k, v in one.items()}
    assert torch.equal(call(one, kw), call(same, kw))


def test_shared_rows_and_dtypes(gpu):
    """B and C without a group dimension, in fp32 beside bf16 rows, parameters in bf16."""
    from mogt_amd import ops
    t, kw = make(2, 30, 64, 16, 1, BF16, seed=7)
    want = call(t, kw)
    flat = {**t, "B": t["B"].squeeze(2), "C": t["C"].squeeze(2)}
    assert torch.equal(call(flat, kw), want)
    wide = {**t, "B": t["B"].float(), "C": t["C"].float()}
    assert torch.equal(call(wide, kw), want)
    half = {k: t[k].bfloat16() for k in ("A", "D", "delta_bias")}
    assert torch.equal(call({**t, **half}, kw), call({**t, **{k: v.float() for k, v in half.items()}}, kw))
    with torch.enable_grad():
        leaf = half["A"].requires_grad_(True)
        flat["B"] = flat["B"].requires_grad_(True)
        dA, dB = torch.autograd.grad(call({**flat, "A": leaf}, kw).float().sum(), [leaf, flat["B"]])
    assert dA.dtype == BF16 and dA.shape == leaf.shape and dB.shape == flat["B"].shape
    assert ops.ssm_scan(t["x"][:, :0], t["delta"][:, :0], t["A"], t["B"][:, :0], t["C"][:, :0]).shape == (2, 0, 64)


@pytest.mark.parametrize("shape", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_empty(gpu, shape):
    t, kw = make(*shape, 4, seed=1)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    out, state = call(leaves, kw, return_state=True)
    assert out.shape == shape and state.shape == (shape[0], shape[2], 4)
    if shape[1] == 0:
        assert torch.equal(state, t["initial_state"])
    grads = torch.autograd.grad([out, state], list(leaves.values()), [torch.ones_like(out), torch.ones_like(state)])
    for (k, v), g in zip(leaves.items(), grads):
        assert g.shape == v.shape
        assert bool((g == (1.0 if k == "initial_state" and shape[1] == 0 else 0.0)).all()) or g.numel() == 0


def test_gradient_is_the_difference_quotient(gpu):
    """Along a random direction of all inputs.  The quotient's own error: the
    rounding of two fp32 results, (bound S) / eps with eps = 2^-6, beside the
    eps^2 of the third derivative; measured against the sum of the gradient's
    magnitudes along the direction."""
    t, kw = make(1, 24, 32, 16, seed=12)
    leaves = {k: v.double().float().requires_grad_(True) for k, v in t.items()}
    g = torch.Generator(device="cuda").manual_seed(3)
    way = {k: torch.randn(v.shape, generator=g, device="cuda") for k, v in t.items()}
    dout = torch.randn(1, 24, 32, generator=g, device="cuda")
    grads = torch.autograd.grad(call(leaves, kw), list(leaves.values()), dout)
    along = sum(float((v.double() * way[k].double()).sum()) for k, v in zip(leaves, grads))
    eps = 2.0 ** -6

    def loss(s):
        return float((call({k: v + s * way[k] for k, v in t.items()}, kw).double() * dout.double()).sum())

    # four-point quotient: its error is eps^4 of the fifth derivative
    quotient = (8 * (loss(eps) - loss(-eps)) - (loss(2 * eps) - loss(-2 * eps))) / (12 * eps)
    size = sum(float((v.double() * way[k].double()).abs().sum()) for k, v in zip(leaves, grads))
    assert abs(quotient - along) <= 1e-3 * size


def test_pieces_and_steps_continue_one_another(gpu):
    """A prompt in one call, in pieces, and token by token: the same outputs and
    state up to the order of their roundings."""
    from mogt_amd import ops
    t, kw = make(2, 45, 96, 16, 1, F32, seed=10)
    want, wstate = call(t, kw, return_state=True)
    _, mag = oracle(t, kw)
    outs, state = [], t["initial_state"]
    rows = ("x", "delta", "B", "C", "z")
    for lo, hi in ((0, 20), (20, 21), (21, 40)):
        piece = {**t, **{k: t[k][:, lo:hi] for k in rows}, "initial_state": state}
        o, state = call(piece, kw, return_state=True)
        outs.append(o)
    for i in range(40, 45):
        s = {k: t[k][:, i] for k in rows}
        outs.append(ops.ssm_step(s["x"], state, s["delta"], t["A"], s["B"], s["C"], D=t["D"], z=s["z"],
                                 delta_bias=t["delta_bias"], delta_softplus=True)[:, None])
    check("out", torch.cat(outs, 1), want.double().cpu(), mag["out"], 2 * bound(t))
    check("state", state, wstate.double().cpu(), mag["state"], 2 * bound(t))


@pytest.mark.parametrize("B,D,N,G,dtype", [(1, 1, 1, 1, F32), (3, 65, 16, 1, BF16), (2, 130, 17, 2, F32),
                                           (5, 64, 128, 1, BF16), (2, 96, 6, 3, BF16), (300, 64, 16, 1, BF16)])
@pytest.mark.parametrize("plain", [False, True])
def test_step(gpu, B, D, N, G, dtype, plain):
    from mogt_amd import ops
    announce(f"ssm_step B={B} D={D} N={N} G={G} {dtype}")
    opt = dict(z=False, skip=False, bias=False, softplus=False) if plain else {}
    t, kw = make(B, 1, D, N, G, dtype, seed=N, **opt)
    state = t["initial_state"].clone()
    version = state._version
    one = {k: v if v is None or k not in ("x", "delta", "B", "C", "z") else v[:, 0] for k, v in t.items()}
    out = ops.ssm_step(one["x"], state, one["delta"], t["A"], one["B"], one["C"], D=t["D"], z=one["z"],
                       delta_bias=t["delta_bias"], delta_softplus=kw["delta_softplus"])
    assert state._version > version
    want, mag = oracle(t, kw)
    check("out", out[:, None], want["out"], mag["out"], bound(t))
    check("state", state, want["state"], mag["state"], bound(t))


def test_runs_repeat_bit_for_bit(gpu):
    t, kw = make(2, 500, 128, 16, 2, BF16, seed=11)
    first = [v for v in run_once_all(t, kw)]
    for a, b in zip(first, run_once_all(t, kw)):
        assert torch.equal(a, b)


def run_once_all(t, kw):
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    out, state = call(leaves, kw, return_state=True)
    return [out, state, *torch.autograd.grad([out, state], list(leaves.values()),
                                             [torch.ones_like(out), torch.ones_like(state)])]


def test_other_stream_and_two_calls_at_once(gpu):
    """Calls on two streams at a time, each with memory of its own."""
    t, kw = make(1, 400, 64, 16, 1, F32, seed=13)
    u, _ = make(1, 400, 64, 16, 1, F32, seed=14)
    want = call(t, kw), call(u, kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call((t, u)[i], kw))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_captured_graphs(gpu):
    """Forward, backward and steps in two captured graphs, replayed in turn with
    eager calls between; every replay equals the eager result."""
    from mogt_amd import ops
    sets = [make(1, 200, 64, 16, 1, F32, seed=s) for s in (20, 21)]
    wants = [[v.clone() for v in run_once_all(*s)] for s in sets]
    step_state = sets[0][0]["initial_state"].clone()

    def step():
        t = sets[0][0]
        return ops.ssm_step(t["x"][:, 0], step_state, t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0])

    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            run_once_all(*s)
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = run_once_all(*s)
            if s is sets[0]:
                o = o + [step()]
        graphs.append(g)
        outs.append(o)
    fresh = sets[0][0]["initial_state"].clone()
    for turn in range(4):
        step_state.copy_(fresh)
        eager = fresh.clone()
        t = sets[0][0]
        want_step = ops.ssm_step(t["x"][:, 0], eager, t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0])
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            for k, (a, b) in enumerate(zip(outs[i], wants[i])):
                assert torch.equal(a, b), (turn, i, k)
        assert torch.equal(outs[0][-1], want_step) and torch.equal(step_state, eager)
        assert torch.equal(call(*sets[1]), wants[1][0])


def test_partial_gradients_and_second_derivatives(gpu):
    """Only what is asked for is formed; a second derivative is refused."""
    t, kw = make(1, 20, 64, 16, seed=15)
    full = dict(zip(NAMES, run_once_all(t, kw)[2:]))
    assert list(t) == ["x", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state"]
    for k in NAMES:
        leaf = {**t, k: t[k].detach().requires_grad_(True)}
        out, state = call(leaf, kw, return_state=True)
        (g,) = torch.autograd.grad([out, state], [leaf[k]], [torch.ones_like(out), torch.ones_like(state)])
        assert torch.equal(g, full[k]), k
    x = t["x"].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(call({**t, "x": x}, kw).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("lengths", [None, [4200, 4111]])
def test_more_segments_than_are_folded_at_once(gpu, lengths):
    """525 segments of 8 steps: the carries go round three times (256 segments a
    time), with a channel block that is not full and a sequence that ends early."""
    announce(f"ssm_scan 4200 steps {lengths}")
    run_both(*make(2, 4200, 70, 2, 1, F32, lengths=lengths, seed=16))


@pytest.mark.parametrize("N", [9, 12, 20, 28, 32, 40, 41])
def test_states_of_a_wave(gpu, N):
    """State counts on both sides of each rule for how many a wave holds."""
    announce(f"ssm_scan N={N}")
    run_both(*make(1, 35, 66, N, 1, BF16, seed=N))


def test_rows_past_32_bit_offsets(gpu):
    """Row strides that put x, delta and B beyond 2^31 elements."""
    announce("ssm_scan rows past 2^31 elements")
    t, kw = make(1, 20, 64, 16, 1, BF16, seed=17)
    far = dict(t)
    base = torch.zeros(2_500_000_000, dtype=BF16, device="cuda")
    for i, k in enumerate(("x", "delta", "B")):
        v = t[k]
        view = base.as_strided(v.shape, (0, 130_000_000, *v.stride()[2:]), 1000 * i)
        view.copy_(v)
        far[k] = view
    for a, b in zip(run_once_all(far, kw), run_once_all(t, kw)):
        assert torch.equal(a, b)


def test_one_tensor_in_several_places(gpu):
    """x given as delta and as z too, B as C: the gradients add up."""
    from mogt_amd import ops
    t, _ = make(1, 30, 64, 16, 1, F32, seed=18)
    x, B = t["x"].detach().requires_grad_(True), t["B"].detach().requires_grad_(True)
    shared = torch.autograd.grad(ops.ssm_scan(x, x, t["A"], B, B, z=x, delta_softplus=True).sum(), (x, B))
    own = [v.detach().clone().requires_grad_(True) for v in (x, x, x, B, B)]
    out = ops.ssm_scan(own[0], own[1], t["A"], own[3], own[4], z=own[2], delta_softplus=True)
    g = torch.autograd.grad(out.sum(), own)
    # three terms in either order: two roundings of the sum of their magnitudes
    for got, parts in ((shared[0], g[:3]), (shared[1], g[3:])):
        want, mag = sum(p.double() for p in parts), sum(p.double().abs() for p in parts)
        assert bool(((got.double() - want).abs() <= 2 * 2.0 ** -24 * mag + 1e-30).all())


def growing(L, zero_rows, N=4, D=66, quiet=None, seed=30, init=None):
    """A of 1, 0.5, 0 and -1, steps of 1: zero input rows first, then 30 with
    values; output gradients in the first rows up to ``quiet`` only."""
    t, kw = make(1, L, D, N, 1, F32, z=False, softplus=False, bias=False, init=init is not None, seed=seed)
    t["delta"].fill_(1.0)
    t["A"][:] = torch.tensor([1.0, 0.5, 0.0, -1.0], device="cuda")[:N]
    t["x"][:, :zero_rows] = 0.0
    if init is not None:
        t["initial_state"].fill_(init)
    return t, kw


@pytest.mark.parametrize("segment", [8, 104, 400])
def test_growth_over_zero_rows(gpu, monkeypatch, segment):
    """A decay above one, exp(400) in all, on a state of zero: the state stays
    zero until the first value, and the gradient zero after the last one."""
    from mogt_amd import ops
    announce(f"ssm_scan growth, segments of {segment}")
    monkeypatch.setattr(ops, "SSM_MIN_SEGMENT", segment)
    t, kw = growing(400, 370)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    out, state = call({**{k: None for k in NAMES}, **leaves}, kw, return_state=True)
    dout = torch.zeros_like(out)
    dout[:, :30] = torch.randn(1, 30, 66, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    want, mag = oracle(t, kw, dout=dout, dstate=torch.zeros_like(state))
    tol = bound(t, 26 * 60)   # 30 steps of A = 1 forward and 30 backward, undamped
    check("out", out, want["out"], mag["out"], tol)
    check("state", state, want["state"], mag["state"], tol)
    for k, g in zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout)):
        check("d" + k, g, want["d" + k], mag["d" + k], tol)


@pytest.mark.parametrize("segment", [8, 104])
def test_growth_of_a_small_state(gpu, monkeypatch, segment):
    """exp(104) = 1.5e45 lies beyond fp32, exp(104) 1e-30 does not; and the same
    for the gradient on its way back."""
    from mogt_amd import ops
    monkeypatch.setattr(ops, "SSM_MIN_SEGMENT", segment)
    t, kw = growing(130, 130, init=1e-30)
    t["delta"][:, 104:] = 0.0
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    out, state = call({**{k: None for k in NAMES}, **leaves}, kw, return_state=True)
    dout, dstate = torch.zeros_like(out), torch.full_like(state, 1e-20)
    want, mag = oracle(t, kw, dout=dout, dstate=dstate)
    tol = bound(t, 26 * 208)
    check("state", state, want["state"], mag["state"], tol)
    for k, g in zip(leaves, torch.autograd.grad([out, state], list(leaves.values()), [dout, dstate])):
        check("d" + k, g, want["d" + k], mag["d" + k], tol)


def test_negated_gradient_of_the_state(gpu):
    """A gradient of the final state that is a lazily negated view."""
    t, kw = make(1, 20, 64, 16, 1, F32, seed=31)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    g = torch.Generator(device="cuda").manual_seed(4)
    dout = torch.randn(1, 20, 64, generator=g, device="cuda")
    dstate = torch.randn(1, 64, 16, generator=g, device="cuda")
    for a, b in ((dout, torch._neg_view(dstate)), (torch._neg_view(dout), dstate)):
        assert a.is_neg() or b.is_neg()
        got, want = (torch.autograd.grad(list(call(leaves, kw, return_state=True)), list(leaves.values()), list(d))
                     for d in ((a, b), (a.resolve_neg(), b.resolve_neg())))
        for k, u, v in zip(leaves, got, want):
            assert torch.equal(u, v), k


@pytest.mark.parametrize("N", [8, 16, 24, 64])
def test_infinity_in_a_channel_block_that_is_not_full(gpu, N):
    """An infinite input of the last channel makes infinities of the sums over
    the channels, as in the definition: idle lanes add nothing to them."""
    t, kw = make(1, 10, 65, N, 1, F32, z=False, seed=33)
    t["x"][0, 6, 64] = float("inf")
    g = torch.Generator(device="cuda").manual_seed(5)
    dout = torch.randn(1, 10, 65, generator=g, device="cuda")
    want, _ = oracle(t, kw, dout=dout)
    leaves = {k: t[k].detach().requires_grad_(True) for k in ("B", "C")}
    got = torch.autograd.grad(call({**t, **leaves}, kw), list(leaves.values()), dout)
    for k, v in zip(leaves, got):
        v, w = v.double().cpu(), want["d" + k]
        assert bool(w[0, 6].isinf().all()) and not w.isnan().any()
        assert torch.equal(v.isnan(), w.isnan()) and torch.equal(v.isinf(), w.isinf()), k
        assert torch.equal(v[v.isinf()].sign(), w[w.isinf()].sign()), k


@pytest.mark.parametrize("N", [8, 16, 24, 64])
@pytest.mark.parametrize("L", [5, 6, 7, 8])
def test_infinity_in_the_last_step(gpu, N, L):
    """An infinite last input reaches the last output only: no gradient of A goes
    through its state."""
    t, kw = make(1, L, 64, N, 1, F32, z=False, seed=34)
    t["x"][0, L - 1, 3] = float("inf")
    g = torch.Generator(device="cuda").manual_seed(5)
    dout = torch.randn(1, L, 64, generator=g, device="cuda")
    want, mag = oracle(t, kw, dout=dout)
    A = t["A"].detach().requires_grad_(True)
    (dA,) = torch.autograd.grad(call({**t, "A": A}, kw), [A], dout)
    assert bool(want["dA"].isfinite().all())
    check("dA", dA, want["dA"], mag["dA"], bound(t))


def test_a_group_for_every_channel(gpu):
    """More groups than a grid's second dimension holds."""
    announce("ssm_scan 65600 groups")
    t, kw = make(1, 3, 65600, 2, 65600, F32, seed=35)
    run_both(t, kw, tol=(64 + 4 * (3 + 2 + 1)) * U)


def test_the_most_channels(gpu):
    """Sums of more columns than one dimension of a launch takes: the channels'
    gradients are those of a call on a part of them."""
    announce("ssm_scan 16700032 channels")
    D, N, part = 16_700_032, 15, 64_000
    g = torch.Generator(device="cuda").manual_seed(36)
    x, delta, dout = (torch.randn(1, 1, D, generator=g, device="cuda") for _ in range(3))
    A = torch.rand(D, N, generator=g, device="cuda").neg_()
    B, C = (torch.randn(1, 1, N, generator=g, device="cuda") for _ in range(2))
    skip, bias = (torch.randn(D, generator=g, device="cuda") for _ in range(2))

    def grads(at):
        from mogt_amd import ops
        leaves = [v[at].detach().requires_grad_(True) for v in (A, skip, bias)]
        out = ops.ssm_scan(x[..., at], delta[..., at], leaves[0], B, C, D=leaves[1], delta_bias=leaves[2],
                           delta_softplus=True, initial_state=torch.ones_like(leaves[0])[None])
        return torch.autograd.grad(out, leaves, dout[..., at])

    whole = grads(slice(None))
    for at in (slice(0, part), slice(D - part, D)):
        for a, b in zip(whole, grads(at)):
            assert torch.equal(a[at], b)


@pytest.mark.parametrize("N", [8, 16, 24, 64])
def test_float32_rows_of_b_and_c_beside_bf16(gpu, N):
    """Gradients and steps with B and C in fp32 and the other rows in bf16."""
    from mogt_amd import ops
    announce(f"ssm_scan fp32 B and C beside bf16, N={N}")
    t, kw = make(2, 21, 66, N, 1, BF16, seed=N + 1)
    g = torch.Generator(device="cuda").manual_seed(N)
    t["B"], t["C"] = (torch.randn(2, 21, 1, N, generator=g, device="cuda") for _ in range(2))
    run_both(t, kw)
    state = t["initial_state"].clone()
    one = {k: t[k][:, 0] for k in ("x", "delta", "B", "C", "z")}
    out = ops.ssm_step(one["x"], state, one["delta"], t["A"], one["B"], one["C"], D=t["D"], z=one["z"],
                       delta_bias=t["delta_bias"], delta_softplus=True)
    first = {k: v[:, :1] if k in one else v for k, v in t.items()}
    want, mag = oracle(first, kw)
    check("out", out[:, None], want["out"], mag["out"], bound(first))
    check("state", state, want["state"], mag["state"], bound(first))


def test_lengths_of_eight_bytes(gpu):
    t, kw = make(3, 30, 64, 16, 1, F32, lengths=[30, 0, 13], seed=32)
    wide = dict(kw, lengths=kw["lengths"].long())
    for a, b in zip(run_once_all(t, wide), run_once_all(t, kw)):
        assert torch.equal(a, b)
    run_both(t, wide)


def roundings(name, t):
    """The sums an output really runs over: states for all, channels for dB and
    dC, the batch's steps for what channels share, and twice the steps for the
    product of decays that every state and gradient of a state carries."""
    B, L, D = t["x"].shape
    n = 64 + 4 * t["A"].shape[1] + 2 * L
    return (n + (4 * D if name in ("dB", "dC") else 4 * B * L if name in ("dA", "dD", "ddelta_bias") else 0)) * U


@pytest.mark.parametrize("segment", [24, 56, 304])
@pytest.mark.parametrize("N,G,dtype", [(8, 1, F32), (16, 1, BF16), (12, 2, F32), (24, 1, BF16), (40, 1, F32),
                                       (64, 1, BF16), (128, 2, F32)])
@pytest.mark.parametrize("ragged", [False, True])
def test_segments_of_several_blocks(gpu, monkeypatch, segment, N, G, dtype, ragged):
    """Long calls walk many blocks of steps a segment, short ones a single one:
    here 3, 7 and all of them, with a last block that is not full, a channel
    block that is not full, and sequences that end inside a later block, at a
    segment's end and one step past it."""
    from mogt_amd import ops
    announce(f"ssm_scan segments of {segment} N={N} G={G} {dtype} ragged={ragged}")
    monkeypatch.setattr(ops, "SSM_MIN_SEGMENT", segment)
    lengths = [151, 93, 56, 25] if ragged else None
    t, kw = make(4 if ragged else 1, 151, 70, N, G, dtype, lengths=lengths, seed=segment + N)
    assert ops._ssm_segment(*t["x"].shape, N, G) == segment
    g = torch.Generator(device="cuda").manual_seed(1)
    dout = torch.randn(t["x"].shape, generator=g, device="cuda").to(dtype)
    dstate = torch.randn(t["initial_state"].shape, generator=g, device="cuda")
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    out, state = call(leaves, kw, return_state=True)
    grads = torch.autograd.grad([out, state], list(leaves.values()), [dout, dstate])
    want, mag = oracle(t, kw, dout=dout, dstate=dstate)
    for k, v in {"out": out, "state": state, **{"d" + k: v for k, v in zip(leaves, grads)}}.items():
        check(k, v, want[k], mag[k], roundings(k, t))


@pytest.mark.parametrize("z,softplus", [(True, True), (False, False)])
def test_gradients_are_the_definitions_differences(gpu, z, softplus):
    """Each gradient along a random direction against the four-point quotient of
    the float64 definition, to the kernel's roundings, 1e-5 of the magnitudes, and a
    twentieth of them for the quotient.  Its steps of 1e-5 leave 1e-20 / 30 of the
    fifth derivative: a decay's exponent changes by at most |A way| <= 16 a step, 384
    over 24 steps, whose fifth power is 8e12: 3e-9 of the magnitudes, which the
    slopes of softplus and gate, of order one, change little.  Its own roundings are
    (24 + 16 + 768) 2^-53 of the loss's magnitudes, over 1e-5: 1e-8 of them."""
    t, kw = make(1, 24, 32, 16, z=z, softplus=softplus, seed=37)
    g = torch.Generator(device="cuda").manual_seed(6)
    dout = torch.randn(1, 24, 32, generator=g, device="cuda")
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    grads = torch.autograd.grad(call({**t, **leaves}, kw), list(leaves.values()), dout)
    _, mag = oracle(t, kw, dout=dout)
    wide = {k: None if v is None else v.double().cpu() for k, v in t.items()}

    def value(k, s, way):
        u = {**wide, k: wide[k] + s * way}
        r = so.ssm_scan(*(u[n] for n in ("x", "delta", "A", "B", "C")),
                        **{n: u[n] for n in ("D", "z", "delta_bias", "initial_state")}, **kw)
        return float((r["out"] * dout.double().cpu()).sum())

    for k, v in zip(leaves, grads):
        way = torch.randn(v.shape, generator=g, device="cuda").double().cpu().clamp(-4, 4)
        s = 1e-5
        quotient = (8 * (value(k, s, way) - value(k, -s, way)) - (value(k, 2 * s, way) - value(k, -2 * s, way))) / (12 * s)
        along = float((v.double().cpu() * way).sum())
        limit = 1.05 * roundings("d" + k, t) * float((mag["d" + k] * way.abs()).sum())
        assert abs(along - quotient) <= limit, (k, along, quotient, limit)
