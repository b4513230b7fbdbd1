"""Linear attention with a decay for each head (``ops.linear_attention``,
``ops.linear_attention_step``) against the float64 loops of
``oracle/linear_attn_oracle.py``.

Tolerances, derived: every result is a sum of products, and its error is
measured against the same sum with absolute values (the oracle's ``mag``), S.
One fp32 rounding is 2^-24 of what it rounds.  A product of two widths adds at
most 128 of them, a chunk's sum 64, a decay 4 (its exponential's two ulp and its
argument's, |x| 2^-|x| < 0.54 of one); the state takes 2 + 64 a chunk, of which a
sequence of L steps has at most L / 32 + 1.  A value goes through the product of a
pair, the chunk's sum and the state: (128 + 4 + 64 + 66 (L / 32 + 1) + 128) 2^-24
S = (390 + 2.1 L) 2^-24 S.  On bf16 rows an fp32 operand is held in two bf16 pieces:
half a step of the second, 2^-8 of the first's rest, is 2^-16 S, met by pairs,
states and writes once each; the state's part is met again at each chunk that
reads it, but not kept: 3 * 2^-16 S.  The decays' gradient adds the rows' products
of a segment, each within those bounds, and 128 more roundings.  bf16 outputs add
half a step, 2^-8 of the value."""
import pytest
import torch

from conftest import announce
from oracle import linear_attn_oracle as lo

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("q", "k", "v", "log_decay", "initial_state")


def make(B, L, H, G, dk, dv, dtype=F32, per_head=False, init=True, lengths=None, seed=0, rate=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = dict(q=r(B, L, G, dk).to(dtype), k=r(B, L, G, dk).to(dtype), v=r(B, L, H, dv).to(dtype),
             log_decay=-rate * (r(H) if per_head else r(B, L, H)).abs(),
             initial_state=r(B, H, dk, dv) if init else None)
    return t, dict(lengths=None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32))


def call(t, kw, **more):
    from mogt_amd import ops
    return ops.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], initial_state=t.get("initial_state"), **kw,
                                **more)


def bound(t):
    return (390 + 2.1 * t["v"].shape[1]) * 2.0 ** -24 + (3 * 2.0 ** -16 if t["q"].dtype == BF16 else 0.0)


def check(name, got, want, mag, tol):
    got = got.detach()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.double().cpu() - want).abs()
    lim = tol * mag + half * (want.abs() + tol * mag) + 1e-30
    assert bool((err <= lim).all()), f"{name}: {float((err / lim).max()):.3g} of the bound"


def run_both(t, kw, seed=1, **more):
    """Forward and all gradients, through both outputs, against the oracle."""
    from mogt_amd import ops
    B, L, H, dv = t["v"].shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    dout = torch.randn(B, L, H, dv, generator=g, device="cuda").to(t["v"].dtype)
    dstate = torch.randn(B, H, t["q"].shape[-1], dv, generator=g, device="cuda")
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items() if x is not None}
    out, state = call(leaves, kw, return_state=True, **more)
    grads = dict(zip(leaves, torch.autograd.grad([out, state], list(leaves.values()), [dout, dstate])))
    segment = ops._linear_attn_segment(B, L, H, t["q"].shape[-1], dv, t["v"].dtype)
    want, mag = [lo.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], initial_state=t["initial_state"],
                                     dout=dout, dstate=dstate, mag=m, segment=segment, **kw, **more) for m in (0, 1)]
    tol = bound(t)
    check("out", out, want["out"], mag["out"], tol)
    check("state", state, want["state"], mag["state"], tol)
    for n, x in grads.items():
        assert x.dtype == t[n].dtype
        check("d" + n, x, want["d" + n], mag["d" + n], tol + 128 * 2.0 ** -24 * (n == "log_decay"))
    return out, state, grads


SHAPES = [  # B, L, H, G, dk, dv, dtype: single tokens, edges of chunks and segments, odd widths, shared heads
    (1, 1, 1, 1, 1, 1, F32), (2, 1, 3, 3, 64, 64, BF16), (1, 2, 2, 1, 16, 16, BF16), (1, 31, 2, 2, 33, 17, F32),
    (1, 32, 1, 1, 64, 64, F32), (2, 33, 2, 1, 48, 64, F32), (1, 63, 2, 2, 64, 64, BF16), (1, 64, 2, 2, 64, 64, BF16),
    (2, 65, 4, 2, 64, 64, BF16), (1, 70, 3, 1, 24, 100, BF16), (1, 95, 2, 2, 128, 128, F32),
    (1, 130, 2, 2, 128, 128, BF16), (2, 129, 2, 2, 65, 66, BF16), (1, 97, 6, 2, 40, 127, F32), (1, 66, 2, 2, 128, 32, BF16),
    (1, 67, 2, 1, 31, 128, F32), (1, 257, 2, 2, 64, 64, BF16), (1, 300, 2, 1, 32, 64, F32), (2, 513, 2, 2, 16, 24, BF16),
    (1, 700, 1, 1, 64, 128, BF16), (1, 777, 2, 2, 48, 33, F32),
]


@pytest.mark.parametrize("B,L,H,G,dk,dv,dtype", SHAPES)
def test_forward_and_gradients(gpu, B, L, H, G, dk, dv, dtype):
    announce(f"linear_attention B={B} L={L} H={H} G={G} dk={dk} dv={dv} {dtype}")
    run_both(*make(B, L, H, G, dk, dv, dtype, seed=L))


@pytest.mark.parametrize("opt", [dict(per_head=True), dict(init=False), dict(rate=5.0), dict(rate=0.001)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_options(gpu, opt, dtype):
    announce(f"linear_attention {opt} {dtype}")
    run_both(*make(2, 300, 4, 2, 32, 48, dtype, seed=4, **opt))


@pytest.mark.parametrize("scale", [0.0, 1.0, -2.5])
def test_scale(gpu, scale):
    announce(f"linear_attention scale {scale}")
    run_both(*make(1, 100, 2, 2, 32, 48, BF16, seed=4), scale=scale)


@pytest.mark.parametrize("lengths", [[300, 0, 1, 64], [0, 0, 0, 0], [256, 257, 63, 65], [400, -3, 32, 33]])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths(gpu, lengths, dtype):
    """Empty and single-token sequences, lengths at the edges of chunks and
    segments, and lengths outside the batch, which count as its ends."""
    announce(f"linear_attention lengths {lengths} {dtype}")
    t, kw = make(4, 300, 2, 1, 32, 48, dtype, lengths=lengths, seed=2)
    out, state, grads = run_both(t, kw)
    for i, n in enumerate(lengths):
        n = min(max(n, 0), 300)
        for x in (out, grads["q"], grads["k"], grads["v"], grads["log_decay"]):
            assert not x[i, n:].any()
        if n == 0:
            assert torch.equal(state[i], t["initial_state"][i])


def test_step_continues_the_sequence(gpu):
    from mogt_amd import ops
    for dtype, per_head, dk, dv in ((F32, False, 33, 18), (BF16, True, 64, 64), (BF16, False, 128, 7)):
        announce(f"linear_attention_step {dtype} {dk} {dv}")
        t, _ = make(3, 20, 4, 2, dk, dv, dtype, per_head=per_head, seed=9)
        g = t["log_decay"]
        want = lo.linear_attention(t["q"], t["k"], t["v"], g, initial_state=t["initial_state"])
        mag = lo.linear_attention(t["q"], t["k"], t["v"], g, initial_state=t["initial_state"], mag=True)
        out, state = ops.linear_attention(t["q"][:, :15], t["k"][:, :15], t["v"][:, :15],
                                          g if per_head else g[:, :15], initial_state=t["initial_state"],
                                          return_state=True)
        for i in range(15, 20):
            o = ops.linear_attention_step(t["q"][:, i], t["k"][:, i], t["v"][:, i], state, g if per_head else g[:, i])
            check("step", o, want["out"][:, i], mag["out"][:, i], bound(t))
        check("state", state, want["state"], mag["state"], bound(t))


@pytest.mark.parametrize("segment", [64, 128, 320])
@pytest.mark.parametrize("dtype,dk,dv", [(F32, 33, 64), (BF16, 64, 64), (BF16, 128, 100)])
def test_segments_of_several_chunks(gpu, monkeypatch, segment, dtype, dk, dv):
    """Long calls walk many chunks a segment, short ones one: here 1 to 10, with
    sequences that end inside a chunk, at a segment's end and one step past it."""
    from mogt_amd import ops
    announce(f"linear_attention segments of {segment} {dtype} {dk} {dv}")
    monkeypatch.setattr(ops, "LINEAR_ATTN_MIN_SEGMENT", segment)
    monkeypatch.setattr(ops, "LINEAR_ATTN_ONE_SEGMENT", 0)
    t, kw = make(4, 330, 2, 1, dk, dv, dtype, lengths=[330, 129, 128, 65], seed=segment)
    assert ops._linear_attn_segment(4, 330, 2, dk, dv, dtype) == segment
    run_both(t, kw)


def run_all(t, kw, dout, dstate, **more):
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items() if x is not None}
    out, state = call(leaves, kw, return_state=True, **more)
    return [out.detach(), state.detach(), *torch.autograd.grad([out, state], list(leaves.values()), [dout, dstate])]


def gradients_in(t, seed=3):
    B, L, H, dv = t["v"].shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, L, H, dv, generator=g, device="cuda").to(t["v"].dtype),
            torch.randn(B, H, t["q"].shape[-1], dv, generator=g, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padding_is_not_read(gpu, dtype):
    """NaN and infinities in the padded rows reach nothing."""
    announce(f"linear_attention padding {dtype}")
    t, kw = make(3, 300, 4, 2, 32, 48, dtype, lengths=[300, 130, 0], seed=3)
    dout, dstate = gradients_in(t)
    clean = run_all(t, kw, dout, dstate)
    bad, dbad = {n: x.clone() for n, x in t.items()}, dout.clone()
    for i, n in ((1, 130), (2, 0)):
        for x, v in ((bad["q"], float("nan")), (bad["k"], float("inf")), (bad["v"], float("-inf")),
                     (bad["log_decay"], float("nan")), (dbad, float("nan"))):
            x[i, n:] = v
    for a, b in zip(run_all(bad, kw, dbad, dstate), clean):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_what_is_not_finite_reaches_no_earlier_output(gpu, dtype, name, value):
    """Within a chunk too; and no later step's gradient.  A chunk that holds such a
    value adds its pairs in another order than one that does not, so these are held
    to the bound of the definition's values, not to the other run's bits."""
    announce(f"linear_attention {value} in {name} {dtype}")
    t, kw = make(1, 200, 2, 2, 32, 48, dtype, seed=5)
    dout, dstate = gradients_in(t)
    bad = {n: x.clone() for n, x in t.items()}
    bad[name][0, 77, 1, 3] = value
    got = dict(zip(("out", "state", "dq", "dk", "dv"), run_all(bad, kw, dout, dstate)))
    want, mag = [lo.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], initial_state=t["initial_state"],
                                     dout=dout, dstate=dstate, mag=m) for m in (0, 1)]
    assert not got["out"][0, 77, 1].isfinite().all()
    parts = [("out", slice(0, 77), slice(None)), ("out", slice(None), 0)]
    parts += [("out", slice(78, None), slice(None)), ("dk", slice(78, None), slice(None)),
              ("dv", slice(78, None), slice(None))] if name == "q" else [("dq", slice(0, 77), slice(None))]
    for n, rows, heads in parts:
        check(n, got[n][0, rows][:, heads], want[n][0, rows][:, heads], mag[n][0, rows][:, heads], bound(t))


@pytest.mark.parametrize("dtype,dk,dv", [(F32, 64, 128), (BF16, 32, 128), (BF16, 128, 96), (BF16, 128, 100), (F32, 128, 65)])
def test_wide_values(gpu, dtype, dk, dv):
    """More than 64 value columns (whole vectors and single elements): ragged, in
    segments, a decay of zero, and an infinity that reaches no earlier step."""
    announce(f"linear_attention wide {dk} {dv} {dtype}")
    t, kw = make(3, 330, 2, 1, dk, dv, dtype, seed=dv)
    t["log_decay"][1, 100] = float("-inf")
    kw["lengths"] = torch.tensor([330, 201, 0], device="cuda", dtype=torch.int32)
    out, state, _ = run_both(t, kw)
    assert not out[1, 201:].any() and not out[2].any()
    bad = dict(t, v=t["v"].clone())
    bad["v"][0, 177, 1, dv - 1] = float("inf")
    leaves = {n: x.detach() for n, x in bad.items() if x is not None}
    got, got_state = call(leaves, kw, return_state=True)
    rest = torch.ones(dv, dtype=torch.bool)
    rest[dv - 1] = False
    want, mag = [lo.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], initial_state=t["initial_state"], mag=m,
                                     lengths=kw["lengths"]) for m in (0, 1)]
    for rows, heads, cols in ((slice(0, 177), slice(None), slice(None)), (slice(None), 0, slice(None)),
                              (slice(None), slice(None), rest)):
        check("out", got[0, rows][:, heads][..., cols], want["out"][0, rows][:, heads][..., cols],
              mag["out"][0, rows][:, heads][..., cols], bound(t))
    assert not got[0, 177, 1, dv - 1].isfinite() and torch.equal(got[1:], out[1:]) and torch.equal(got_state[1:], state[1:])


@pytest.mark.parametrize("B,L,H,G,dk,dv", [(2, 300, 2, 1, 100, 100), (1, 333, 3, 3, 36, 60), (1, 130, 2, 2, 12, 124),
                                           (2, 90, 4, 2, 4, 4)])
def test_rows_of_half_vectors(gpu, B, L, H, G, dk, dv):
    """bf16 rows that are whole in 8 bytes and not in 16: the same values from rows
    that are whole in neither, to the bit."""
    announce(f"linear_attention half vectors {B} {L} {H} {G} {dk} {dv}")
    t, kw = make(B, L, H, G, dk, dv, BF16, seed=dk)
    out, state, grads = run_both(t, kw)
    dout, dstate = gradients_in(t)
    odd = dict(t)
    for n in ("q", "k", "v"):
        wide = torch.zeros(*t[n].shape[:-1], t[n].shape[-1] + 3, device="cuda", dtype=BF16)
        wide[..., 1:-2] = t[n]
        odd[n] = wide[..., 1:-2]
    for a, b in zip(run_all(odd, kw, dout, dstate)[:5], run_all(t, kw, dout, dstate)[:5]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_output_memory_at_any_element(gpu, dtype):
    """Through the C entry: an output that no vector is aligned in, and the elements
    around it."""
    from mogt_amd import _lib, ops
    announce(f"linear_attention output alignment {dtype}")
    t, _ = make(1, 90, 2, 2, 32, 64, dtype, seed=3)
    want, _ = call(t, {}, return_state=True)
    p, held = ops._linear_attn_problem(t["q"], t["k"], t["v"], t["log_decay"], t["initial_state"], None, 32 ** -0.5, 128)
    y = torch.full((want.numel() + 8,), 7.0, device="cuda", dtype=dtype)
    rc = _lib.load().mogt_linear_attn_fwd(p, y.data_ptr() + 3 * y.element_size(), None, None, None, 0,
                                          torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(y[3:-5].view(want.shape), want) and bool((y[:3] == 7).all()) and bool((y[-5:] == 7).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decay_of_minus_infinity_and_growth(gpu, dtype):
    """A state emptied in the middle of a chunk, decays far below fp32's least,
    and states that grow."""
    announce(f"linear_attention extreme decays {dtype}")
    t, kw = make(1, 300, 2, 2, 32, 48, dtype, seed=6)
    t["log_decay"][0, 100] = float("-inf")
    t["log_decay"][0, 170:175] = -1e30
    t["log_decay"][0, 200] = -300.0
    _, _, grads = run_both(t, kw)
    assert not grads["log_decay"][0, [100, 170, 171, 172, 173, 174, 200]].any()
    # rows of zeros first, over which a decay of exp(0.9) a step grows by exp(270)
    t, kw = make(1, 340, 2, 2, 32, 48, dtype, init=False, seed=7)
    t["k"][:, :300] = 0
    t["log_decay"].fill_(0.9)
    t["log_decay"][:, 300:] = 0.1
    dout, _ = gradients_in(t)
    dout[:, :300] = 0
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items() if x is not None}
    out = call(leaves, kw)
    assert not out[:, :300].any() and bool(out.isfinite().all())
    want, mag = [lo.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], mag=m) for m in (0, 1)]
    check("out", out, want["out"], mag["out"], bound(t))


def test_growth_of_a_small_state(gpu):
    """exp(104) = 1.5e45 lies beyond fp32, exp(104) 1e-30 does not."""
    announce("linear_attention growth of a small state")
    t, kw = make(1, 600, 1, 1, 16, 16, F32, seed=8)
    t["k"].zero_()
    t["initial_state"].fill_(1e-30)
    t["log_decay"].fill_(104.0 / 600)
    out, state = call(t, kw, return_state=True)
    want, mag = [lo.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], initial_state=t["initial_state"], mag=m)
                 for m in (0, 1)]
    check("state", state, want["state"], mag["state"], bound(t))
    check("out", out, want["out"], mag["out"], bound(t))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(gpu, dtype):
    """Rows of one projection, heads before time, transposed and expanded rows, odd
    offsets: the same values give the same bits."""
    from mogt_amd import ops
    announce(f"linear_attention strides {dtype}")
    t, kw = make(2, 150, 4, 2, 32, 48, dtype, seed=9)
    dout, dstate = gradients_in(t)
    want = run_all(t, kw, dout, dstate)

    def layouts(x):
        yield x.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.zeros(*x.shape[:2], 3 * x.shape[2] * x.shape[3] + 16, dtype=x.dtype, device="cuda")
        for off in (16, 7):
            part = wide[..., off:off + x.shape[2] * x.shape[3]].unflatten(-1, x.shape[2:])
            part.copy_(x)
            yield part
        yield x.transpose(0, 3).contiguous().transpose(0, 3)

    for q, k, v in zip(layouts(t["q"]), layouts(t["k"]), layouts(t["v"])):
        g = t["log_decay"].transpose(1, 2).contiguous().transpose(1, 2)
        u = dict(t, q=q, k=k, v=v, log_decay=g)
        for a, b in zip(run_all(u, kw, dout.transpose(0, 1).contiguous().transpose(0, 1), dstate.transpose(2, 3).contiguous().transpose(2, 3)), want):
            assert torch.equal(a, b)
    one = t["q"][:, :1]
    a = ops.linear_attention(one.expand(2, 150, 2, 32), t["k"], t["v"], t["log_decay"])
    b = ops.linear_attention(one.expand(2, 150, 2, 32).contiguous(), t["k"], t["v"], t["log_decay"])
    assert torch.equal(a, b)
    s, r = t["initial_state"].clone(), t["initial_state"].clone()
    a = ops.linear_attention_step(t["q"][:, 3], t["k"][:, 3], t["v"][:, 3], s, t["log_decay"][:, 3])
    b = ops.linear_attention_step(t["q"][:, 3].clone(), t["k"][:, 3].clone(), t["v"][:, 3].clone(), r,
                                  t["log_decay"][:, 3].clone())
    assert torch.equal(a, b) and torch.equal(s, r)


def test_rows_past_32_bit_offsets(gpu):
    """Rows 2 MB apart, and rows too far apart for a segment's offsets (copied)."""
    from mogt_amd import ops
    for L, wide in ((2200, 1 << 20), (6, 220_000_000)):
        announce(f"linear_attention {L} rows {2 * wide} bytes apart")
        base = torch.empty(1, L, wide, dtype=BF16, device="cuda")
        t, kw = make(1, L, 1, 1, 64, 64, BF16, seed=10)
        far = {}
        for i, n in enumerate(("q", "k", "v")):
            far[n] = base[..., 64 * i:64 * i + 64].unsqueeze(2)
            far[n].copy_(t[n])
        dout, dstate = gradients_in(t)
        for a, b in zip(run_all({**t, **far}, kw, dout, dstate), run_all(t, kw, dout, dstate)):
            assert torch.equal(a, b)
        del base, far
    torch.cuda.empty_cache()
    announce("linear_attention_step on states past 2^32 bytes")
    t, _ = make(1500, 1, 12, 12, 128, 128, BF16, init=False, seed=11)
    state = torch.zeros(1500, 12, 128, 128, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    part = state[-2:].clone()
    args = [t[n][:, 0] for n in ("q", "k", "v")]
    out = ops.linear_attention_step(*args, state, t["log_decay"][:, 0])
    last = ops.linear_attention_step(*[a[-2:] for a in args], part, t["log_decay"][-2:, 0])
    assert torch.equal(out[-2:], last) and torch.equal(state[-2:], part)


@pytest.mark.parametrize("shape", [(0, 5, 2), (2, 0, 2), (2, 5, 0)])
def test_empty(gpu, shape):
    announce(f"linear_attention empty {shape}")
    B, L, H = shape
    t, kw = make(B, L, H, 1, 16, 24, F32, seed=12)
    dout, dstate = gradients_in(t)
    out, state, *grads = run_all(t, kw, dout, dstate)
    assert out.shape == (B, L, H, 24) and torch.equal(state, t["initial_state"])
    for (n, x), g in zip(t.items(), grads):
        assert g.shape == x.shape
        assert torch.equal(g, dstate) if n == "initial_state" else not g.any()
    t["log_decay"] = torch.zeros(H, device="cuda")
    assert not run_all(t, kw, dout, dstate)[5].any()


def test_runs_repeat_bit_for_bit(gpu):
    announce("linear_attention repeated")
    for dtype, G, per_head in ((BF16, 4, False), (F32, 2, True)):
        t, kw = make(2, 500, 4, G, 64, 64, dtype, per_head=per_head, seed=13)
        dout, dstate = gradients_in(t)
        first = run_all(t, kw, dout, dstate)
        for _ in range(3):
            for a, b in zip(run_all(t, kw, dout, dstate), first):
                assert torch.equal(a, b)


def test_other_stream_and_two_calls_at_once(gpu):
    announce("linear_attention on two streams")
    t, kw = make(2, 700, 4, 2, 64, 64, BF16, seed=14)
    u, _ = make(1, 400, 3, 3, 32, 100, F32, seed=15)
    dt, du = gradients_in(t), gradients_in(u)
    want = run_all(t, kw, *dt), run_all(u, kw, *du)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for s, x, d, g in zip(streams, (t, u), (dt, du), got):
            with torch.cuda.stream(s):
                g.append(run_all(x, kw, *d))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for r in g:
            for a, b in zip(r, w):
                assert torch.equal(a, b)


def test_captured_graphs(gpu):
    """A forward, its gradients and steps captured and replayed on changing
    inputs, with eager work between the replays."""
    from mogt_amd import ops
    announce("linear_attention captured")
    t, kw = make(2, 400, 4, 2, 32, 64, BF16, seed=16, lengths=[400, 130])
    dout, dstate = gradients_in(t)
    held = {n: x.clone().requires_grad_(True) for n, x in t.items()}
    sstate = t["initial_state"].clone()

    def work():
        out, state = call(held, kw, return_state=True)
        return [out, state, *torch.autograd.grad([out, state], list(held.values()), [dout, dstate])]

    def step():
        return ops.linear_attention_step(held["q"].detach()[:, 0], held["k"].detach()[:, 0], held["v"].detach()[:, 0],
                                         sstate, held["log_decay"].detach()[:, 0])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
        sout = step()
    for seed in range(20, 24):
        fresh, _ = make(2, 400, 4, 2, 32, 64, BF16, seed=seed)
        with torch.no_grad():
            for n, x in held.items():
                x.copy_(fresh[n])
            sstate.copy_(fresh["initial_state"])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run_all(fresh, kw, dout, dstate)):
            assert torch.equal(a, b)
        own = fresh["initial_state"].clone()
        out = ops.linear_attention_step(fresh["q"][:, 0], fresh["k"][:, 0], fresh["v"][:, 0], own, fresh["log_decay"][:, 0])
        assert torch.equal(out, sout) and torch.equal(own, sstate)


def test_partial_gradients_and_outputs_alone(gpu):
    """Each input's gradient alone is the one of all; through either output alone."""
    announce("linear_attention partial gradients")
    t, kw = make(1, 300, 4, 2, 32, 64, BF16, seed=17)
    dout, dstate = gradients_in(t)
    want = dict(zip(NAMES, run_all(t, kw, dout, dstate)[2:]))
    for n in NAMES:
        u = {**t, n: t[n].detach().requires_grad_(True)}
        out, state = call(u, kw, return_state=True)
        (g,) = torch.autograd.grad([out, state], [u[n]], [dout, dstate])
        assert torch.equal(g, want[n]), n
    zero = torch.zeros_like
    for d in ((dout, None), (None, dstate)):
        leaves = {n: x.detach().requires_grad_(True) for n, x in t.items()}
        out, state = call(leaves, kw, return_state=True)
        o, g = [(x, y) for x, y in zip((out, state), d) if y is not None][0]
        got = torch.autograd.grad(o, list(leaves.values()), g, allow_unused=True)
        full = run_all(t, kw, d[0] if d[0] is not None else zero(dout), d[1] if d[1] is not None else zero(dstate))[2:]
        for a, b in zip(got, full):
            assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        q = t["q"].detach().requires_grad_(True)
        (g,) = torch.autograd.grad(call({**t, "q": q}, kw).float().sum(), q, create_graph=True)
        torch.autograd.grad(g.float().sum(), q)


def test_one_tensor_in_several_places(gpu):
    announce("linear_attention of one tensor")
    t, kw = make(1, 130, 2, 2, 48, 48, F32, seed=18)
    x = t["q"].detach().requires_grad_(True)
    dout, _ = gradients_in(t)
    (g,) = torch.autograd.grad(call({**t, "q": x, "k": x, "v": x}, kw), [x], dout)
    same = {n: t["q"] for n in ("q", "k", "v")}
    parts = run_all({**t, **same}, kw, dout, torch.zeros_like(t["initial_state"]))[2:5]
    torch.testing.assert_close(g, sum(parts), rtol=1e-6, atol=1e-5)


def test_lengths_of_eight_bytes(gpu):
    t, kw = make(3, 150, 2, 1, 32, 48, F32, lengths=[150, 0, 77], seed=19)
    dout, dstate = gradients_in(t)
    for a, b in zip(run_all(t, dict(kw, lengths=kw["lengths"].long()), dout, dstate), run_all(t, kw, dout, dstate)):
        assert torch.equal(a, b)


def test_other_dtypes_of_the_decay(gpu):
    t, kw = make(1, 100, 2, 2, 32, 48, BF16, seed=21)
    for dtype in (torch.float64, BF16):
        g = t["log_decay"].to(dtype).requires_grad_(True)
        out = call({**t, "log_decay": g}, kw)
        (d,) = torch.autograd.grad(out, g, torch.ones_like(out))
        assert d.dtype == dtype and torch.equal(out, call({**t, "log_decay": g.detach().float()}, kw))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_are_the_definitions_differences(gpu, dtype):
    """Each gradient along a random direction against the four-point quotient of
    the float64 definition, to the kernel's roundings and a twentieth of them for
    the quotient: its steps of 1e-4 leave 1e-16 / 30 of the fifth derivative, which in
    log_decay is at most 40^5 = 1e8 times the loss's magnitudes over 40 steps of
    directions of 1, and nothing in the others, in which the loss is of first degree;
    its own roundings are 1e-11 of the magnitudes."""
    t, kw = make(1, 40, 2, 1, 16, 16, dtype, seed=22)
    dout, dstate = gradients_in(t)
    grads = dict(zip(NAMES, run_all(t, kw, dout, dstate)[2:]))
    args = lambda u: [u[n] for n in NAMES[:4]]  # noqa: E731
    mag = lo.linear_attention(*args(t), initial_state=t["initial_state"], dout=dout, dstate=dstate, mag=True, segment=64)
    wide = {n: x.double().cpu() for n, x in t.items()}
    g = torch.Generator(device="cuda").manual_seed(6)

    def value(n, s, way):
        u = {**wide, n: wide[n] + s * way}
        r = lo.linear_attention(*args(u), initial_state=u["initial_state"])
        return float((r["out"] * dout.double().cpu()).sum() + (r["state"] * dstate.double().cpu()).sum())

    for n, x in grads.items():
        way = torch.rand(x.shape, generator=g, device="cuda").double().cpu() * 2 - 1
        s = 1e-4
        quotient = (8 * (value(n, s, way) - value(n, -s, way)) - (value(n, 2 * s, way) - value(n, -2 * s, way))) / (12 * s)
        along = float((x.double().cpu() * way).sum())
        half = torch.finfo(x.dtype).eps / 2 if x.dtype != F32 else 0.0
        limit = 1.05 * (bound(t) + 128 * 2.0 ** -24 + half) * float((mag["d" + n] * way.abs()).sum())
        assert abs(along - quotient) <= limit, (n, along, quotient, limit)


def test_a_layer_served_in_eight_bits(gpu):
    """Norm, projection, attention and the way out for a prompt, then for a token
    at a time on the state it left: each product against its operands, the
    attention's outputs against the recurrence over the rows that both made."""
    from mogt_amd import ops
    from test_gpu_fp8 import check_product
    announce("a linear attention layer in 8 bits")
    B, L, T, D, H, d = 2, 90, 5, 768, 12, 64
    g = torch.Generator(device="cuda").manual_seed(23)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    norm, w_in, w_out = 1 + 0.1 * r(D), r(3 * D, D) / D ** 0.5, r(D, D) / D ** 0.5
    w_in, w_out = (ops.quantize_fp8(w.bfloat16(), block_rows=128) for w in (w_in, w_out))
    rate = -0.02 * torch.exp(0.3 * r(H)) * torch.arange(1, H + 1, device="cuda")
    x, z = r(B, L + T, D), r(B, L + T, D).bfloat16()
    rows, outs, state = [], [], None
    for at in (slice(0, L), *range(L, L + T)):
        step = isinstance(at, int)
        res, q8, s8 = ops.add_rmsnorm_fp8(x[:, at], z[:, at], 0.5, norm)
        qkv = ops.linear_fp8(q8, s8, *w_in)
        check_product(qkv.flatten(0, -2), q8.flatten(0, -2), s8.flatten(0, -2), *w_in)
        q, k, v = (p.unflatten(-1, (H, d)) for p in qkv.split(D, -1))
        if step:
            o = ops.linear_attention_step(q, k, v, state, rate)
        else:
            o, state = ops.linear_attention(q, k, v, rate, return_state=True)
        y = ops.linear_fp8(*ops.quantize_fp8(o.flatten(-2)), *w_out, out_dtype=F32)
        assert y.shape == res.shape and bool(y.isfinite().all())
        rows.append([p.unsqueeze(1) if step else p for p in (q, k, v)])
        outs.append(o.unsqueeze(1) if step else o)
    q, k, v = (torch.cat(p, 1) for p in zip(*rows))
    t = dict(q=q, v=v)
    want, mag = [lo.linear_attention(q, k, v, rate, mag=m) for m in (0, 1)]
    check("out", torch.cat(outs, 1), want["out"], mag["out"], bound(t))
    check("state", state, want["state"], mag["state"], bound(t))
