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
