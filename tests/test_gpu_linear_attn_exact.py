"""What bf16 rows keep of linear attention's fp32 operands (states, weighted pairs,
decayed values): all 24 bits, in three bf16 pieces.  Inputs are chosen so that the
terms cancel and the results are exact, or zero; in 16 bits they would be off by
more than a bf16 output's rounding."""
import pytest
import torch

from conftest import announce
from oracle import linear_attn_oracle as lo
from test_gpu_linear_attn import BF16, F32, NAMES, call, gradients_in, make, run_all

pytestmark = pytest.mark.gpu
EXACT = [(64, 64), (128, 128), (128, 100), (33, 64), (32, 17)]


def whole(*s, lo=-1, hi=1, seed=0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi + 1, s, generator=g, device="cuda").to(dtype)


def differences(n, d, seed):
    """Rows e_i - e_j, i != j."""
    i = whole(n, lo=0, hi=d - 1, seed=seed, dtype=torch.long)
    j = (i + whole(n, lo=1, hi=d - 1, seed=seed + 1, dtype=torch.long)) % d
    eye = torch.eye(d, device="cuda")
    return (eye[i] - eye[j]).to(BF16)


@pytest.mark.parametrize("dk,dv", EXACT)
def test_states_are_read_in_full_fp32(gpu, dk, dv):
    """Whole numbers below 2^22 at a decay and scale of one: every sum is exact in
    fp32 in any order, so bf16 outputs are the exact numbers rounded once.  States of
    20 bits whose rows differ by little are read by rows e_i - e_j: in 16 bits the
    differences are lost."""
    announce(f"linear_attention exact states {dk} {dv}")
    L = 300
    large = whole(1, 1, 1, dv, lo=2 ** 19, hi=2 ** 20 - 1, seed=1, dtype=F32) + whole(1, 1, dk, dv, lo=-30, hi=30, seed=2, dtype=F32)
    pick, ones = differences(L, dk, 3).view(1, L, 1, dk), whole(1, L, 1, dk, seed=5)
    g, rows = torch.zeros(1, L, 1, device="cuda"), whole(1, L, 1, dv, seed=6)
    t = dict(q=pick, k=ones, v=rows, log_decay=g, initial_state=large)
    want = lo.linear_attention(t["q"], t["k"], t["v"], g, initial_state=large, scale=1.0)["out"]
    assert torch.equal(call(t, {}, scale=1.0).double().cpu(), want.to(BF16).double())
    # the same of dv, backwards from the final state's gradient
    t = dict(t, q=ones, k=pick, v=rows.clone().requires_grad_(True), initial_state=None)
    out, state = call(t, {}, scale=1.0, return_state=True)
    (got,) = torch.autograd.grad([out, state], [t["v"]], [rows, large])
    want = lo.linear_attention(ones, pick, rows, g, scale=1.0, dout=rows, dstate=large)["dv"]
    assert torch.equal(got.double().cpu(), want.to(BF16).double())


@pytest.mark.parametrize("dk,dv", EXACT)
def test_pairs_are_weighted_in_full_fp32(gpu, dk, dv):
    """As above: products q_t . k_s of up to 20 bits, of neighbouring steps whose
    values are of opposite signs and whose keys differ by one in one place.  Six steps
    have values, up to 2: sums stay below 12 * 2^20 < 2^24."""
    announce(f"linear_attention exact pairs {dk} {dv}")
    L = 150
    q, k = whole(1, L, 1, dk, lo=0, hi=90 if dk > 64 else 127, seed=1), whole(1, L, 1, dk, lo=0, hi=90 if dk > 64 else 126, seed=2)
    v = torch.zeros(1, L, 1, dv, device="cuda", dtype=BF16)
    q[..., 0] = whole(1, L, 1, lo=0, hi=5, seed=3)
    for i, s in enumerate((10, 40, 70)):
        k[0, s + 1] = k[0, s]
        k[0, s + 1, 0, 0] += 1
        v[0, s] = whole(1, dv, lo=1, hi=2, seed=4 + i)
        v[0, s + 1] = -v[0, s]
    g = torch.zeros(1, L, 1, device="cuda")
    want = lo.linear_attention(q, k, v, g, scale=1.0)["out"]
    assert torch.equal(call(dict(q=q, k=k, v=v, log_decay=g), {}, scale=1.0).double().cpu(), want.to(BF16).double())


@pytest.mark.parametrize("dk,dv", EXACT)
def test_decayed_values_are_written_in_full_fp32(gpu, monkeypatch, dk, dv):
    """Three steps write 255, 254 and 1 times one value under one decay, and a later
    chunk of the same segment reads the first less the others: zero.  In fp32 each
    write rounds its product (1 in 2^24), is added in three parts (3) and read in three
    (3, and 5 more for the sum of the three rows): 12 of 2^-24 of the terms' sum, and
    the decay between them is common to all.  In 16 bits a write is off by up to 64."""
    from mogt_amd import ops
    announce(f"linear_attention exact writes {dk} {dv}")
    monkeypatch.setattr(ops, "LINEAR_ATTN_MIN_SEGMENT", 128)
    monkeypatch.setattr(ops, "LINEAR_ATTN_ONE_SEGMENT", 0)
    L = 384
    assert ops._linear_attn_segment(1, L, 1, dk, dv, BF16) == 128
    q, k, v = (torch.zeros(1, L, 1, d, device="cuda", dtype=BF16) for d in (dk, dk, dv))
    g = -0.05 * torch.rand(1, L, 1, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    value = whole(dv, lo=1, hi=1, seed=8) * torch.exp2(whole(dv, lo=-3, hi=3, seed=9))
    for at in (20, 150):
        g[0, at + 1:at + 3] = 0.0
        for i, x in enumerate((255.0, 254.0, 1.0)):
            k[0, at + i, 0, 3 * i] = 1.0
            v[0, at + i, 0] = x * value
    q[0, 64:, 0, 0] = 1.0
    q[0, 64:, 0, 3] = q[0, 64:, 0, 6] = -1.0
    g[0, 64] = -0.3
    mag = lo.linear_attention(q, k, v, g, scale=1.0, mag=True)["out"]
    got = call(dict(q=q, k=k, v=v, log_decay=g), {}, scale=1.0).double().cpu()
    assert bool((got[0, 64:128].abs() <= 12 * 2.0 ** -24 * mag[0, 64:128]).all())
    assert bool((got[0, 192:256].abs() <= 40 * 2.0 ** -24 * mag[0, 192:256]).all())   # two states, two more chunks, a carry


@pytest.mark.parametrize("dk,dv", EXACT)
def test_gradients_read_states_in_full_fp32(gpu, dk, dv):
    """dq and dk: columns of the initial state, and of the final one's gradient, that
    differ by little, read by rows e_i - e_j."""
    announce(f"linear_attention exact gradients {dk} {dv}")
    L = 300
    large = whole(1, 1, dk, 1, lo=2 ** 19, hi=2 ** 20 - 1, seed=1, dtype=F32) + whole(1, 1, dk, dv, lo=-30, hi=30, seed=2, dtype=F32)
    pick, ones, more = differences(L, dv, 3).view(1, L, 1, dv), whole(1, L, 1, dk, seed=5), whole(1, L, 1, dk, seed=6)
    g, rows = torch.zeros(1, L, 1, device="cuda"), whole(1, L, 1, dv, seed=7)
    for n, v, dout, init, dstate in (("q", rows, pick, large, None), ("k", pick, rows, None, large)):
        t = dict(q=ones, k=more, v=v, log_decay=g, initial_state=init)
        leaf = t[n].clone().requires_grad_(True)
        out, state = call({**t, n: leaf}, {}, scale=1.0, return_state=True)
        (got,) = torch.autograd.grad([out] if dstate is None else [out, state], [leaf], [dout] if dstate is None else [dout, dstate])
        want = lo.linear_attention(ones, more, v, g, scale=1.0, initial_state=init, dout=dout, dstate=dstate)["d" + n]
        assert torch.equal(got.double().cpu(), want.to(BF16).double()), n


@pytest.mark.parametrize("L", [100, 384])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dk,dv", EXACT)
def test_states_left_behind_are_in_full_fp32(gpu, monkeypatch, dk, dv, dtype, L):
    """The final state, and the initial one's gradient: three rows, written 255, 254
    and 1 times one value under one decay; the first less the others is zero, to a
    rounding each for the product with the decay, three for its parts, and one for each
    chunk and segment that the state goes through after that (16 are allowed for)."""
    from mogt_amd import ops
    announce(f"linear_attention exact states {dk} {dv} {dtype} {L}")
    monkeypatch.setattr(ops, "LINEAR_ATTN_MIN_SEGMENT", 128)
    monkeypatch.setattr(ops, "LINEAR_ATTN_ONE_SEGMENT", 0)
    q, k, v, dout = (torch.zeros(1, L, 1, d, device="cuda", dtype=dtype) for d in (dk, dk, dv, dv))
    g = -0.05 * torch.rand(1, L, 1, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    value = torch.exp2(whole(dv, lo=-3, hi=3, seed=9).float()).to(dtype)
    for at in (20, 70) if L == 100 else (20, 150, 300):
        g[0, at + 1:at + 3] = 0.0
        for i, x in enumerate((255.0, 254.0, 1.0)):
            q[0, at + i, 0, 3 * i] = k[0, at + i, 0, 3 * i] = 1.0
            v[0, at + i, 0] = dout[0, at + i, 0] = x * value
    init = torch.zeros(1, 1, dk, dv, device="cuda", requires_grad=True)
    out, state = ops.linear_attention(q, k, v, g, initial_state=init, scale=1.0, return_state=True)
    (dinit,) = torch.autograd.grad(out, init, dout)
    for name, s in (("state", state.detach()), ("dinitial_state", dinit)):
        s = s[0, 0].double()
        assert bool((s[0] > 0).all()), name
        assert bool(((s[0] - s[3] - s[6]).abs() <= 20 * 2.0 ** -24 * 2 * s[0]).all()), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (33, 20)])
def test_the_decays_gradient_of_whole_numbers_is_exact(gpu, dk, dv, dtype):
    """Its sums are in 64 bits and the rows' products of numbers below 2^24 exact, so
    what is left is one rounding: for one decay a step, and for one a head."""
    announce(f"linear_attention exact decay gradient {dk} {dv} {dtype}")
    L, H = 700, 2
    q, k = (whole(2, L, 1, dk, seed=s, dtype=dtype) for s in (1, 2))
    v, dout = (whole(2, L, H, dv, seed=s, dtype=dtype) for s in (3, 4))
    init, dstate = (whole(2, H, dk, dv, lo=-1000, hi=1000, seed=s, dtype=F32) for s in (5, 6))
    kw = dict(lengths=torch.tensor([L, 333], device="cuda", dtype=torch.int32))
    for g in (torch.zeros(2, L, H, device="cuda"), torch.zeros(H, device="cuda")):
        got = run_all(dict(q=q, k=k, v=v, log_decay=g, initial_state=init), kw, dout, dstate, scale=1.0)[5]
        want = lo.linear_attention(q, k, v, g, initial_state=init, scale=1.0, dout=dout, dstate=dstate, **kw)["dlog_decay"]
        assert torch.equal(got.cpu(), want.float())


@pytest.mark.parametrize("B,L,H,G,dk,dv", [(2, 700, 4, 2, 64, 64), (1, 600, 3, 3, 128, 128), (3, 330, 2, 1, 40, 100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_errors_of_fp32_results_are_a_walk_of_roundings(gpu, B, L, H, G, dk, dv, dtype):
    """As 2-norms: of the 390 + 2.1 L roundings that bound one result's error (see
    test_gpu_linear_attn) each is independent of the others and of 2^-24 of a partial
    sum, which for terms of random signs is no larger than its sum: their root times
    2^-24.  The decays' gradient is a difference of two running sums of its segment, and
    is held to those."""
    from mogt_amd import ops
    announce(f"linear_attention errors {B} {L} {H} {G} {dk} {dv} {dtype}")
    t, kw = make(B, L, H, G, dk, dv, dtype, seed=L)
    dout, dstate = gradients_in(t)
    got = dict(zip(("out", "state", *("d" + n for n in NAMES)), run_all(t, kw, dout, dstate)))
    segment = ops._linear_attn_segment(B, L, H, dk, dv, dtype)
    want, mag = [lo.linear_attention(t["q"], t["k"], t["v"], t["log_decay"], initial_state=t["initial_state"], dout=dout,
                                     dstate=dstate, mag=m, segment=segment) for m in (0, 1)]
    tol = (390 + 2.1 * L) ** 0.5 * 2.0 ** -24
    for n, x in got.items():
        if x.dtype == F32:
            size = (mag if n == "dlog_decay" else want)[n].norm()
            err = float((x.double().cpu() - want[n]).norm() / size)
            assert err <= tol, n
