"""What bf16 rows keep of linear attention's fp32 operands (states, weighted pairs,
decayed values): all 24 bits, in three bf16 pieces.  Inputs are chosen so that the
terms cancel and the results are exact, or zero; in 16 bits they would be off by
more than a bf16 output's rounding."""
import pytest
import torch

from conftest import announce
from oracle import linear_attn_oracle as lo
from test_gpu_linear_attn import BF16, F32, call

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
