"""The float64 oracle of the selective scan and the short convolution against
autograd of its own definitions and against difference quotients (CPU)."""
import pytest
import torch

from oracle import ssm_oracle as so

CASES = [dict(softplus=True, z=True, G=2, ragged=True), dict(softplus=False, z=False, G=1, ragged=False),
         dict(softplus=True, z=False, G=4, ragged=True)]


def scan_inputs(case, seed=0):
    g = torch.Generator().manual_seed(seed)
    b, L, ch, N, G = 3, 6, 4, 3, case["G"]
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    t = dict(x=r(b, L, ch), delta=0.5 * r(b, L, ch), A=-r(ch, N).abs(), B=r(b, L, G, N), C=r(b, L, G, N), D=r(ch),
             delta_bias=r(ch), initial_state=r(b, ch, N))
    if case["z"]:
        t["z"] = r(b, L, ch)
    lengths = torch.tensor([L, 0, 1]) if case["ragged"] else None
    return t, lengths, r(b, L, ch), r(b, ch, N)


def scan_loss(t, lengths, dout, dstate, softplus):
    """sum(out dout) + sum(state dstate), step by step in differentiable torch."""
    b, L, ch = t["x"].shape
    group = torch.arange(ch) // (ch // t["B"].shape[2])
    total = torch.zeros((), dtype=torch.float64)
    for i in range(b):
        h = t["initial_state"][i]
        for s in range(L if lengths is None else int(lengths[i])):
            dt = t["delta"][i, s] + t["delta_bias"]
            dt = torch.nn.functional.softplus(dt) if softplus else dt
            h = torch.exp(dt[:, None] * t["A"]) * h + (dt * t["x"][i, s])[:, None] * t["B"][i, s][group]
            y = (t["C"][i, s][group] * h).sum(-1) + t["D"] * t["x"][i, s]
            if "z" in t:
                y = y * torch.nn.functional.silu(t["z"][i, s])
            total = total + (y * dout[i, s]).sum()
        total = total + (h * dstate[i]).sum()
    return total


@pytest.mark.parametrize("case", CASES)
def test_scan_gradients_are_autograds_and_the_differences(case):
    t, lengths, dout, dstate = scan_inputs(case)
    kw = {k: v for k, v in t.items() if k not in ("x", "delta", "A", "B", "C")}
    r = so.ssm_scan(*(t[k] for k in ("x", "delta", "A", "B", "C")), **kw, delta_softplus=case["softplus"],
                    lengths=lengths, dout=dout, dstate=dstate)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    loss = scan_loss(leaves, lengths, dout, dstate, case["softplus"])
    torch.testing.assert_close((r["out"] * dout).sum() + (r["state"] * dstate).sum(), loss.detach(), rtol=1e-12,
                               atol=1e-12)
    grads = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    for k, g in grads.items():
        torch.testing.assert_close(r["d" + k], g, rtol=1e-11, atol=1e-12)
        v = torch.randn(t[k].shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
        eps = 1e-5
        hi, lo = (scan_loss({**t, k: t[k] + s * eps * v}, lengths, dout, dstate, case["softplus"]) for s in (1, -1))
        # the third derivative's share of the quotient is eps^2, its rounding 2^-53 |loss| / eps
        torch.testing.assert_close((hi - lo) / (2 * eps), (r["d" + k] * v).sum(), rtol=1e-7, atol=1e-7)


@pytest.mark.parametrize("K", [1, 2, 4])
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("ragged", [True, False])
def test_conv_gradients_are_the_differences(K, silu, ragged):
    g = torch.Generator().manual_seed(K)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    b, L, ch = 3, 5, 3
    t = dict(x=r(b, L, ch), weight=r(ch, K), bias=r(ch), initial_state=r(b, K - 1, ch))
    lengths = torch.tensor([L, 0, 2]) if ragged else None
    dy, ds = r(b, L, ch), r(b, K - 1, ch)

    def loss(t):
        o = so.short_conv(t["x"], t["weight"], t["bias"], silu=silu, initial_state=t["initial_state"],
                          lengths=lengths)
        return (o["y"] * dy).sum() + (o["state"] * ds).sum()

    got = so.short_conv(t["x"], t["weight"], t["bias"], silu=silu, initial_state=t["initial_state"], lengths=lengths,
                        dy=dy, dstate=ds)
    for k in t:
        v, eps = r(*t[k].shape), 1e-5
        hi, lo = (loss({**t, k: t[k] + s * eps * v}) for s in (1, -1))
        torch.testing.assert_close((hi - lo) / (2 * eps), (got["d" + k] * v).sum(), rtol=1e-7, atol=1e-7)


def test_conv_is_the_library_convolution():
    g = torch.Generator().manual_seed(3)
    x, w, bias = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 9, 5), (5, 4), (5,)))
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.transpose(1, 2), (3, 0)), w[:, None], bias, groups=5)
    torch.testing.assert_close(so.short_conv(x, w, bias)["y"], want.transpose(1, 2), rtol=1e-13, atol=1e-13)


@pytest.mark.parametrize("case", CASES)
def test_magnitudes_bound_the_results(case):
    t, lengths, dout, dstate = scan_inputs(case, seed=9)
    kw = {k: v for k, v in t.items() if k not in ("x", "delta", "A", "B", "C")}
    args = [t[k] for k in ("x", "delta", "A", "B", "C")]
    r, m = (so.ssm_scan(*args, **kw, delta_softplus=case["softplus"], lengths=lengths, dout=dout, dstate=dstate,
                        mag=mag) for mag in (False, True))
    for k in r:
        assert bool((r[k].abs() <= m[k] * (1 + 1e-12)).all()), k
