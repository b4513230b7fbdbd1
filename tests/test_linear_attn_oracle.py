"""The linear attention oracle's gradients against autograd through its own
definition, and its bounds, on the CPU."""
import pytest
import torch

from oracle import linear_attn_oracle as lo


def definition(q, k, v, g, init, lengths, scale):
    B, L, H, dv = v.shape
    n = H // q.shape[2]
    outs, states = [], []
    for b in range(B):
        S, rows = init[b], []
        for t in range(L):
            if t < lengths[b]:
                S = torch.exp(g[b, t])[:, None, None] * S \
                    + k[b, t].repeat_interleave(n, 0)[:, :, None] * v[b, t][:, None, :]
                rows.append(scale * torch.einsum("hi,hij->hj", q[b, t].repeat_interleave(n, 0), S))
            else:
                rows.append(torch.zeros(H, dv, dtype=v.dtype))
        outs.append(torch.stack(rows))
        states.append(S)
    return torch.stack(outs), torch.stack(states)


@pytest.mark.parametrize("H,G,per_head", [(4, 4, False), (6, 2, False), (3, 1, True)])
def test_gradients_are_those_of_the_definition(H, G, per_head):
    torch.manual_seed(H)
    B, L, dk, dv, lengths = 3, 9, 5, 4, [9, 0, 4]
    r = lambda *s: torch.randn(*s, dtype=torch.float64)  # noqa: E731
    q, k, v, init = r(B, L, G, dk), r(B, L, G, dk), r(B, L, H, dv), r(B, H, dk, dv)
    g = -r(H).abs() if per_head else -r(B, L, H).abs()
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, init)]
    out, state = definition(q, k, v, g.expand(B, L, H), init, lengths, 0.7)
    go, gs = r(*out.shape), r(*state.shape)
    want = torch.autograd.grad([out, state], leaves, [go, gs])
    kw = dict(scale=0.7, initial_state=init, lengths=torch.tensor(lengths), dout=go, dstate=gs)
    got = lo.linear_attention(q, k, v, g, **kw)
    mag = lo.linear_attention(q, k, v, g, **kw, mag=True, segment=4)
    torch.testing.assert_close(got["out"], out)
    torch.testing.assert_close(got["state"], state)
    for name, t in zip(("dq", "dk", "dv", "dlog_decay", "dinitial_state"), want):
        torch.testing.assert_close(got[name], t)
    for name, t in got.items():
        assert bool((mag[name] >= t.abs() * (1 - 1e-12)).all()), name
