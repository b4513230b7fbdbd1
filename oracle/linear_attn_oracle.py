"""Float64 CPU oracle of linear attention with a decay for each head: the
recurrence as a loop over time, and the gradients from their formulas.  With
``mag`` every signed term is taken by its absolute value (the decays stay), which
bounds what the terms of each result add up to: rounding errors are measured
against it.  The decays' gradient is one product per step by its formula; a
kernel that forms it as a running difference of the rows' products, started
afresh every ``segment`` steps, rounds against the sum of those (``mag``)."""
from __future__ import annotations

import torch


def _d(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, dout=None, dstate=None,
                     mag=False, segment=None):
    """Outputs by name: out, state; with ``dout`` (and ``dstate``) also dq, dk,
    dv, dlog_decay, dinitial_state."""
    q, k, v, g, init, dout, dstate = (_d(t) for t in (q, k, v, log_decay, initial_state, dout, dstate))
    B, L, H, dv = v.shape
    G, dk = q.shape[-2:]
    scale = dk ** -0.5 if scale is None else scale
    per_head = g.ndim == 1
    decay = torch.exp(g.expand(B, L, H))
    if mag:
        q, k, v, init, dout, dstate, scale = (t if t is None else abs(t) for t in (q, k, v, init, dout, dstate, scale))
    group = torch.arange(H) // (H // G)
    zero = torch.zeros(H, dk, dv, dtype=torch.float64)
    r = {"out": torch.zeros_like(v), "state": torch.zeros(B, H, dk, dv, dtype=torch.float64)}
    if dout is not None:
        r.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v),
                 dlog_decay=torch.zeros(B, L, H, dtype=torch.float64), dinitial_state=torch.zeros_like(r["state"]))
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        S = [zero if init is None else init[b]]
        qs, ks = q[b][:, group], k[b][:, group]
        for t in range(n):
            S.append(decay[b, t][:, None, None] * S[-1] + ks[t][:, :, None] * v[b, t][:, None, :])
            r["out"][b, t] = scale * (qs[t][:, :, None] * S[-1]).sum(1)
        r["state"][b] = S[-1]
        if dout is None:
            continue
        X = zero if dstate is None else dstate[b]
        run = torch.zeros(H, dtype=torch.float64)
        for t in reversed(range(n)):
            if mag and segment is not None and (t + 1) % segment == 0 or t == n - 1:
                run = (S[t + 1] * X).sum((1, 2))
            X = X + scale * qs[t][:, :, None] * dout[b, t][:, None, :]
            dq = scale * (S[t + 1] * dout[b, t][:, None, :]).sum(2)
            dk_ = (X * v[b, t][:, None, :]).sum(2)
            r["dq"][b, t].index_add_(0, group, dq)
            r["dk"][b, t].index_add_(0, group, dk_)
            r["dv"][b, t] = (X * ks[t][:, :, None]).sum(1)
            X = X * decay[b, t][:, None, None]
            if mag:
                run = run + (qs[t] * dq).sum(1) + (ks[t] * dk_).sum(1)
                r["dlog_decay"][b, t] = run
            else:
                r["dlog_decay"][b, t] = (X * S[t]).sum((1, 2))
        r["dinitial_state"][b] = X
    if dout is not None and per_head:
        r["dlog_decay"] = r["dlog_decay"].sum((0, 1))
    return r
