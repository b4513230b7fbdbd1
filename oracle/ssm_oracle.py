"""Float64 CPU oracle of the selective state space scan and its short causal
convolution: the definitions as loops over time, and the gradients from their
formulas.  With ``mag`` every signed term is taken by its absolute value (the
decays stay), which bounds what the terms of each result add up to: rounding
errors are measured against it."""
from __future__ import annotations

import torch


def _d(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def _abs(t, mag):
    return t.abs() if mag and t is not None else t


def _lens(lengths, B, L):
    return [L] * B if lengths is None else [min(max(int(n), 0), L) for n in lengths.tolist()]


def _slope(v, mag=False):
    """silu'(v); with ``mag`` the sum of its terms' absolute values."""
    s = torch.sigmoid(v)
    return s * (1 + (v.abs() if mag else v) * (1 - s))


def softplus(v):
    return torch.logaddexp(v, torch.zeros_like(v))


def ssm_scan(x, delta, A, B, C, *, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
             lengths=None, dout=None, dstate=None, mag=False):
    """Outputs by name: out, state; with ``dout`` (and ``dstate``) also the
    gradients dx, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dinitial_state.
    B and C are [b, L, G, N].  Sequences run one at a time, on their own steps
    only."""
    x, delta, A, B, C, D, z, bias = (_d(t) for t in (x, delta, A, B, C, D, z, delta_bias))
    b, L, ch = x.shape
    G, N = B.shape[2:]
    lens = _lens(lengths, b, L)
    group = torch.arange(ch) // (ch // G)
    skip = torch.zeros(ch, dtype=torch.float64) if D is None else D
    r = {"out": torch.zeros_like(x), "state": torch.zeros(b, ch, N, dtype=torch.float64)}
    back = dout is not None
    if back:
        dout = _d(dout)
        r.update(dx=torch.zeros_like(x), ddelta=torch.zeros_like(x), dz=torch.zeros_like(x), dA=torch.zeros_like(A),
                 dB=torch.zeros_like(B), dC=torch.zeros_like(C), dD=torch.zeros(ch, dtype=torch.float64),
                 ddelta_bias=torch.zeros(ch, dtype=torch.float64),
                 dinitial_state=torch.zeros(b, ch, N, dtype=torch.float64))
    for i in range(b):
        n = lens[i]
        raw = delta[i, :n] + (0 if bias is None else bias)
        dt = softplus(raw) if delta_softplus else raw
        a = torch.exp(dt[..., None] * A)                                     # [n, ch, N]
        xs, dts, sk = _abs(x[i, :n], mag), _abs(dt, mag), _abs(skip, mag)
        Bs, Cs = _abs(B[i, :n][:, group], mag), _abs(C[i, :n][:, group], mag)
        zi = None if z is None else z[i, :n]
        h = torch.zeros(ch, N, dtype=torch.float64) if initial_state is None else _abs(_d(initial_state[i]), mag)
        hs = [h]
        for t in range(n):
            hs.append(a[t] * hs[-1] + (dts[t] * xs[t])[:, None] * Bs[t])
        y = torch.stack([(Cs[t] * hs[t + 1]).sum(-1) + sk * xs[t] for t in range(n)]) if n else x.new_zeros(0, ch)
        gate = 1.0 if zi is None else _abs(zi * torch.sigmoid(zi), mag)
        r["out"][i, :n] = y * gate
        r["state"][i] = hs[-1]
        if not back:
            continue
        go = _abs(dout[i, :n], mag)
        dy = go * gate
        if zi is not None:
            r["dz"][i, :n] = go * y * _slope(zi, mag)
        g = torch.zeros(ch, N, dtype=torch.float64) if dstate is None else _abs(_d(dstate[i]), mag)
        As = _abs(A, mag)
        for t in reversed(range(n)):
            g = g + Cs[t] * dy[t][:, None]
            r["dC"][i, t].index_add_(0, group, dy[t][:, None] * hs[t + 1])
            r["dB"][i, t].index_add_(0, group, g * (dts[t] * xs[t])[:, None])
            dw = (g * Bs[t]).sum(-1)
            q = g * a[t] * hs[t]
            dd = dw * xs[t] + (q * As).sum(-1)
            if delta_softplus:
                dd = dd * torch.sigmoid(raw[t])
            r["dx"][i, t] = dw * dts[t] + sk * dy[t]
            r["ddelta"][i, t] = dd
            r["dA"] += q * dts[t][:, None]
            g = g * a[t]
        r["dinitial_state"][i] = g
        r["dD"] += (dy * xs).sum(0)
        r["ddelta_bias"] += r["ddelta"][i, :n].sum(0)
    return r


def short_conv(x, weight, bias=None, *, silu=False, initial_state=None, lengths=None, dy=None, dstate=None,
               mag=False):
    """Outputs by name: y, state; with ``dy`` (and ``dstate``) also dx, dweight,
    dbias, dinitial_state."""
    x, w = _abs(_d(x), mag), _abs(_d(weight), mag)
    b, L, ch = x.shape
    K = w.shape[1]
    bias_ = torch.zeros(ch, dtype=torch.float64) if bias is None else _abs(_d(bias), mag)
    init = torch.zeros(b, K - 1, ch, dtype=torch.float64) if initial_state is None else _abs(_d(initial_state), mag)
    r = {"y": torch.zeros_like(x), "state": torch.zeros_like(init)}
    back = dy is not None
    if back:
        dy = _abs(_d(dy), mag)
        r.update(dx=torch.zeros_like(x), dweight=torch.zeros_like(w), dbias=torch.zeros_like(bias_),
                 dinitial_state=torch.zeros_like(init))
    for i, n in enumerate(_lens(lengths, b, L)):
        e = torch.cat([init[i], x[i, :n]])
        s = bias_ + sum(w[:, k] * e[k:k + n] for k in range(K))
        r["y"][i, :n] = s * (1.0 if mag else torch.sigmoid(s)) if silu else s
        r["state"][i] = e[n:]
        if not back:
            continue
        ds = dy[i, :n] * (1.1 if mag else _slope(s)) if silu else dy[i, :n]   # |silu'| < 1.1
        de = torch.zeros_like(e)
        for k in range(K):
            de[k:k + n] += w[:, k] * ds
            r["dweight"][:, k] += (ds * e[k:k + n]).sum(0)
        if dstate is not None:
            de[n:] += _abs(_d(dstate[i]), mag)
        r["dx"][i, :n], r["dinitial_state"][i] = de[K - 1:], de[:K - 1]
        r["dbias"] += ds.sum(0)
    return r
