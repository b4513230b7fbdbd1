"""Performance cases of the selective state space operators: the scan, its short causal convolution, and their single-token forms.

``listed()`` is the fixed set, ``draw(rng)`` one more case of the same ranges.
``prepare`` makes what the program holds before the call (inputs on the GPU,
made from the seed alone), ``run`` is one pass and returns its whole outputs,
``work`` the bytes and operations the pass cannot do without, and ``exact`` the
same outputs in 64 bits from the operators' definitions.  With ``own`` false
``run`` computes in plain torch (32 bits, rounded once), with ``own`` true
through the framework's entry points.

Kinds of case (tensors are channels last, [batch, time, channel]):

* ``conv``   y = silu(bias + depthwise causal convolution of K taps)
* ``scan``   h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t,  y_t = C_t . h_t + D x_t,
             times silu(z); dt = softplus(delta + bias), N states per channel,
             B and C shared by the channels of a group
* ``conv_step``, ``scan_step``  one token of either, the state updated in place

``train`` adds the backward pass; ``carry`` an initial state that comes in and
the final one that goes out; ``ragged`` a length for each sequence of the
padded batch (zero and one among them).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # A short prompt in fp32, one sequence: latency of the smallest call.
        dict(name="conv_short", kind="conv", B=1, L=200, D=768, K=4, dtype="f32", train=False, carry=True,
             ragged=False),
        # The longest context of the framework's benchmark (32768 steps), bf16,
        # the input a half of its projection's rows: one piece of a long prompt.
        dict(name="conv_long", kind="conv", B=1, L=32768, D=2048, K=4, dtype="bf16", train=False, carry=True,
             ragged=False),
        # One layer of a training step: four sequences, a length that no tile divides.
        dict(name="conv_train", kind="conv", B=4, L=4095, D=1280, K=4, dtype="bf16", train=True, carry=False,
             ragged=False),
        # One token of an interactive program, and of a server with 256 sequences.
        dict(name="conv_step_1", kind="conv_step", B=1, D=1280, K=4, dtype="bf16"),
        dict(name="conv_step_256", kind="conv_step", B=256, D=2048, K=4, dtype="bf16"),
        # A short prompt: too few rows for one wave per 64 channels to fill the GPU.
        dict(name="scan_short", kind="scan", B=1, L=200, D=1280, N=16, G=1, dtype="bf16", train=False, carry=True,
             ragged=False),
        # A padded batch of prompts of different lengths in fp32, two groups of channels.
        dict(name="scan_ragged", kind="scan", B=8, L=1001, D=768, N=16, G=2, dtype="f32", train=False, carry=True,
             ragged=True),
        # The longest context, one sequence: the largest forward pass.
        dict(name="scan_long", kind="scan", B=1, L=32768, D=2048, N=16, G=1, dtype="bf16", train=False, carry=True,
             ragged=False),
        # A small training step in fp32, odd length, eight states.
        dict(name="scan_train_small", kind="scan", B=2, L=513, D=768, N=8, G=1, dtype="f32", train=True, carry=False,
             ragged=False),
        # One layer of a training step, the largest case.
        dict(name="scan_train", kind="scan", B=2, L=8192, D=1280, N=16, G=1, dtype="bf16", train=True, carry=False,
             ragged=False),
        # One token of an interactive program, and of a server with 256 sequences.
        dict(name="scan_step_1", kind="scan_step", B=1, D=1280, N=16, G=1, dtype="bf16"),
        dict(name="scan_step_256", kind="scan_step", B=256, D=2048, N=16, G=1, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["conv", "conv", "scan", "scan", "scan", "conv_step", "scan_step"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    D = rng.choice([64, 200, 333, 768, 1000, 1280, 2048])
    K = rng.choice([2, 3, 4, 4])
    N = rng.choice([4, 8, 15, 16, 16, 16, 24, 64])
    G = rng.choice([1, 1, 1, 2, 4] if D % 4 == 0 else [1])
    if kind == "conv_step":
        return dict(kind=kind, B=_log(rng, 1, 256), D=D, K=K, dtype=dtype)
    if kind == "scan_step":
        return dict(kind=kind, B=_log(rng, 1, 256), D=D, N=N if N < 64 or D < 1280 else 16, G=G, dtype=dtype)
    train = rng.random() < 0.5
    carry = not train and rng.random() < 0.5
    B = rng.choice([1, 1, 2, 3, 8])
    ragged = B > 1 and rng.random() < 0.4
    if kind == "conv":
        most = (4 * 4095 * 1280 if train else 32768 * 2048) // (2 if dtype == "f32" else 1)
        return dict(kind=kind, B=B, L=max(1, min(_log(rng, 16, 32768), most // (B * D))), D=D, K=K, dtype=dtype,
                    train=train, carry=carry, ragged=ragged)
    most = 2 * 8192 * 1280 * 16 if train else 32768 * 2048 * 16
    return dict(kind=kind, B=B, L=max(1, min(_log(rng, 16, 32768), most // (B * D * N))), D=D, N=N, G=G, dtype=dtype,
                train=train, carry=carry, ragged=ragged)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case, g):
    """Lengths of a padded batch: an empty sequence, one of a single token, one
    that fills the batch, the rest in between."""
    B, L = case["B"], case["L"]
    n = torch.randint(0, L + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    n[0] = L
    n[1] = 0
    if B > 2:
        n[2] = 1
    return n


def _inputs(case, seed):
    """The tensors of a case in its own dtype, by name."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, B, D = DT[case["dtype"]], case["B"], case["D"]

    def rnd(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    step = case["kind"].endswith("_step")
    rows = (B,) if step else (B, case["L"])
    s = {"lengths": _lengths(case, g) if case.get("ragged") else None}
    if case["kind"].startswith("conv"):
        K = case["K"]
        s["x"] = rnd(*rows, 2 * D, dtype=dt)[..., :D]   # the projection's rows hold the gate too
        s["weight"] = rnd(D, K) / math.sqrt(K)
        s["bias"] = 0.1 * rnd(D)
        s["state"] = rnd(B, K - 1, D, dtype=dt) if step or case["carry"] else None
    else:
        N, G = case["N"], case["G"]
        x = rnd(*rows, D)
        s["x"] = (x * torch.sigmoid(x)).to(dt)           # what the convolution's activation gives
        s["z"] = rnd(*rows, 2 * D, dtype=dt)[..., D:]
        s["delta"] = rnd(*rows, D, dtype=dt)
        # step sizes spread over 0.001 .. 0.1 by the bias, as such layers are initialised
        dt0 = torch.exp(torch.rand(D, generator=g, device=DEV) * math.log(100.0) + math.log(0.001))
        s["delta_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
        s["A"] = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32).expand(D, N) * torch.exp(0.1 * rnd(D, N))
        s["D"] = 1.0 + 0.1 * rnd(D)
        bc = rnd(*rows, 2 * G * N, dtype=dt)             # one projection's rows hold B and C
        s["B"] = bc[..., :G * N].unflatten(-1, (G, N))
        s["C"] = bc[..., G * N:].unflatten(-1, (G, N))
        s["state"] = rnd(B, D, N) if step or case["carry"] else None
    if case.get("train"):
        s["gout"] = rnd(*rows, D, dtype=dt)
    return s


CONV_LEAVES = ("x", "weight", "bias")
SCAN_LEAVES = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias")


def prepare(case, seed):
    s = _inputs(case, seed)
    if case.get("train"):
        for k in CONV_LEAVES if case["kind"] == "conv" else SCAN_LEAVES:
            s[k] = s[k].detach().requires_grad_(True)
    return {"case": case, **s}


# ---------------------------------------------------------------------------
# the plain form: 32 bits, elementary operations
# ---------------------------------------------------------------------------
def _keep(s, L):
    """[B, L, 1] truth values of the steps inside each sequence, or None."""
    if s["lengths"] is None:
        return None
    return (torch.arange(L, device=DEV) < s["lengths"][:, None])[..., None]


def _silu(v):
    return v * torch.sigmoid(v)


def _silu_slope(v):
    p = torch.sigmoid(v)
    return p * (1 + v * (1 - p))


def _plain_conv(s):
    x, w, dt = s["x"].detach().float(), s["weight"].detach(), s["x"].dtype
    (B, L, D), K = x.shape, w.shape[1]
    keep = _keep(s, L)
    before = x.new_zeros(B, K - 1, D) if s["state"] is None else s["state"].float()
    ext = torch.cat([before, x], dim=1)
    win = ext.unfold(1, K, 1)                                   # [B, L, D, K]
    pre = s["bias"].detach() + (win * w).sum(-1)
    y = _silu(pre)
    out = {"y": (y if keep is None else torch.where(keep, y, 0.0)).to(dt)}
    if s["case"]["carry"]:
        n = torch.full((B,), L, device=DEV) if s["lengths"] is None else s["lengths"].long()
        at = n[:, None, None] + torch.arange(K - 1, device=DEV)[:, None]
        out["state"] = ext.gather(1, at.expand(B, K - 1, D)).to(dt)
    if s["case"]["train"]:
        ds = s["gout"].float() * _silu_slope(pre)
        if keep is not None:
            ds = torch.where(keep, ds, 0.0)
        after = torch.cat([ds, ds.new_zeros(B, K - 1, D)], dim=1).unfold(1, K, 1)
        out["dx"] = (after * w.flip(1)).sum(-1).to(dt)
        out["dweight"] = (ds[..., None] * win).sum((0, 1))
        out["dbias"] = ds.sum((0, 1))
    return out


def _plain_conv_step(s):
    x, state, dt = s["x"].float(), s["state"], s["x"].dtype
    ext = torch.cat([state.float(), x[:, None]], dim=1)
    y = _silu(s["bias"] + (ext * s["weight"].t()).sum(1))
    state.copy_(ext[:, 1:])
    return {"y": y.to(dt), "state": state}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 by recursive doubling, in place."""
    d, L = 1, a.shape[1]
    while d < L:
        b[:, d:] += a[:, d:] * b[:, :-d]
        if 2 * d < L:
            a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return b


def _step_size(s):
    v = s["delta"].detach().float() + s["delta_bias"].detach()
    return v, torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _to_channels(m, D):
    """[..., G, N] of each channel's group as [..., D, N]."""
    return m.detach().float().repeat_interleave(D // m.shape[-2], dim=-2)


def _plain_scan(s):
    x, z, A, skip, dt = (s["x"].detach().float(), s["z"].detach().float(), s["A"].detach(), s["D"].detach(),
                         s["x"].dtype)
    B, L, D = x.shape
    G = s["case"]["G"]
    keep = _keep(s, L)
    raw, step = _step_size(s)
    if keep is not None:
        step = torch.where(keep, step, 0.0)
    w = step * x
    Bc, Cc = _to_channels(s["B"], D), _to_channels(s["C"], D)
    h = w[..., None] * Bc                                       # [B, L, D, N]
    a = torch.exp(step[..., None] * A)
    if s["state"] is not None:
        h[:, 0] += a[:, 0] * s["state"]
    h = _doubling(a, h)
    y = (h * Cc).sum(-1) + skip * x
    o = y * _silu(z)
    out = {"out": (o if keep is None else torch.where(keep, o, 0.0)).to(dt)}
    if s["case"]["carry"]:
        out["state"] = h[:, -1]
    if not s["case"]["train"]:
        return out
    go = s["gout"].float()
    if keep is not None:
        go = torch.where(keep, go, 0.0)
    dy = go * _silu(z)
    out["dz"] = (go * y * _silu_slope(z)).to(dt)
    out["dD"] = (dy * x).sum((0, 1))
    out["dC"] = (dy[..., None] * h).unflatten(2, (G, D // G)).sum(3).to(dt)
    a = torch.exp(step[..., None] * A)
    g = (dy[..., None] * Cc).flip(1)
    later = torch.cat([a.new_ones(B, 1, *a.shape[2:]), a[:, 1:].flip(1)], dim=1)
    g = _doubling(later, g).flip(1)                             # gradient of h_t
    out["dB"] = (g * w[..., None]).unflatten(2, (G, D // G)).sum(3).to(dt)
    dw = (g * Bc).sum(-1)
    out["dx"] = (dw * step + skip * dy).to(dt)
    g[:, 1:] *= a[:, 1:] * h[:, :-1]
    g[:, 0] = 0.0                                               # gradient of dt A now
    out["dA"] = (g * step[..., None]).sum((0, 1))
    ddelta = (dw * x + (g * A).sum(-1)) * torch.sigmoid(raw)
    if keep is not None:
        ddelta = torch.where(keep, ddelta, 0.0)
    out["ddelta"] = ddelta.to(dt)
    out["ddelta_bias"] = ddelta.sum((0, 1))
    return out


def _plain_scan_step(s):
    x, z, state, dt = s["x"].float(), s["z"].float(), s["state"], s["x"].dtype
    D = x.shape[1]
    _, step = _step_size(s)
    h = torch.exp(step[..., None] * s["A"]) * state + (step * x)[..., None] * _to_channels(s["B"], D)
    y = (h * _to_channels(s["C"], D)).sum(-1) + s["D"] * x
    state.copy_(h)
    return {"out": (y * _silu(z)).to(dt), "state": state}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_conv(s):
    from mogt_amd import ops
    got = ops.short_conv(s["x"], s["weight"], s["bias"], activation="silu", initial_state=s["state"],
                         lengths=s["lengths"], return_state=s["case"]["carry"])
    if s["case"]["carry"]:
        return {"y": got[0], "state": got[1]}
    if not s["case"]["train"]:
        return {"y": got}
    grads = torch.autograd.grad(got, [s[k] for k in CONV_LEAVES], s["gout"])
    return {"y": got, **{"d" + k: g for k, g in zip(CONV_LEAVES, grads)}}


def _own_conv_step(s):
    from mogt_amd import ops
    return {"y": ops.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu"),
            "state": s["state"]}


def _own_scan(s):
    from mogt_amd import ops
    got = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                       delta_softplus=True, initial_state=s["state"], lengths=s["lengths"],
                       return_state=s["case"]["carry"])
    if s["case"]["carry"]:
        return {"out": got[0], "state": got[1]}
    if not s["case"]["train"]:
        return {"out": got}
    grads = torch.autograd.grad(got, [s[k] for k in SCAN_LEAVES], s["gout"])
    return {"out": got, **{"d" + k: g for k, g in zip(SCAN_LEAVES, grads)}}


def _own_scan_step(s):
    from mogt_amd import ops
    out = ops.ssm_step(s["x"], s["state"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                       delta_bias=s["delta_bias"], delta_softplus=True)
    return {"out": out, "state": s["state"]}


PLAIN = {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step}
OWN = {"conv": _own_conv, "conv_step": _own_conv_step, "scan": _own_scan, "scan_step": _own_scan_step}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    es, D, kind = SIZE[case["dtype"]], case["D"], case["kind"]
    step = kind.endswith("_step")
    rows = case["B"] * (1 if step else case["L"])
    if kind.startswith("conv"):
        K = case["K"]
        carried = 2 * case["B"] * (K - 1) * D * es if step or case["carry"] else 0
        if case.get("train"):   # x, gradient of y; y, gradient of x; weight and bias, their gradients
            return {"bytes": 4 * rows * D * es + 2 * D * (K + 1) * 4, "flops": rows * D * (6 * K + 16)}
        return {"bytes": 2 * rows * D * es + D * (K + 1) * 4 + carried, "flops": rows * D * (2 * K + 5)}
    N, G = case["N"], case["G"]
    carried = 2 * case["B"] * D * N * 4 if step or case["carry"] else 0
    weights = D * (N + 2) * 4
    if case.get("train"):       # x, delta, z, gradient of out; out, dx, ddelta, dz; B, C and theirs
        return {"bytes": 8 * rows * D * es + 4 * rows * G * N * es + 2 * weights, "flops": rows * D * (26 * N + 50)}
    return {"bytes": 4 * rows * D * es + 2 * rows * G * N * es + weights + carried,
            "flops": rows * D * (7 * N + 20)}


# ---------------------------------------------------------------------------
# the outputs in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _steps(decay, write, h0):
    """h_t = decay_t * h_{t-1} + write_t with h_{-1} = h0 in float64, along
    dim 1: stretches of about sqrt(L) steps side by side, then the states
    between them one after the other, then what they add."""
    B, L = decay.shape[:2]
    m = max(1, math.isqrt(L))
    n = -(-L // m)
    pad = n * m - L
    if pad:
        decay = torch.cat([decay, decay.new_ones(B, pad, *decay.shape[2:])], 1)
        write = torch.cat([write, write.new_zeros(B, pad, *write.shape[2:])], 1)
    decay = decay.reshape(B, n, m, *decay.shape[2:])
    h = write.reshape(decay.shape).clone()
    prod = decay.clone()
    for i in range(1, m):
        h[:, :, i] += decay[:, :, i] * h[:, :, i - 1]
        prod[:, :, i] *= prod[:, :, i - 1]
    carry = h0
    for j in range(n):
        h[:, j] += prod[:, j] * carry[:, None]
        carry = h[:, j, -1]
    return h.reshape(B, n * m, *h.shape[3:])[:, :L]


def _exact_conv(case, s):
    x, w, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
    B, L, D = x.shape
    K = w.shape[1]
    n = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    y, dx, dw, db, last = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias), []
    for b in range(B):
        head = x.new_zeros(K - 1, D) if s["state"] is None else s["state"][b].double()
        e = torch.cat([head, x[b, :n[b]]])
        pre = bias.expand(n[b], D).clone()
        for k in range(K):
            pre += w[:, k] * e[k:k + n[b]]
        p = 1 / (1 + torch.exp(-pre))
        y[b, :n[b]] = pre * p
        last.append(e[n[b]:])
        if case["train"]:
            ds = s["gout"][b, :n[b]].double() * (p + pre * p * (1 - p))
            de = torch.zeros_like(e)
            for k in range(K):
                de[k:k + n[b]] += w[:, k] * ds
                dw[:, k] += (ds * e[k:k + n[b]]).sum(0)
            dx[b, :n[b]] = de[K - 1:]
            db += ds.sum(0)
    out = {"y": y}
    if case["carry"]:
        out["state"] = torch.stack(last)
    if case["train"]:
        out.update(dx=dx, dweight=dw, dbias=db)
    return out


def _exact_scan(case, s):
    x, raw = s["x"].double(), s["delta"].double() + s["delta_bias"].double()
    B, L, D = x.shape
    G, N = case["G"], case["N"]
    live = torch.ones(B, L, 1, device=DEV, dtype=torch.float64)
    if s["lengths"] is not None:
        live = (torch.arange(L, device=DEV)[None, :] < s["lengths"][:, None]).double()[..., None]
    step = torch.logaddexp(raw, torch.zeros_like(raw)) * live
    z = s["z"].double()
    p = 1 / (1 + torch.exp(-z))
    A, skip = s["A"].double(), s["D"].double()
    names = ["out"] + (["dx", "ddelta", "dz"] if case["train"] else [])
    out = {k: torch.zeros_like(x) for k in names}
    if case["carry"]:
        out["state"] = torch.zeros(B, D, N, device=DEV, dtype=torch.float64)
    if case["train"]:
        out.update(dA=torch.zeros_like(A), dB=torch.zeros(B, L, G, N, device=DEV, dtype=torch.float64),
                   dC=torch.zeros(B, L, G, N, device=DEV, dtype=torch.float64), dD=torch.zeros_like(skip),
                   ddelta_bias=torch.zeros_like(skip))
    per = D // G
    wide = max(1, (1 << 26) // (B * L * N))                     # channels at a time
    for g in range(G):
        Bg, Cg = s["B"][:, :, g].double()[:, :, None], s["C"][:, :, g].double()[:, :, None]
        for lo in range(g * per, (g + 1) * per, wide):
            c = slice(lo, min(lo + wide, (g + 1) * per))
            a = torch.exp(step[..., c, None] * A[c])
            w = step[..., c] * x[..., c]
            h0 = a.new_zeros(B, c.stop - c.start, N) if s["state"] is None else s["state"][:, c].double()
            h = _steps(a, w[..., None] * Bg, h0)
            y = (h * Cg).sum(-1) + skip[c] * x[..., c]
            out["out"][..., c] = y * z[..., c] * p[..., c] * live
            if case["carry"]:
                out["state"][:, c] = h[:, -1]
            if not case["train"]:
                continue
            go = s["gout"][..., c].double() * live
            dy = go * z[..., c] * p[..., c]
            out["dz"][..., c] = go * y * (p[..., c] + z[..., c] * p[..., c] * (1 - p[..., c]))
            out["dD"][c] = (dy * x[..., c]).sum((0, 1))
            out["dC"][:, :, g] += (dy[..., None] * h).sum(2)
            # gradient of h_t, backwards in time: its decay is the next step's
            nxt = torch.cat([a[:, 1:], a.new_zeros(B, 1, *a.shape[2:])], 1)
            gh = _steps(nxt.flip(1), (dy[..., None] * Cg).flip(1), torch.zeros_like(h0)).flip(1)
            out["dB"][:, :, g] += (gh * w[..., None]).sum(2)
            dw = (gh * Bg).sum(-1)
            prev = torch.cat([h0[:, None], h[:, :-1]], 1)
            dexp = gh * a * prev                                # gradient of the exponent
            out["dx"][..., c] = dw * step[..., c] + skip[c] * dy
            out["dA"][c] = (dexp * step[..., c, None]).sum((0, 1))
            dd = (dw * x[..., c] + (dexp * A[c]).sum(-1)) / (1 + torch.exp(-raw[..., c])) * live
            out["ddelta"][..., c] = dd
            out["ddelta_bias"][c] = dd.sum((0, 1))
    return out


def _exact_step(case, s):
    if case["kind"] == "conv_step":
        rows = [s["state"][:, k].double() for k in range(case["K"] - 1)] + [s["x"].double()]
        pre = s["bias"].double()
        for k, r in enumerate(rows):
            pre = pre + s["weight"][:, k].double() * r
        return {"y": pre / (1 + torch.exp(-pre)), "state": torch.stack(rows[1:], 1)}
    x, z, per = s["x"].double(), s["z"].double(), case["D"] // case["G"]
    step = torch.logaddexp(s["delta"].double() + s["delta_bias"].double(), torch.zeros_like(x))
    group = torch.arange(case["D"], device=DEV) // per
    h = torch.exp(step[..., None] * s["A"].double()) * s["state"].double() \
        + (step * x)[..., None] * s["B"].double()[:, group]
    y = torch.einsum("bdn,bdn->bd", h, s["C"].double()[:, group]) + s["D"].double() * x
    return {"out": y * z / (1 + torch.exp(-z)), "state": h}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"].endswith("_step"):
        return _exact_step(case, s)
    return (_exact_conv if case["kind"] == "conv" else _exact_scan)(case, s)
