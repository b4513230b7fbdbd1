"""Performance cases of the operators of a linear attention layer: linear attention with a decay for each head (prompts, training, single tokens), the residual norm with an 8-bit output, and the matrix product on 8-bit blocks.

``listed()`` is the fixed set, ``draw(rng)`` one more case of the same ranges.
``prepare`` makes what the program holds before the call (inputs on the GPU,
made from the seed alone), ``run`` is one pass and returns its whole outputs,
``work`` the bytes and operations the pass cannot do without, and ``exact`` the
same outputs in 64 bits from the operators' definitions.  With ``own`` false
``run`` computes in plain torch (32 bits, rounded once), with ``own`` true
through the framework's entry points.

Kinds of case:

* ``attn``    S_t = exp(g_t) S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t  per head;
              q, k [batch, time, groups, dk], v [batch, time, heads, dv], each
              group's q and k shared by heads / groups consecutive heads; the
              log decay g [batch, time, heads], or [heads] (``decay`` "head")
* ``step``    one token of it, the states updated in place
* ``norm``    x' = x + scale z,  n = rmsnorm(x') weight, each row's blocks of 128
              values of n in e4m3 with a scale
* ``linear``  y = x w^T for x in e4m3 with a scale for every row's 128 values and
              w in e4m3 with a scale for every 128 by 128 values

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
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
TINY = 2.0 ** -126
BLOCK = 128
EPS = 1e-6
RES_SCALE = 0.5


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # A short prompt, one sequence of the framework's 12 heads of 64: latency of the smallest call.
        dict(name="attn_short", kind="attn", B=1, L=200, H=12, G=12, dk=64, dv=64, dtype="bf16", decay="token",
             train=False, carry=True, ragged=False),
        # A padded batch of prompts of different lengths in fp32, q and k shared by three heads each.
        dict(name="attn_ragged", kind="attn", B=8, L=1001, H=12, G=4, dk=64, dv=64, dtype="f32", decay="token",
             train=False, carry=True, ragged=True),
        # The longest context of the framework's benchmark (32768 steps), one sequence, wide heads.
        dict(name="attn_long", kind="attn", B=1, L=32768, H=16, G=16, dk=128, dv=128, dtype="bf16", decay="token",
             train=False, carry=True, ragged=False),
        # A small training step in fp32: odd length, narrow shared keys, one decay a head, states carried across pieces.
        dict(name="attn_train_small", kind="attn", B=2, L=513, H=6, G=2, dk=48, dv=64, dtype="f32", decay="head",
             train=True, carry=True, ragged=False),
        # One layer of a training step.
        dict(name="attn_train", kind="attn", B=2, L=8192, H=12, G=12, dk=64, dv=64, dtype="bf16", decay="token",
             train=True, carry=False, ragged=False),
        # One token of an interactive program, and of a server with 256 sequences.
        dict(name="step_1", kind="step", B=1, H=12, G=12, dk=64, dv=64, dtype="bf16", decay="token"),
        dict(name="step_256", kind="step", B=256, H=16, G=16, dk=128, dv=128, dtype="bf16", decay="token"),
        # The norm before a projection: a short prompt, and the longest context.
        dict(name="norm_short", kind="norm", M=200, D=768, dtype="bf16"),
        dict(name="norm_long", kind="norm", M=32768, D=2048, dtype="bf16"),
        # A projection for one token, for a few hundred odd rows, and for the longest context.
        dict(name="linear_1", kind="linear", M=1, N=6144, K=2048, dtype="bf16"),
        dict(name="linear_odd", kind="linear", M=501, N=2304, K=768, dtype="f32"),
        dict(name="linear_long", kind="linear", M=32768, N=6144, K=2048, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "step", "norm", "linear", "linear"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    if kind == "norm":
        return dict(kind=kind, M=_log(rng, 1, 32768), D=16 * _log(rng, 4, 128), dtype=dtype)
    if kind == "linear":
        M, N, K = _log(rng, 1, 32768), _log(rng, 17, 6144), 16 * _log(rng, 4, 128)
        return dict(kind=kind, M=M, N=N, K=K, dtype=dtype)
    H = rng.choice([1, 3, 4, 6, 12, 16])
    G = H // rng.choice([n for n in (1, 1, 1, 2, 3, 4) if H % n == 0])
    dk, dv = (rng.choice([16, 24, 33, 48, 64, 64, 100, 128, 128]) for _ in range(2))
    decay = rng.choice(["token", "token", "head"])
    if kind == "step":
        return dict(kind=kind, B=_log(rng, 1, 256), H=H, G=G, dk=dk, dv=dv, dtype=dtype, decay=decay)
    train = rng.random() < 0.5
    B = rng.choice([1, 1, 2, 3, 8])
    most = (2 * 8192 * 12 * 128 if train else 32768 * 16 * 256) // (2 if dtype == "f32" else 1)
    return dict(kind=kind, B=B, L=max(1, min(_log(rng, 16, 32768), most // (B * H * (dk + dv)))), H=H, G=G, dk=dk,
                dv=dv, dtype=dtype, decay=decay, train=train, carry=rng.random() < 0.5,
                ragged=B > 1 and rng.random() < 0.4)


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


def _eight_bits(x, rows):
    """x [M, K] in e4m3 with a scale for every block of ``rows`` by 128 values."""
    M, K = x.shape
    pad = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -M % rows))
    tiles = pad.view(pad.shape[0] // rows, rows, pad.shape[1] // BLOCK, BLOCK)
    scale = (tiles.abs().amax((1, 3)) / F8_MAX).clamp(min=TINY)
    q = (tiles / scale[:, None, :, None]).view(pad.shape)[:M, :K].contiguous().to(F8)
    return q, scale


def _inputs(case, seed):
    """The tensors of a case in its own dtype, by name."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, kind = DT[case["dtype"]], case["kind"]

    def rnd(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    if kind == "norm":
        M, D = case["M"], case["D"]
        return {"x": rnd(M, D) * 2.0, "z": rnd(M, D, dtype=dt), "weight": 1.0 + 0.1 * rnd(D)}
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x, xs = _eight_bits(rnd(M, K) * torch.exp(0.5 * rnd(M, 1)), 1)
        w, ws = _eight_bits(rnd(N, K) / math.sqrt(K), BLOCK)
        return {"x": x, "x_scale": xs, "w": w, "w_scale": ws}
    B, H, G, dk, dv = (case[n] for n in ("B", "H", "G", "dk", "dv"))
    rows = (B,) if kind == "step" else (B, case["L"])
    s = {"lengths": _lengths(case, g) if case.get("ragged") else None}
    qkv = rnd(*rows, 2 * G * dk + H * dv, dtype=dt)             # one projection's rows hold all three
    s["q"] = qkv[..., :G * dk].unflatten(-1, (G, dk))
    s["k"] = qkv[..., G * dk:2 * G * dk].unflatten(-1, (G, dk))
    s["v"] = qkv[..., 2 * G * dk:].unflatten(-1, (H, dv))
    # heads that forget within a few tokens beside heads that remember hundreds
    rate = torch.exp(torch.rand(H, generator=g, device=DEV) * math.log(100.0) + math.log(0.002))
    s["log_decay"] = -rate if case["decay"] == "head" else -rate * torch.log1p(torch.exp(rnd(*rows, H)))
    s["state"] = rnd(B, H, dk, dv) if kind == "step" or case["carry"] else None
    if case.get("train"):
        s["gout"] = rnd(*rows, H, dv, dtype=dt)
        if case["carry"]:
            s["gstate"] = rnd(B, H, dk, dv)
    return s


def _leaves(case):
    return ("q", "k", "v", "log_decay") + (("state",) if case["carry"] else ())


def prepare(case, seed):
    s = _inputs(case, seed)
    if case.get("train"):
        for n in _leaves(case):
            s[n] = s[n].detach().requires_grad_(True)
    return {"case": case, **s}


# ---------------------------------------------------------------------------
# the plain form: 32 bits, elementary operations
# ---------------------------------------------------------------------------
T = 64      # steps of a chunk


def _chunks(t, L):
    """[B, L, H, d] as fp32 [B, H, chunks, T, d], zero past L."""
    t = torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, -L % T))
    return t.unflatten(1, (-1, T)).permute(0, 3, 1, 2, 4)


def _rows(t, L):
    """The inverse of _chunks."""
    return t.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :L]


def _plain_attn(s):
    case, q, k, v = s["case"], s["q"].detach(), s["k"].detach(), s["v"].detach()
    B, L, H, dv = v.shape
    G, dk, dt, scale, device = q.shape[2], q.shape[3], q.dtype, q.shape[3] ** -0.5, q.device
    g = s["log_decay"].detach().expand(B, L, H)[..., None]
    keep = None
    if s["lengths"] is not None:
        keep = (torch.arange(L, device=device) < s["lengths"][:, None])[..., None, None]
        q, k, v, g = (torch.where(keep, t, 0.0) for t in (q, k, v, g))
    q, k, v = (_chunks(t, L) for t in (q.repeat_interleave(H // G, 2), k.repeat_interleave(H // G, 2), v))
    c = _chunks(g, L)[..., 0].double().cumsum(-1)               # log decay since the chunk's start
    n = c.shape[2]
    start = torch.nn.functional.pad(c[..., -1].cumsum(-1), (1, 0))   # ... of the chunks' starts, and the end
    tri = torch.ones(T, T, dtype=torch.bool, device=device).tril()
    D = torch.exp(torch.where(tri, c[..., :, None] - c[..., None, :], -math.inf)).float() * scale
    into, rest = torch.exp(c).float()[..., None], torch.exp(c[..., -1:] - c).float()[..., None]
    # the states at the chunks' starts and at the end, from what each chunk writes
    before = torch.arange(n + 1, device=device)[:, None] > torch.arange(n, device=device)
    M = torch.exp(torch.where(before, start[..., :, None] - start[..., None, 1:], -math.inf)).float()
    wrote = k.transpose(-1, -2) @ (rest * v)
    S = (M @ wrote.flatten(3)).unflatten(3, (dk, dv))
    if s["state"] is not None:
        S = S + torch.exp(start).float()[..., None, None] * s["state"].detach()[:, :, None]
    P = (q @ k.transpose(-1, -2)) * D
    o = P @ v + scale * into * (q @ S[:, :, :-1])
    out = {"o": _rows(o, L).to(dt)}
    if case["carry"]:
        out["state"] = S[:, :, -1]
    if not case["train"]:
        return out
    do = s["gout"] if keep is None else torch.where(keep, s["gout"], 0.0)
    do = _chunks(do, L)
    # the states' gradients at the chunks' ends, and at the start of all
    read = scale * (q.transpose(-1, -2) @ (into * do))
    after = torch.arange(n, device=device) >= torch.arange(n + 1, device=device)[:, None]
    M = torch.exp(torch.where(after, start[..., None, :-1] - start[..., :, None], -math.inf)).float()
    dS = (M @ read.flatten(3)).unflatten(3, (dk, dv))
    if case["carry"]:
        dS = dS + torch.exp(start[..., -1:] - start).float()[..., None, None] * s["gstate"][:, :, None]
        out["dstate"] = dS[:, :, 0]
    dS, S, end = dS[:, :, 1:], S[:, :, :-1], S[:, :, 1:]
    dP = (do @ v.transpose(-1, -2)) * D
    far_q = scale * into * (do @ S.transpose(-1, -2))
    far_k = rest * (v @ dS.transpose(-1, -2))
    dq, dk_ = dP @ k + far_q, dP.transpose(-1, -2) @ q + far_k
    dv_ = P.transpose(-1, -2) @ do + rest * (k @ dS)
    W = P * (do @ v.transpose(-1, -2))
    dc = W.sum(-1) - W.sum(-2) + (q * far_q).sum(-1) - (k * far_k).sum(-1)
    dc[..., -1] += (end * dS).sum((-1, -2))
    dg = _rows(dc.flip(-1).cumsum(-1).flip(-1)[..., None], L)[..., 0]
    if keep is not None:
        dg = torch.where(keep[..., 0], dg, 0.0)
    out["dlog_decay"] = dg.sum((0, 1)) if case["decay"] == "head" else dg
    out["dq"] = _rows(dq, L).unflatten(2, (G, H // G)).sum(3).to(dt)
    out["dk"] = _rows(dk_, L).unflatten(2, (G, H // G)).sum(3).to(dt)
    out["dv"] = _rows(dv_, L).to(dt)
    return out


def _plain_step(s):
    q, k, v, state = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    n = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(n, 1), k.repeat_interleave(n, 1)
    S = torch.exp(s["log_decay"])[..., None, None] * state + k[..., None] * v[..., None, :]
    o = q.shape[-1] ** -0.5 * (q[..., None] * S).sum(-2)
    state.copy_(S)
    return {"o": o.to(s["v"].dtype), "state": state}


def _plain_norm(s):
    x = s["x"] + RES_SCALE * s["z"].float()
    n = (x * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float()) * s["weight"]
    q, scale = _eight_bits(n, 1)
    return {"x": x, "q": q, "scale": scale}


def _plain_linear(s):
    x, w, K = s["x"].float(), s["w"].float(), s["x"].shape[1]
    x = x * s["x_scale"].repeat_interleave(BLOCK, 1)[:, :K]
    w = w * s["w_scale"].repeat_interleave(BLOCK, 1)[:, :K].repeat_interleave(BLOCK, 0)[:w.shape[0]]
    return {"y": (x @ w.t()).to(DT[s["case"]["dtype"]])}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_attn(s):
    from mogt_amd import ops
    case = s["case"]
    got = ops.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state"],
                               lengths=s["lengths"], return_state=case["carry"])
    out = {"o": got[0], "state": got[1]} if case["carry"] else {"o": got}
    if case["train"]:
        names = _leaves(case)
        grads = torch.autograd.grad(list(out.values()), [s[n] for n in names],
                                    [s["gout"]] + ([s["gstate"]] if case["carry"] else []))
        out.update({"d" + n: t for n, t in zip(names, grads)})
    return out


def _own_step(s):
    from mogt_amd import ops
    return {"o": ops.linear_attention_step(s["q"], s["k"], s["v"], s["state"], s["log_decay"]), "state": s["state"]}


def _own_norm(s):
    from mogt_amd import ops
    x, q, scale = ops.add_rmsnorm_fp8(s["x"], s["z"], RES_SCALE, s["weight"], EPS)
    return {"x": x, "q": q, "scale": scale}


def _own_linear(s):
    from mogt_amd import ops
    return {"y": ops.linear_fp8(s["x"], s["x_scale"], s["w"], s["w_scale"], out_dtype=DT[s["case"]["dtype"]])}


PLAIN = {"attn": _plain_attn, "step": _plain_step, "norm": _plain_norm, "linear": _plain_linear}
OWN = {"attn": _own_attn, "step": _own_step, "norm": _own_norm, "linear": _own_linear}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    es, kind = SIZE[case["dtype"]], case["kind"]
    if kind == "norm":          # x and z; the sum, its norm and the scales
        M, D = case["M"], case["D"]
        return {"bytes": M * (D * (4 + es + 4 + 1) + 4 * -(-D // BLOCK)) + 4 * D, "flops": 8 * M * D}
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // BLOCK)
        return {"bytes": M * K + N * K + M * N * es + 4 * kb * (M + -(-N // BLOCK)), "flops": 2 * M * N * K}
    B, H, G, dk, dv = (case[n] for n in ("B", "H", "G", "dk", "dv"))
    rows = B * (1 if kind == "step" else case["L"])
    read = (2 * G * dk + H * dv) * es + (4 * H if case["decay"] == "token" else 0)
    states = 2 * B * H * dk * dv * 4 if kind == "step" or case["carry"] else 0
    # a token's read and write of a state: the recurrence itself, the least that a form of it computes
    if not case.get("train"):
        return {"bytes": rows * (read + H * dv * es) + states, "flops": rows * H * dk * dv * 5}
    return {"bytes": rows * (2 * read + 2 * H * dv * es) + 2 * states, "flops": rows * H * dk * dv * 18}


# ---------------------------------------------------------------------------
# the outputs in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_attn(case, s):
    """Every pair of steps by itself, rows of 1024 outputs at a time."""
    B, L, H, G, dk, dv = (case[n] for n in ("B", "L", "H", "G", "dk", "dv"))
    carry, train, scale = case["carry"], case["train"], 1.0 / math.sqrt(case["dk"])

    def zeros(*shape):
        return torch.zeros(*shape, device=DEV, dtype=torch.float64)

    out = {"o": zeros(B, L, H, dv)}
    if carry:
        out["state"] = zeros(B, H, dk, dv)
    if train:
        out.update(dq=zeros(B, L, G, dk), dk=zeros(B, L, G, dk), dv=zeros(B, L, H, dv), dlog_decay=zeros(B, L, H))
        if carry:
            out["dstate"] = zeros(B, H, dk, dv)
    lens = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = lens[b]
        for h in range(H):
            S0 = s["state"][b, h].double() if carry else zeros(dk, dv)
            dSn = s["gstate"][b, h].double() if train and carry else zeros(dk, dv)
            if n == 0:
                if carry:
                    out["state"][b, h] = S0
                if train and carry:
                    out["dstate"][b, h] = dSn
                continue
            j = h // (H // G)
            q, k, v = s["q"][b, :n, j].double() * scale, s["k"][b, :n, j].double(), s["v"][b, :n, h].double()
            ld = s["log_decay"]
            c = (ld[h].expand(n) if ld.ndim == 1 else ld[b, :n, h]).double().cumsum(0)
            e, r = torch.exp(c)[:, None], torch.exp(c[-1] - c)[:, None]
            if carry:
                out["state"][b, h] = e[-1] * S0 + k.t() @ (r * v)
            if train:
                do = s["gout"][b, :n, h].double()
                dq, dk_, dv_, dc = e * (do @ S0.t()), r * (v @ dSn.t()), r * (k @ dSn), zeros(n)
                dc += (q * dq).sum(1) - (k * dk_).sum(1)
                dc[-1] += (dSn * (e[-1] * S0 + k.t() @ (r * v))).sum()
                if carry:
                    out["dstate"][b, h] = e[-1] * dSn + q.t() @ (e * do)
            for lo in range(0, n, 1024):
                hi = min(lo + 1024, n)
                w = (c[lo:hi, None] - c[None, :hi]).exp_().tril_(lo)
                p = (q[lo:hi] @ k[:hi].t()) * w
                out["o"][b, lo:hi, h] = p @ v[:hi] + e[lo:hi] * (q[lo:hi] @ S0)
                if train:
                    x = do[lo:hi] @ v[:hi].t()
                    dv_[:hi] += p.t() @ do[lo:hi]
                    p *= x
                    dc[lo:hi] += p.sum(1)
                    dc[:hi] -= p.sum(0)
                    x *= w
                    dq[lo:hi] += x @ k[:hi]
                    dk_[:hi] += x.t() @ q[lo:hi]
            if train:
                out["dq"][b, :n, j] += dq * scale
                out["dk"][b, :n, j] += dk_
                out["dv"][b, :n, h] = dv_
                out["dlog_decay"][b, :n, h] = dc.flip(0).cumsum(0).flip(0)
    if train and case["decay"] == "head":
        out["dlog_decay"] = out["dlog_decay"].sum((0, 1))
    return out


def _exact_step(case, s):
    h = torch.arange(case["H"], device=DEV) // (case["H"] // case["G"])
    q, k, v = s["q"].double()[:, h], s["k"].double()[:, h], s["v"].double()
    a = torch.exp(s["log_decay"].double())
    S = a[..., None, None] * s["state"].double() + torch.einsum("bhi,bhj->bhij", k, v)
    return {"o": torch.einsum("bhi,bhij->bhj", q, S) / math.sqrt(case["dk"]), "state": S}


def _exact_norm(case, s):
    x = s["x"].double() + RES_SCALE * s["z"].double()
    n = x / torch.sqrt((x * x).sum(1, keepdim=True) / case["D"] + EPS) * s["weight"].double()
    scale = torch.stack([b.abs().amax(1) / F8_MAX for b in n.split(BLOCK, 1)], 1).clamp(min=TINY)
    # e4m3 by hand: 3 bits below the leading one, and 2^-9 the least
    u = n / scale.repeat_interleave(BLOCK, 1)[:, :case["D"]]
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return {"x": x, "q": torch.round(u / step) * step, "scale": scale}


def _exact_linear(case, s):
    y = torch.zeros(case["M"], case["N"], device=DEV, dtype=torch.float64)
    for i, lo in enumerate(range(0, case["K"], BLOCK)):
        k = slice(lo, lo + BLOCK)
        w = s["w"][:, k].double() * s["w_scale"][:, i].double().repeat_interleave(BLOCK)[:case["N"], None]
        y += (s["x"][:, k].double() * s["x_scale"][:, i, None].double()) @ w.t()
    return {"y": y}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"attn": _exact_attn, "step": _exact_step, "norm": _exact_norm, "linear": _exact_linear}[case["kind"]](case, s)
