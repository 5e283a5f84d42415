"""The gated delta rule (whole sequences, training, single tokens) and group
norm with an activation: the cases that are timed, their plain form and their
exact values.

Notation, per batch row b and head h: values u_t [P], keys B_t [N], queries
C_t [N] (G key heads; head h reads key head h // (H // G)), step dt_t, write
strength beta_t, state S [N, P]:

    S' = exp(-exp(A_log) dt_t) S_{t-1}
    S_t = S' + beta_t B_t (u_t - S'^T B_t)^T ,   y_t = scale * S_t^T C_t

Group norm: x [Bt, L, C]; mean and variance over the L positions and the
C / groups channels of a group, then weight and bias per channel, then the
activation.  L = 1 is the norm of one token's head groups.
"""
import math

import torch

own = False

CHUNK = 64
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one stream's next token: launch latency
        _step("step_one_stream", 1, 16, 16, 128, 128, "bf16"),
        # a full serving batch: the states stream through HBM
        _step("step_batch", 192, 32, 16, 128, 128, "bf16"),
        # a short odd prompt continued from a state, in f32
        _delta("prompt_short_f32", 1, 77, 8, 4, 64, 64, "f32", True),
        # ordinary prefill: a few sequences, final states kept for decoding
        _delta("prefill", 2, 2048, 16, 16, 128, 128, "bf16", False),
        # the largest prefill: every GPU's worth of heads, shared key heads
        _delta("prefill_large", 8, 4096, 32, 16, 128, 128, "bf16", True),
        # training on a ragged, narrow model in f32 (gradient checks, small studies)
        _train("train_ragged_f32", 2, 333, 4, 2, 64, 48, "f32"),
        # an ordinary training step of one layer
        _train("train", 4, 2048, 16, 8, 128, 128, "bf16"),
        # head norm of one decoded token per stream
        _norm("norm_tokens_small", 16, 1, 2048, 32, "bf16", "silu", False),
        # head norm of a prefill's outputs
        _norm("norm_tokens", 32768, 1, 4096, 32, "bf16", "silu", False),
        # feature maps of irregular series, stats over odd lengths
        _norm("norm_maps_f32", 4, 5000, 768, 24, "f32", "none", False),
        # training over feature maps
        _norm("norm_maps_train", 8, 4096, 1024, 16, "bf16", "silu", True),
        # training the head norm
        _norm("norm_tokens_train_f32", 6000, 1, 1536, 24, "f32", "silu", True),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def _step(name, S, H, G, N, P, dtype):
    return _named(name, {"op": "step", "S": S, "H": H, "G": G, "N": N, "P": P, "dtype": dtype})


def _delta(name, Bt, L, H, G, N, P, dtype, h0):
    return _named(name, {"op": "delta", "Bt": Bt, "L": L, "H": H, "G": G, "N": N, "P": P, "dtype": dtype, "h0": h0})


def _train(name, Bt, L, H, G, N, P, dtype):
    return _named(name, {"op": "train", "Bt": Bt, "L": L, "H": H, "G": G, "N": N, "P": P, "dtype": dtype})


def _norm(name, Bt, L, C, groups, dtype, act, train):
    return _named(name, {"op": "norm", "Bt": Bt, "L": L, "C": C, "groups": groups, "dtype": dtype, "act": act,
                         "train": train})


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["step", "delta", "train", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        groups = rng.choice([1, 2, 4, 8, 16, 24, 32])
        train = rng.random() < 0.5
        width = rng.choice([4, 16, 32, 48, 64, 128])
        C = groups * width
        most = (1 << 24) if dtype == "f32" or train else (1 << 26)
        if rng.random() < 0.5:
            return _norm(None, _log(rng, 1, min(40000, max(1, most // C))), 1, C, groups, dtype,
                         rng.choice(["silu", "none"]), train)
        Bt = _log(rng, 1, 12)
        return _norm(None, Bt, _log(rng, 2, min(20000, max(2, most // (C * Bt)))), C, groups, dtype,
                     rng.choice(["silu", "none"]), train)
    G = _log(rng, 1, 16)
    H = G * rng.choice([1, 1, 2, 4] if G <= 8 else [1, 2])
    N = rng.choice([64, 128, 128, rng.randrange(16, 129, 8)])
    P = rng.choice([64, 128, 128, rng.randrange(16, 129, 8)])
    if op == "step":
        return _step(None, _log(rng, 1, min(256, 6144 // H)), H, G, N, P, dtype)
    heads = 256 if op == "delta" else 64
    Bt = _log(rng, 1, min(8, heads // H) or 1)
    most = (1 << 20 if op == "delta" else 1 << 17) // (Bt * H)
    if dtype == "f32":
        most //= 4
    L = _log(rng, 1, max(1, min(4096 if op == "delta" else 2048, most)))
    if op == "delta":
        return _delta(None, Bt, L, H, G, N, P, dtype, rng.random() < 0.5)
    return _train(None, Bt, L, H, G, N, P, dtype)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device=dev) * (hi - lo) + lo

    def unit(*shape):
        x = normal(*shape)
        return (x / x.norm(dim=-1, keepdim=True)).to(t)

    if case["op"] == "norm":
        Bt, L, C = case["Bt"], case["L"], case["C"]
        offset = normal(Bt, 1, C) * 0.5
        s = {"x": (normal(Bt, L, C) * uniform(0.5, 2.0, C) + offset).to(t), "weight": 1.0 + 0.2 * normal(C),
             "bias": 0.2 * normal(C)}
        if case["train"]:
            s["dy"] = normal(Bt, L, C).to(t)
        return dict(s, case=case)
    H, G, N, P = case["H"], case["G"], case["N"], case["P"]
    s = {"A_log": torch.log(uniform(0.5, 16.0, H)), "case": case, "scale": N ** -0.5}
    if case["op"] == "step":
        S = case["S"]
        s.update(x=normal(S, H, P).to(t), B=unit(S, G, N), C=(unit(S, G, N).float() * N ** 0.5).to(t),
                 dt=torch.exp(uniform(-6.9, 0.0, S, H)), beta=torch.sigmoid(normal(S, H)), h=normal(S, H, P, N) * 0.3)
        return s
    Bt, L = case["Bt"], case["L"]
    s.update(u=normal(Bt, L, H * P).to(t), B=unit(Bt, L, G, N), C=(unit(Bt, L, G, N).float() * N ** 0.5).to(t),
             dt=torch.exp(uniform(-6.9, 0.0, Bt, L, H)), beta=torch.sigmoid(normal(Bt, L, H)))
    s["h0"] = normal(Bt, H, P, N) * 0.3 if case.get("h0", True) else None
    if case["op"] == "train":
        s["dy"] = normal(Bt, L, H * P).to(t)
        s["dh_last"] = normal(Bt, H, P, N) * 0.3
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"step": _own_step, "delta": _own_delta, "train": _own_train, "norm": _own_norm}[op](s)
    return {"step": _plain_step, "delta": _plain_delta, "train": _plain_train, "norm": _plain_norm}[op](s)


def _own_step(s):
    import triton_ssm_b200 as ts
    y = ts.gated_delta_step(s["x"], s["dt"], s["h"], s["A_log"], s["B"], s["C"], s["beta"], scale=s["scale"])
    return {"y": y, "h": s["h"]}


def _own_delta(s):
    import triton_ssm_b200 as ts
    y, h = ts.gated_delta_rule(s["u"], s["A_log"], s["B"], s["C"], s["dt"], s["beta"], scale=s["scale"], h0=s["h0"],
                               return_state=True)
    return {"y": y, "h": h}


_GRADS = ("du", "dA_log", "dB", "dC", "ddt", "dbeta", "dh0")


def _own_train(s):
    import triton_ssm_b200 as ts
    a = (s["u"], s["A_log"], s["B"], s["C"], s["dt"], s["beta"])
    y, saved = ts.gated_delta_rule(*a, scale=s["scale"], h0=s["h0"], save=True)
    grads = ts.gated_delta_rule_bwd(*a, s["dy"], saved, scale=s["scale"], dh_last=s["dh_last"])
    return dict(zip(_GRADS, grads), y=y)


def _own_norm(s):
    import triton_ssm_b200 as ts
    c = s["case"]
    if not c["train"]:
        return {"y": ts.group_norm_act(s["x"], s["weight"], s["bias"], c["groups"], act=c["act"])}
    y, mean, rstd = ts.group_norm_act(s["x"], s["weight"], s["bias"], c["groups"], act=c["act"], return_stats=True)
    dx, dw, db = ts.group_norm_act_bwd(s["dy"], s["x"], s["weight"], s["bias"], mean, rstd, act=c["act"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


# ------------------------------------------------------------------ plain form
def _plain_step(s):
    x, h, t = s["x"].float(), s["h"], s["x"].dtype
    rep = x.shape[1] // s["B"].shape[1]
    k, q = (s[n].float().repeat_interleave(rep, 1) for n in ("B", "C"))
    hd = h * torch.exp(-torch.exp(s["A_log"]) * s["dt"])[..., None, None]
    e = s["beta"][..., None] * (x - (hd @ k[..., None])[..., 0])
    h.copy_(hd + e[..., :, None] * k[..., None, :])
    return {"y": (s["scale"] * (h @ q[..., None])[..., 0]).to(t), "h": h}


def _blocks(x, n):
    """[Bt, L, H, ...] -> [Bt, H, n, CHUNK, ...] in f32, zeros behind the end."""
    x = x.to(torch.float64 if x.dtype == torch.float64 else torch.float32)
    x = torch.cat([x, x.new_zeros(x.shape[0], n * CHUNK - x.shape[1], *x.shape[2:])], 1)
    return x.unflatten(1, (n, CHUNK)).movedim(3, 1)


def _rows(x, L):
    """The inverse of _blocks, cut to L tokens."""
    return x.movedim(1, 3).flatten(1, 2)[:, :L]


def _plain_chunks(s):
    """The chunked form's inputs: everything that no state enters."""
    Bt, L, HP = s["u"].shape
    G, N = s["B"].shape[2:]
    H = s["dt"].shape[2]
    n = -(-L // CHUNK)
    v = _blocks(s["u"].unflatten(2, (H, HP // H)), n)
    k, q = (_blocks(s[m], n).repeat_interleave(H // G, 1) for m in ("B", "C"))
    beta = _blocks(s["beta"], n)
    lam = torch.cumsum(_blocks(s["dt"].double() * -torch.exp(s["A_log"].double()), n), -1)   # differences of long sums
    low = torch.ones(CHUNK, CHUNK, device=v.device).tril().bool()
    D = torch.exp((lam[..., :, None] - lam[..., None, :]).masked_fill(~low, -math.inf)).float()
    c = {"v": v, "k": k, "q": q, "beta": beta, "D": D, "eg": torch.exp(lam).float(),
         "w": torch.exp(lam[..., -1:] - lam).float(), "scale": s["scale"]}
    c["A"] = (D * (k @ k.mT)).tril(-1)
    M = c["A"] * beta[..., None, :]
    T = torch.zeros_like(M) + torch.eye(CHUNK, device=v.device)
    for i in range(1, CHUNK):   # (I + A diag(beta))^-1, row by row
        T[..., i, :i] = -(M[..., i:i + 1, :i] @ T[..., :i, :i])[..., 0, :]
    c["T"], c["Aq"] = T, s["scale"] * D * (q @ k.mT)
    return c


def _plain_scan(s, c):
    Bt, H, n, _, P = c["v"].shape
    N = c["k"].shape[-1]
    S = s["h0"].mT.float() if s["h0"] is not None else c["v"].new_zeros(Bt, H, N, P)
    ys, es, starts = [], [], []
    for i in range(n):
        k, eg = c["k"][:, :, i], c["eg"][:, :, i, :, None]
        starts.append(S)
        e = c["T"][:, :, i] @ (c["v"][:, :, i] - eg * (k @ S))
        r = c["beta"][:, :, i, :, None] * e
        ys.append(c["scale"] * eg * (c["q"][:, :, i] @ S) + c["Aq"][:, :, i] @ r)
        S = eg[:, :, -1:] * S + k.mT @ (c["w"][:, :, i, :, None] * r)
        es.append(e)
    return torch.stack(ys, 2), S, starts, es


def _plain_delta(s):
    Bt, L, HP = s["u"].shape
    y, S, _, _ = _plain_scan(s, _plain_chunks(s))
    return {"y": _rows(y, L).reshape(Bt, L, HP).to(s["u"].dtype), "h": S.mT.contiguous()}


def _suffix(x, dim):
    return torch.flip(torch.cumsum(torch.flip(x, (dim,)), dim), (dim,))


def _plain_train(s):
    c = _plain_chunks(s)
    y, S, starts, es = _plain_scan(s, c)
    Bt, L, HP = s["u"].shape
    H, t, scale = s["dt"].shape[2], s["u"].dtype, s["scale"]
    n = len(starts)
    dO = _blocks(s["dy"].unflatten(2, (H, HP // H)), n)
    dS = s["dh_last"].mT.float()
    out = {m: [] for m in ("dv", "dk", "dq", "dbeta", "dlam")}
    for i in reversed(range(n)):
        k, q, e, do = c["k"][:, :, i], c["q"][:, :, i], es[i], dO[:, :, i]
        eg, w, b = (c[m][:, :, i, :, None] for m in ("eg", "w", "beta"))
        D, A, S0 = c["D"][:, :, i], c["A"][:, :, i], starts[i]
        dr = c["Aq"][:, :, i].mT @ do + w * (k @ dS)
        de = c["T"][:, :, i].mT @ (b * dr)
        m1 = scale * D * (do @ (b * e).mT)
        ee = de @ e.mT
        m2 = D.tril(-1) * ee * b.mT
        dq0, dk0, dk1 = scale * eg * (do @ S0.mT), -eg * (de @ S0.mT), (w * b * e) @ dS.mT
        dq = dq0 + m1 @ k
        dk = dk0 + dk1 + m1.mT @ q - m2 @ k - m2.mT @ k
        # dlam_t: every path over token t's decay (from before it to t or later), so that nothing cancels
        X = _suffix(torch.cumsum((c["Aq"][:, :, i] * (do @ e.mT) - A * ee) * b.mT, -1), -2)
        into, outof = ((dq0 * q + dk0 * k)).sum(-1), torch.cumsum((dk1 * k).sum(-1), -1)
        dl = _suffix(into, -1) + (eg[:, :, -1:] * dS * S0).sum((-1, -2))[..., None]
        dl[..., 1:] += outof[..., :-1] + torch.diagonal(X, -1, -2, -1)
        out["dlam"].append(dl)
        out["dbeta"].append((e * dr).sum(-1) - (A * ee).sum(-2))
        for m, x in (("dv", de), ("dk", dk), ("dq", dq)):
            out[m].append(x)
        dS = eg[:, :, -1:] * dS + k.mT @ (-eg * de) + q.mT @ (scale * eg * do)
    o = {m: _rows(torch.stack(x[::-1], 2), L) for m, x in out.items()}
    G = s["B"].shape[2]
    dk, dq = (o[m].unflatten(2, (G, H // G)).sum(3).to(t) for m in ("dk", "dq"))
    a = -torch.exp(s["A_log"])
    return {"y": _rows(y, L).reshape(Bt, L, HP).to(t), "du": o["dv"].reshape(Bt, L, HP).to(t), "dB": dk, "dC": dq,
            "ddt": o["dlam"] * a, "dbeta": o["dbeta"], "dA_log": (o["dlam"] * s["dt"]).double().sum((0, 1)).float() * a,
            "dh0": dS.mT.contiguous()}


def _plain_norm(s):
    c, t = s["case"], s["x"].dtype
    x = s["x"].float().unflatten(2, (c["groups"], -1))
    mean = x.double().mean((1, 3), keepdim=True)        # long sums
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + 1e-5).float()
    xh = ((x - mean.float()) * rstd).flatten(2)
    z = xh * s["weight"] + s["bias"]
    sg = torch.sigmoid(z)
    y = (z * sg if c["act"] == "silu" else z).to(t)
    if not c["train"]:
        return {"y": y}
    dz = s["dy"].float()
    if c["act"] == "silu":
        dz = dz * sg * (1.0 + z * (1.0 - sg))
    gx = (dz * s["weight"]).unflatten(2, (c["groups"], -1))
    xg = xh.unflatten(2, (c["groups"], -1))
    m0 = gx.mean((1, 3), keepdim=True)
    m1 = (gx * xg).mean((1, 3), keepdim=True)
    dx = (rstd * (gx - m0 - xg * m1)).flatten(2).to(t)
    return {"y": y, "dx": dx, "dweight": (dz * xh).double().sum((0, 1)).float(),
            "dbias": dz.double().sum((0, 1)).float()}


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "norm":
        n = c["Bt"] * c["L"] * c["C"]
        return {"bytes": n * e * (4 if c["train"] else 2) + 4 * c["C"] * (4 if c["train"] else 2),
                "flops": n * (30 if c["train"] else 10)}
    H, G, N, P = c["H"], c["G"], c["N"], c["P"]
    rows = c["S"] if c["op"] == "step" else c["Bt"] * c["L"]
    seqs = c["S"] if c["op"] == "step" else c["Bt"]
    tokens = rows * ((H * P + 2 * G * N) * e + 8 * H)   # u, B, C, dt, beta
    state = 4 * seqs * H * N * P
    if c["op"] == "train":
        return {"bytes": 2 * tokens + 2 * rows * H * P * e + 3 * state, "flops": 18 * rows * H * N * P}
    has = 1 if c["op"] == "step" or c["h0"] else 0
    return {"bytes": tokens + rows * H * P * e + (1 + has) * state, "flops": 6 * rows * H * N * P}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "step":
        d = {m: s[m].double() for m in ("x", "dt", "h", "A_log", "B", "C", "beta")}
        S, y = _exact_token(d["h"], d["x"], d["B"], d["C"], d["dt"], d["beta"], d["A_log"], s["scale"])[:2]
        return {"y": y, "h": S}
    if case["op"] == "delta":
        return _exact_delta(s)
    c = case
    if 8 * c["Bt"] * c["L"] * c["H"] * c["N"] * c["P"] > 40e9:
        return None
    return _exact_train(s)


def _heads(x, H):
    return x.repeat_interleave(H // x.shape[1], 1)


def _exact_token(S, x, B, C, dt, beta, A_log, scale):
    """One token of every row: S [R,H,P,N]; x [R,H,P]; B, C [R,G,N]; dt, beta [R,H], all f64."""
    H = x.shape[1]
    k, q = _heads(B, H), _heads(C, H)
    Sd = torch.exp(-torch.exp(A_log) * dt)[..., None, None] * S
    e = x - torch.einsum("rhpn,rhn->rhp", Sd, k)
    S = Sd + torch.einsum("rhp,rhn->rhpn", beta[..., None] * e, k)
    return S, scale * torch.einsum("rhpn,rhn->rhp", S, q), Sd, e


def _exact_inputs(s):
    d = {m: s[m].double() for m in ("u", "dt", "A_log", "B", "C", "beta")}
    Bt, L, HP = d["u"].shape
    H, N = d["dt"].shape[2], d["B"].shape[3]
    d["u"] = d["u"].view(Bt, L, H, HP // H)
    h0 = s["h0"].double() if s["h0"] is not None else d["u"].new_zeros(Bt, H, HP // H, N)
    return d, h0, Bt, L, H, HP


def _exact_delta(s):
    d, S, Bt, L, H, HP = _exact_inputs(s)
    y = torch.empty_like(d["u"])
    for t in range(L):
        S, y[:, t] = _exact_token(S, d["u"][:, t], d["B"][:, t], d["C"][:, t], d["dt"][:, t], d["beta"][:, t],
                                  d["A_log"], s["scale"])[:2]
    return {"y": y.reshape(Bt, L, HP), "h": S}


def _exact_train(s):
    d, S, Bt, L, H, HP = _exact_inputs(s)
    G = d["B"].shape[2]
    y, starts, errs = torch.empty_like(d["u"]), [], torch.empty_like(d["u"])
    for t in range(L):
        starts.append(S)
        S, y[:, t], _, errs[:, t] = _exact_token(S, d["u"][:, t], d["B"][:, t], d["C"][:, t], d["dt"][:, t],
                                                 d["beta"][:, t], d["A_log"], s["scale"])
    dy = s["dy"].double().view_as(d["u"])
    dS = s["dh_last"].double()
    a = -torch.exp(d["A_log"])
    alpha = torch.exp(a * d["dt"])
    k, q = (_heads(d[m].transpose(0, 1).reshape(L * Bt, G, -1), H).view(L, Bt, H, -1) for m in ("B", "C"))
    du, dbeta, dlam = torch.empty_like(d["u"]), torch.empty_like(d["beta"]), torch.empty_like(d["beta"])
    dk, dq = torch.empty_like(k), torch.empty_like(q)
    for t in reversed(range(L)):
        b, e = d["beta"][:, t], errs[:, t]
        Sd = alpha[:, t, :, None, None] * starts[t]
        St = Sd + torch.einsum("rhp,rhn->rhpn", b[..., None] * e, k[t])
        dq[t] = s["scale"] * torch.einsum("rhpn,rhp->rhn", St, dy[:, t])
        dS = dS + s["scale"] * torch.einsum("rhp,rhn->rhpn", dy[:, t], q[t])
        dSk = torch.einsum("rhpn,rhn->rhp", dS, k[t])
        dbeta[:, t] = (dSk * e).sum(-1)
        de = b[..., None] * dSk
        du[:, t] = de
        dk[t] = b[..., None] * torch.einsum("rhpn,rhp->rhn", dS, e) - torch.einsum("rhpn,rhp->rhn", Sd, de)
        dS = dS - torch.einsum("rhp,rhn->rhpn", de, k[t])
        dlam[:, t] = (dS * Sd).sum((-1, -2))
        dS = alpha[:, t, :, None, None] * dS
    dB, dC = (x.view(L, Bt, G, H // G, -1).sum(3).transpose(0, 1) for x in (dk, dq))
    return {"y": y.reshape(Bt, L, HP), "du": du.reshape(Bt, L, HP), "dB": dB, "dC": dC, "ddt": dlam * a,
            "dbeta": dbeta, "dA_log": (dlam * a * d["dt"]).sum((0, 1)), "dh0": dS}


def _exact_norm(s):
    c = s["case"]
    Bt, L, C = s["x"].shape
    w, b = s["weight"].double(), s["bias"].double()
    x = s["x"].double().view(Bt, L, c["groups"], C // c["groups"])
    var, mean = torch.var_mean(x, (1, 3), correction=0, keepdim=True)
    r = 1.0 / torch.sqrt(var + 1e-5)
    n = ((x - mean) * r).view(Bt, L, C)
    z = n * w + b
    sg = 1.0 / (1.0 + torch.exp(-z))
    y = z * sg if c["act"] == "silu" else z
    if not c["train"]:
        return {"y": y}
    dz = s["dy"].double()
    if c["act"] == "silu":
        dz = dz * (sg + z * sg * (1.0 - sg))
    dn = (dz * w).view(Bt, L, c["groups"], -1)
    ng = n.view_as(dn)
    dx = r * (dn - dn.mean((1, 3), keepdim=True) - ng * (dn * ng).mean((1, 3), keepdim=True))
    return {"y": y, "dx": dx.view(Bt, L, C), "dweight": (dz * n).sum((0, 1)), "dbias": dz.sum((0, 1))}
