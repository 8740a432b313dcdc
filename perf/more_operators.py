"""The operators of a mixing block with memory, as measurable cases: the norms of queries and keys for each head with the
rotation by positions (several axes: frames, rows, columns), the gated delta rule along an axis of a channels-last tensor,
forward and backward, and its form for single tokens, each in two forms: elementary torch operations in 32 bits
(``own = False``) and the calls of ``pyramidconvblock_amd`` (``own = True``).

    listed()            the standing cases
    draw(rng)           one more case from the ranges that these stand for
    prepare(case, seed) inputs on the GPU
    run(state)          one pass: outputs and, in training, every gradient
    exact(case, seed)   the same from the definitions in 64 bits
    work(case)          bytes and operations that a pass cannot do without

The formulas:

    rotary  of a head's row x of d channels: n = x ("none"), x / sqrt(mean x^2 + eps) * weight ("rms") or x / sqrt(sum x^2 + eps) * weight
            ("l2"); the first 2 P channels of n are P pairs, halves (i, P + i) or neighbours (2 i, 2 i + 1), and pair i is turned by the angle
            position * frequency_i, the position along the axis that the pair belongs to
    delta   for every value head, with a state S of dk x dv: a_t = sigmoid(g_t), beta_t = sigmoid(b_t),
            u_t = beta_t (v_t - a_t S_(t-1)^T k_t),   S_t = a_t S_(t-1) + k_t u_t^T,   y_t = dk^-1/2 S_t^T q_t

A case is a dict of plain values:

    op      "rotary", "delta" or "step" (the delta rule for a single token)
    mode    "train": forward and backward, "infer": forward under no_grad
    dtype   "bf16", "fp16" or "fp32" (states are always 32-bit)
    B, F, H, W   batch, frames, rows, columns: the tokens (a step has B tokens)
    hq, hk  rotary: heads of q and k;  delta: heads of q and k, which hv value heads share in groups
    dk, dv  channels of a head of q and k, and of v
    kind    rotary: "none", "rms" or "l2" (no weight in the last case); axes: of positions, 1 to 3; part: pairs that are turned, of dk // 2;
            neighbours: which channels pair; given: positions come as a tensor (1 axis, far from 0), not from the grid
    axis    delta: "seq" (all tokens of an image as one sequence), "h" or "w"; reverse: from the end;
            lengths: a number of valid steps for each sequence; state: an initial state is given
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
BASE = 1e4


def _rotary_case(name, mode, dtype, tokens, hq, hk, d, kind, axes, part=None, neighbours=False, given=False):
    B, F, H, W = tokens
    return {"name": name, "op": "rotary", "mode": mode, "dtype": dtype, "B": B, "F": F, "H": H, "W": W, "hq": hq, "hk": hk, "dk": d,
            "kind": kind, "axes": axes, "part": d // 2 if part is None else part, "neighbours": neighbours, "given": given}


def _delta_case(name, mode, dtype, tokens, hk, hv, dk, dv, axis="seq", reverse=False, lengths=False, state=False):
    B, H, W = tokens
    return {"name": name, "op": "delta", "mode": mode, "dtype": dtype, "B": B, "H": H, "W": W, "hk": hk, "hv": hv, "dk": dk, "dv": dv,
            "axis": axis, "reverse": reverse, "lengths": lengths, "state": state}


def _step_case(name, dtype, B, hk, hv, dk, dv):
    return {"name": name, "op": "step", "mode": "infer", "dtype": dtype, "B": B, "hk": hk, "hv": hv, "dk": dk, "dv": dv}


def listed():
    return [
        # queries and keys of one image, unit rows for the delta rule: serving latency
        _rotary_case("rotary_infer_one_bf16", "infer", "bf16", (1, 1, 56, 56), 4, 4, 32, "l2", 2),
        # video clips: positions of three axes, fewer key heads than query heads, weights that learn
        _rotary_case("rotary_train_video_bf16", "train", "bf16", (4, 16, 28, 28), 8, 4, 64, "rms", 3),
        # odd extents and heads in full precision, neighbours as pairs
        _rotary_case("rotary_train_odd_fp32", "train", "fp32", (3, 1, 57, 61), 5, 5, 40, "rms", 2, neighbours=True),
        # long texts beside images: positions as a tensor, far from 0, a part of each head turned
        _rotary_case("rotary_train_given_fp16", "train", "fp16", (4, 1, 1, 4096), 9, 9, 128, "none", 1, part=32, given=True),
        # one token of one stream: latency
        _step_case("step_one_fp16", "fp16", 1, 8, 16, 64, 64),
        # one token for each of many streams, 1152 channels: the states' way through memory
        _step_case("step_bf16", "bf16", 256, 9, 9, 128, 128),
        # a few tokens for each stream, as after a prompt's end or for drafts that are checked
        _delta_case("delta_infer_few_bf16", "infer", "bf16", (64, 1, 4), 8, 8, 64, 64, state=True),
        # one image as a sequence: few chains, a long way
        _delta_case("delta_infer_one_bf16", "infer", "bf16", (1, 56, 56), 4, 4, 32, 32),
        # a training batch of images
        _delta_case("delta_train_bf16", "train", "bf16", (32, 56, 56), 4, 4, 32, 32),
        # columns of odd images, upwards, each image with a height of its own
        _delta_case("delta_train_ragged_fp32", "train", "fp32", (3, 57, 61), 5, 5, 24, 40, "h", True, lengths=True, state=True),
        # wide heads, two value heads for a key head
        _delta_case("delta_train_shared_bf16", "train", "bf16", (2, 64, 64), 4, 8, 128, 128),
        # high-resolution images as sequences of 16 384 steps
        _delta_case("delta_train_long_fp16", "train", "fp16", (2, 128, 128), 6, 6, 64, 64, state=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "step", "delta", "delta", "delta"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    mode = "infer" if rng.random() < 0.3 else "train"
    wide = lambda hi: rng.choice([16, 24, 32, 40, 48, 64, 80, 96, 128, _log_int(rng, 16, hi)])
    if op == "step":
        hk, group = rng.randint(1, 9), rng.choice([1, 1, 2, 3])
        case = _step_case("", dtype, _log_int(rng, 1, 512), hk, hk * group, wide(128), wide(128))
    elif op == "rotary":
        axes = rng.choice([1, 2, 2, 3])
        d, hk = wide(128), rng.randint(1, 9)
        hq = hk * rng.choice([1, 1, 2])
        F = _log_int(rng, 2, 16) if axes == 3 else 1
        H = 1 if axes == 1 else _log_int(rng, 5, 80)
        W = _log_int(rng, 64, 4096) if axes == 1 else min(80, max(5, H + rng.choice([0, 0, 1, -1, 4, -3])))
        pairs = d // 2
        case = _rotary_case("", mode, dtype, (_log_int(rng, 1, 32), F, H, W), hq, hk, d, rng.choice(["none", "rms", "l2"]), axes,
                            rng.choice([pairs, pairs, max(axes, pairs // 2)]), rng.random() < 0.3, axes == 1 and rng.random() < 0.5)
    else:
        hk, group = rng.randint(1, 8), rng.choice([1, 1, 1, 2, 3])
        dk = wide(128)
        dv = rng.choice([dk, dk, dk, wide(128)])
        H = _log_int(rng, 5, 128)
        W = min(128, max(5, H + rng.choice([0, 0, 1, -1, 4, -3])))
        if rng.random() < 0.15:
            H, W = 1, _log_int(rng, 1, 64)
        case = _delta_case("", mode, dtype, (_log_int(rng, 1, 32), H, W), hk, hk * group, dk, dv, rng.choice(["seq", "seq", "h", "w"]), rng.random() < 0.4,
                           rng.random() < 0.3, rng.random() < 0.5)
    # no more than the largest listed cases
    def most(case):
        w = work(case)
        return w["bytes"] > 2e8 or w["flops"] > 2e10

    while most(case) and case["B"] > 1:
        case["B"] //= 2
    while most(case) and op != "step":
        side = "H" if case["H"] >= case["W"] else "W"
        case[side] = (case[side] + 1) // 2
    del case["name"]
    return case


def _sections(case):
    """Pairs of each axis: equal parts, the first ones one larger where they do not come out even."""
    axes, part = case["axes"], case["part"]
    return tuple(part // axes + (i < part % axes) for i in range(axes))


def _delta_extents(case):
    """Sizes in front of the heads, and the recurrence's place among them."""
    B, H, W = case["B"], case["H"], case["W"]
    if case["axis"] == "seq":
        return (B, H * W), 1
    return (B, H, W), 1 if case["axis"] == "h" else 2


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, mean=0.0, std=1.0, dt=dtype):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dt)

    def unit(*shape):
        """Rows of length 1, as the norm before the rule makes them."""
        t = torch.randn(shape, generator=gen, device="cuda")
        return (t / t.square().sum(-1, keepdim=True).sqrt()).to(dtype)

    train = case["mode"] == "train"
    s = {"case": case, "train": train}
    if case["op"] == "rotary":
        lead = (case["B"],) + tuple(case[n] for n in ("F", "H", "W"))[3 - case["axes"]:]
        d = case["dk"]
        s["q"], s["k"] = rand(*lead, case["hq"], d, std=1.5), rand(*lead, case["hk"], d, std=1.5)
        s["weight"] = s["key_weight"] = s["positions"] = None
        if case["kind"] == "rms":
            s["weight"], s["key_weight"] = rand(d, mean=1.0, std=0.2), rand(d, mean=1.0, std=0.2)
        if case["given"]:
            # each sequence somewhere in a long text
            start = torch.randint(0, 1 << 20, (case["B"], 1), generator=gen, device="cuda")
            s["positions"] = (start + torch.arange(case["W"], device="cuda")).to(torch.int32).unsqueeze(-1)
        if train:
            s["gq"], s["gk"] = rand(*lead, case["hq"], d), rand(*lead, case["hk"], d)
        return s
    hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
    if case["op"] == "step":
        lead, carried = (case["B"],), (case["B"], hv, dk, dv)
    else:
        lead, dim = _delta_extents(case)
        carried = lead[:dim] + lead[dim + 1:] + (hv, dk, dv)
        s["dim"] = dim
    s["q"], s["k"], s["v"] = unit(*lead, hk, dk), unit(*lead, hk, dk), rand(*lead, hv, dv)
    # logits of a trained layer: memories of a few to a few hundred steps, writes of every strength
    s["g"], s["b"] = rand(*lead, hv, mean=3.0, std=1.5), rand(*lead, hv, std=1.5)
    if case["op"] == "step":
        s["state"], s["new_state"] = rand(*carried, std=0.3, dt=torch.float32), torch.empty(carried, device="cuda")
        return s
    s["state"] = rand(*carried, std=0.3, dt=torch.float32) if case["state"] else None
    T = lead[dim]
    s["lengths"] = (torch.randint(T // 2, T + 1, lead[:dim], generator=gen, device="cuda", dtype=torch.int32)
                    if case["lengths"] else None)
    if train:
        s["gy"], s["glast"] = rand(*lead, hv, dv), rand(*carried, std=0.1, dt=torch.float32)
    return s


# ----------------------------------------------------------------------------------------------------------------------
# The framework's calls

def _own(s):
    import pyramidconvblock_amd as pcb

    case = s["case"]
    if case["op"] == "step":
        return list(pcb.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["b"], s["state"], new_state=s["new_state"]))
    names = ("q", "k", "weight", "key_weight") if case["op"] == "rotary" else ("q", "k", "v", "g", "b", "state")
    leaves = [s[n] for n in names if s[n] is not None]
    for t in leaves:
        t.requires_grad_(s["train"])
    with torch.set_grad_enabled(s["train"]):
        if case["op"] == "rotary":
            outs = pcb.head_rotary(s["q"], s["k"], s["weight"], s["key_weight"], positions=s["positions"], axes=case["axes"],
                                   sections=_sections(case), base=BASE, kind=case["kind"], neighbours=case["neighbours"], eps=EPS)
            grads = ("gq", "gk")
        else:
            outs = pcb.gated_delta(s["q"], s["k"], s["v"], s["g"], s["b"], state=s["state"], lengths=s["lengths"], dim=s["dim"],
                                   reverse=case["reverse"])
            grads = ("gy", "glast")
    if not s["train"]:
        return list(outs)
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, [s[n] for n in grads]))


# ----------------------------------------------------------------------------------------------------------------------
# The plain form: elementary operations in 32 bits, gradients by their formulas

def _angles(case, s):
    """-> cos and sin [tokens' axes or 1, ..., pairs], angles in 64 bits."""
    lead = s["q"].shape[:-2]
    dev = s["q"].device
    parts = []
    for a, n in enumerate(_sections(case)):
        f = BASE ** (-torch.arange(n, device=dev, dtype=torch.float64) / max(n, 1))
        if s["positions"] is not None:
            p = s["positions"][..., a].double()
        else:
            grid = lead[len(lead) - case["axes"]:]
            shape = [1] * len(grid)
            shape[a] = grid[a]
            p = torch.arange(grid[a], device=dev, dtype=torch.float64).reshape(shape).expand(grid)
        parts.append(p.unsqueeze(-1) * f)
    t = torch.cat(parts, -1).unsqueeze(-2)
    return torch.cos(t), torch.sin(t)


def _turn(case, x, cos, sin):
    P = case["part"]
    if case["neighbours"]:
        a, b = x[..., 0:2 * P:2], x[..., 1:2 * P:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :P], x[..., P:2 * P]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * P:]], -1)


def _plain_rotary(s):
    case = s["case"]
    kind = case["kind"]
    cos, sin = (t.float() for t in _angles(case, s))
    outs, grads, wgrads = [], [], []
    for x, w, gy in ((s["q"], s["weight"], "gq"), (s["k"], s["key_weight"], "gk")):
        dt, x = x.dtype, x.detach().float()
        w = None if w is None else w.detach().float()
        r, n = None, x
        if kind != "none":
            m = x.square().sum(-1, keepdim=True) / (x.shape[-1] if kind == "rms" else 1)
            r = torch.rsqrt(m + EPS)
            n = x * r
        outs.append(_turn(case, n if w is None else n * w, cos, sin).to(dt))
        if s["train"]:
            g = _turn(case, s[gy].float(), cos, -sin)
            if w is not None:
                wgrads.append((g * n).sum(tuple(range(g.dim() - 1))).to(dt))
                g = g * w
            if r is not None:
                g = (g - n * ((g * n).sum(-1, keepdim=True) / (x.shape[-1] if kind == "rms" else 1))) * r
            grads.append(g.to(dt))
    return outs + grads + wgrads


def _chains(case, s, t, fill=0.0):
    """[lead.., heads(, d)] -> [chains, T, ...] in 32 bits in the order of the recurrence, `fill` behind a length."""
    dim = s["dim"]
    t = t.detach().float().movedim(dim, -2 if t is s["g"] or t is s["b"] else -3)
    tail = 1 if t.dim() == s["g"].dim() else 2
    heads = t.dim() - tail
    t = t.movedim(heads, heads - 1)                    # [.., heads, T, ...]
    if t.shape[heads - 1] != case["hv"]:
        t = t.repeat_interleave(case["hv"] // t.shape[heads - 1], heads - 1)
    t = t.reshape((-1,) + t.shape[heads:])
    on = s["_on"]
    if on is not None:
        t = torch.where(on if t.dim() == 2 else on.unsqueeze(-1), t, fill)
    return t.flip(1) if case["reverse"] else t


def _valid(case, s):
    """[chains, T], or None."""
    if s["lengths"] is None:
        return None
    lead, dim = _delta_extents(case)
    T = lead[dim]
    n = s["lengths"].reshape(lead[:dim] + (1,) * (len(lead) - dim - 1 + 1)).expand(lead[:dim] + lead[dim + 1:] + (case["hv"],))
    return torch.arange(T, device=n.device) < n.reshape(-1, 1)


def _unchains(case, s, t, heads, dtype):
    """Gradients or outputs [chains, T, ...] back to [lead.., heads(, d)]; shared heads' parts are added."""
    lead, dim = _delta_extents(case)
    on = s["_on"]
    t = t.flip(1) if case["reverse"] else t
    if on is not None:
        t = torch.where(on if t.dim() == 2 else on.unsqueeze(-1), t, 0.0)
    rest = lead[:dim] + lead[dim + 1:]
    t = t.reshape(rest + (case["hv"],) + t.shape[1:])
    if heads != case["hv"]:
        t = t.unflatten(len(rest), (heads, case["hv"] // heads)).sum(len(rest) + 1)
    return t.movedim(len(rest) + 1, dim).to(dtype)


def _solve(A, X):
    """(I + A)^-1 X for strictly lower A: row by row."""
    X = X.clone()
    for i in range(1, A.shape[1]):
        X[:, i] -= (A[:, i, :i, None] * X[:, :i]).sum(1)
    return X


def _plain_delta(s):
    case = s["case"]
    hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
    dtype = DTYPES[case["dtype"]]
    s = dict(s)
    s["_on"] = _valid(case, s)
    L = 64
    q, k, v, g, b = (_chains(case, s, s[n]) for n in ("q", "k", "v", "g", "b"))
    N, T = g.shape
    on = s["_on"]
    if on is not None and case["reverse"]:
        on = on.flip(1)
    # log sigmoid, 0 for steps that are not there
    la = torch.clamp(g, max=0) - torch.log1p(torch.exp(-g.abs()))
    beta = 1 / (1 + torch.exp(-b))
    if on is not None:
        la, beta = torch.where(on, la, 0.0), torch.where(on, beta, 0.0)
    M = (T + L - 1) // L
    pad = M * L - T

    def cut(t):
        t = torch.cat([t, t.new_zeros((N, pad) + t.shape[2:])], 1)
        return t.reshape((N * M, L) + t.shape[2:]).contiguous()

    sc = dk ** -0.5
    q, k, v, la_, be = cut(q) * sc, cut(k), cut(v), cut(la), cut(beta)
    c = torch.cumsum(la_.double(), 1)
    lower = torch.ones(L, L, device=g.device, dtype=torch.bool).tril()
    gam = torch.where(lower, torch.exp(torch.where(lower, c[:, :, None] - c[:, None, :], 0.0)).float(), 0.0)
    D, E, eL = torch.exp(c).float()[..., None], torch.exp(c[:, -1:] - c).float()[..., None], torch.exp(c[:, -1]).float()
    tr = lambda t: t.transpose(1, 2).contiguous()
    kk = torch.matmul(k, tr(k))
    A = (be[..., None] * gam * kk).tril(-1)
    P = gam * torch.matmul(q, tr(k))
    X = _solve(A, torch.cat([be[..., None] * D * k, be[..., None] * v], -1))
    Wm, Uv = X[..., :dk].contiguous(), X[..., dk:].contiguous()
    del X
    S = s["state"].detach().float().reshape(N, dk, dv).clone() if s["state"] is not None else torch.zeros(N, dk, dv, device=g.device)
    S0, U = torch.empty(N * M, dk, dv, device=g.device), torch.empty(N * M, L, dv, device=g.device)
    Kt, of = tr(k), lambda t, m: t.view((N, M) + t.shape[1:])[:, m].contiguous()
    for m in range(M):
        S0.view(N, M, dk, dv)[:, m] = S
        u = of(Uv, m) - torch.matmul(of(Wm, m), S)
        U.view(N, M, L, dv)[:, m] = u
        S = of(eL, m)[:, None, None] * S + torch.matmul(of(Kt, m), of(E, m) * u)
    Y = D * torch.matmul(q, S0) + torch.matmul(P, U)
    flat = lambda t: t.reshape((N, M * L) + t.shape[2:])[:, :T]
    lead, dim = _delta_extents(case)
    carried = lead[:dim] + lead[dim + 1:] + (hv, dk, dv)
    outs = [_unchains(case, s, flat(Y), hv, dtype), S.reshape(carried)]
    if not s["train"]:
        return outs

    gy = cut(_chains(case, s, s["gy"]))
    dS = s["glast"].detach().float().reshape(N, dk, dv).clone()
    dS1 = torch.empty_like(S0)
    dU = torch.matmul(tr(P), gy)
    C0 = torch.matmul(tr(q), D * gy)
    Wt = tr(Wm)
    for m in range(M - 1, -1, -1):
        dS1.view(N, M, dk, dv)[:, m] = dS
        du = of(dU, m) + of(E, m) * torch.matmul(of(k, m), dS)
        dU.view(N, M, L, dv)[:, m] = du
        dS = of(eL, m)[:, None, None] * dS + of(C0, m) - torch.matmul(of(Wt, m), du)
    del C0, Wt
    # the substitution with the transposed matrix, from the end
    Z = _solve(tr(A).flip(1).flip(2), dU.flip(1)).flip(1)
    dP, dA = torch.matmul(gy, tr(U)).tril(), -torch.matmul(Z, tr(U)).tril(-1)
    gq, gz, gu = torch.matmul(gy, tr(S0)), torch.matmul(Z, tr(S0)), torch.matmul(U, tr(dS1))
    Pg, Ag = gam * dP, be[..., None] * gam * dA
    dq = sc * (D * gq + torch.matmul(Pg, k))
    dk_ = torch.matmul(tr(Pg), q) - D * be[..., None] * gz + E * gu + torch.matmul(Ag + tr(Ag), k)
    dvv = be[..., None] * Z
    kgz, kgu = (k * gz).sum(-1), (k * gu).sum(-1) * E[..., 0]
    dbeta = (Z * v).sum(-1) - D[..., 0] * kgz + (dA * gam * kk).sum(-1)
    n = dP * P + dA * A
    dc = n.sum(-1) - n.sum(-2) + D[..., 0] * ((q * gq).sum(-1) - be * kgz) - kgu
    dc[:, -1] += kgu.sum(-1) + eL * (S0 * dS1).sum((1, 2))
    dla = dc.double().flip(1).cumsum(1).flip(1).float()
    dg = flat(dla) / (1 + torch.exp(g))
    db = flat(dbeta) * beta * (1 - beta)
    outs += [_unchains(case, s, flat(t), h, dtype) for t, h in ((dq, hk), (dk_, hk), (dvv, hv))]
    outs += [_unchains(case, s, t, hv, dtype) for t in (dg, db)]
    return outs + ([dS.reshape(carried)] if s["state"] is not None else [])


def _plain_step(s):
    case = s["case"]
    group = case["hv"] // case["hk"]
    q, k = (t.float().repeat_interleave(group, 1) for t in (s["q"], s["k"]))
    a, beta = 1 / (1 + torch.exp(-s["g"].float())), 1 / (1 + torch.exp(-s["b"].float()))
    S = a[..., None, None] * s["state"]
    u = beta[..., None] * (s["v"].float() - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    return [((S * q[..., None]).sum(-2) * case["dk"] ** -0.5).to(s["v"].dtype), S]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "delta": _plain_delta, "step": _plain_step}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits: the rule token by token, its gradients backwards through the same steps; the norm and the
# rotation as a product of complex numbers, differentiated

def _exact_rotary(s):
    case = s["case"]
    P, lead = case["part"], s["q"].shape[:-2]
    dev = s["q"].device
    angle = torch.zeros(lead + (1, P), dtype=torch.float64, device=dev)
    first = 0
    for a, n in enumerate(_sections(case)):
        if s["positions"] is not None:
            p = s["positions"][..., a].double()
        else:
            d = len(lead) - case["axes"] + a
            p = torch.arange(lead[d], dtype=torch.float64, device=dev).reshape([-1 if i == d else 1 for i in range(len(lead))])
        for j in range(n):
            angle[..., 0, first + j] = p * math.pow(BASE, -j / n)
        first += n
    unit = torch.polar(torch.ones_like(angle), angle)
    outs, leaves, weights, grads = [], [], [], []
    for n, w, g in (("q", "weight", "gq"), ("k", "key_weight", "gk")):
        x = s[n].detach().double().requires_grad_(s["train"])
        leaves.append(x)
        y = x
        if case["kind"] == "rms":
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
        elif case["kind"] == "l2":
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) + EPS)
        if s[w] is not None:
            weights.append(s[w].detach().double().requires_grad_(s["train"]))
            y = y * weights[-1]
        if case["neighbours"]:
            z = torch.complex(y[..., :2 * P:2], y[..., 1:2 * P:2]) * unit
            z = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(y[..., :P], y[..., P:2 * P]) * unit
            z = torch.cat([z.real, z.imag], -1)
        outs.append(torch.cat([z, y[..., 2 * P:]], -1))
        if s["train"]:
            grads.append(s[g].double())
    if not s["train"]:
        return outs
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves + weights, grads))


def _exact_delta(s):
    case = s["case"]
    hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
    lead, dim = _delta_extents(case)
    T = lead[dim]
    if T > 20000:
        return None
    rest = lead[:dim] + lead[dim + 1:]
    N = math.prod(rest) * hv
    order = range(T - 1, -1, -1) if case["reverse"] else range(T)

    def steps(t, heads):                       # [T, chains(, d)]
        t = t.detach().double().movedim(dim, 0)
        if heads != hv:
            t = t.repeat_interleave(hv // heads, len(rest) + 1)
        return t.reshape((T, N) + t.shape[len(rest) + 2:]).contiguous()

    q, k, v, g, b = steps(s["q"], hk), steps(s["k"], hk), steps(s["v"], hv), steps(s["g"], hv), steps(s["b"], hv)
    a, beta = torch.sigmoid(g), torch.sigmoid(b)
    on = None
    if s["lengths"] is not None:
        n = s["lengths"].reshape(lead[:dim] + (1,) * (len(rest) - dim + 1)).expand(rest + (hv,)).reshape(N)
        on = torch.arange(T, device=n.device).unsqueeze(1) < n
        a, beta = torch.where(on, a, 1.0), torch.where(on, beta, 0.0)
    sc = dk ** -0.5
    S = torch.zeros(N, dk, dv, dtype=torch.float64, device=g.device) if s["state"] is None else s["state"].detach().double().reshape(N, dk, dv)
    y, train = torch.zeros_like(v), s["train"]

    def step(t, S):
        """-> the decayed state, what is missing of v, the new state."""
        Sd = a[t][:, None, None] * S
        r = v[t] - torch.einsum("nij,ni->nj", Sd, k[t])
        return Sd, r, Sd + k[t][:, :, None] * (beta[t][:, None] * r)[:, None, :]

    run = max(1, int(T ** 0.5))                # states are kept at every run's start and made again inside
    order = list(order)
    kept = []
    for i, t in enumerate(order):
        if train and i % run == 0:
            kept.append(S)
        S = step(t, S)[2]
        y[t] = sc * (S * q[t][:, :, None]).sum(1)

    def back(t, heads):
        if on is not None:
            t = torch.where(on if t.dim() == 2 else on.unsqueeze(-1), t, 0.0)
        t = t.reshape((T,) + rest + (hv,) + t.shape[2:])
        if heads != hv:
            t = t.unflatten(len(rest) + 1, (heads, hv // heads)).sum(len(rest) + 2)
        return t.movedim(0, dim)

    carried = rest + (hv, dk, dv)
    outs = [back(y, hv), S.reshape(carried)]
    if not train:
        return outs
    gy = steps(s["gy"], hv)
    if on is not None:
        gy = torch.where(on.unsqueeze(-1), gy, 0.0)
    dS = s["glast"].double().reshape(N, dk, dv)
    dq, dk_, dv_, da, db = (torch.zeros_like(t) for t in (q, k, v, a, beta))
    for i0 in range((T - 1) // run * run, -1, -run):
        S, made = kept[i0 // run], []
        for t in order[i0:i0 + run]:
            Sd, r, new = step(t, S)
            made.append((t, S, Sd, r, new))
            S = new
        for t, before, Sd, r, new in reversed(made):
            dq[t] = sc * (new * gy[t][:, None, :]).sum(2)
            dS = dS + sc * q[t][:, :, None] * gy[t][:, None, :]
            du = (dS * k[t][:, :, None]).sum(1)
            u, db[t], dv_[t] = beta[t][:, None] * r, (du * r).sum(1), beta[t][:, None] * du
            dk_[t] = (dS * u[:, None, :]).sum(2) - (Sd * dv_[t][:, None, :]).sum(2)
            dS = dS - k[t][:, :, None] * dv_[t][:, None, :]
            da[t] = (dS * before).sum((1, 2))
            dS = a[t][:, None, None] * dS
    dg, db = da * a * torch.sigmoid(-g), db * beta * torch.sigmoid(-b)
    outs += [back(dq, hk), back(dk_, hk), back(dv_, hv), back(dg, hv), back(db, hv)]
    return outs + ([dS.reshape(carried)] if s["state"] is not None else [])


def _exact_step(s):
    group = s["case"]["hv"] // s["case"]["hk"]
    d = lambda t: t.double()
    q, k = (d(t).repeat_interleave(group, 1) for t in (s["q"], s["k"]))
    a, beta = torch.sigmoid(d(s["g"])), torch.sigmoid(d(s["b"]))
    S = d(s["state"])
    kS = torch.matmul(k.unsqueeze(-2), S).squeeze(-2)
    qS = torch.matmul(q.unsqueeze(-2), S).squeeze(-2)
    u = beta[..., None] * (d(s["v"]) - a[..., None] * kS)
    y = a[..., None] * qS + (q * k).sum(-1, keepdim=True) * u
    return [y * s["case"]["dk"] ** -0.5, a[..., None, None] * S + k.unsqueeze(-1) * u.unsqueeze(-2)]


def exact(case, seed):
    return {"rotary": _exact_rotary, "delta": _exact_delta, "step": _exact_step}[case["op"]](prepare(case, seed))


def work(case):
    """Every input read once and every output written once; operations of the rule token by token, an exponential as one."""
    es = 4 if case["dtype"] == "fp32" else 2
    op, train = case["op"], case["mode"] == "train"
    if op == "rotary":
        tokens = case["B"] * case["F"] * case["H"] * case["W"]
        n = tokens * (case["hq"] + case["hk"]) * case["dk"]
        weights = 2 * case["dk"] * es * (2 if train else 1) if case["kind"] == "rms" else 0
        return {"bytes": float(n) * es * (4 if train else 2) + weights + (4.0 * tokens if case["given"] else 0),
                "flops": float(n) * (22 if train else 8)}
    hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
    tokens = case["B"] * (1 if op == "step" else case["H"] * case["W"])
    row = 2 * hk * dk + hv * dv + 2 * hv
    if op == "step":
        return {"bytes": float(tokens) * ((row + hv * dv) * es + 8.0 * hv * dk * dv), "flops": 7.0 * tokens * hv * dk * dv}
    lead, dim = _delta_extents(case)
    chains = case["B"] * (1 if len(lead) == 2 else lead[3 - dim]) * hv
    states = 4.0 * chains * dk * dv * ((1 + case["state"]) * (2 if train else 1))
    elements = row + hv * dv + ((row + hv * dv) if train else 0)       # inputs and y; gradients and gy
    return {"bytes": float(tokens) * elements * es + states, "flops": (25.0 if train else 7.0) * tokens * hv * dk * dv}
