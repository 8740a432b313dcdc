"""gated_delta and gated_delta_step against the recurrence in 64 bits, one step after another.

Bounds.  A result is rounded once to its type: half a step.  What lies between is rounded on the way: in calls of 16-bit tensors states and the u of
each step are kept in two bfloat16 (2^-17 relative), and so are the factors of products made of them; where the result is a state, in
three, like everything of 32-bit tensors (2^-25), and their products are summed in 32 bits over up to 128 terms (128 2^-24 at worst, some 8 2^-24 in
fact).  So the reference is run again with its states, u, decays and strengths and all their gradients off by E = 2^-16 (results in
32 bits: 2^-21) of themselves at every step, signs at random, and a result may be off by 16 times the most that any element of it moved in three
such runs, and E of its largest element."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ["q", "k", "v", "g", "b"]


def pcb():
    import pyramidconvblock_amd

    return pyramidconvblock_amd


class Off(torch.autograd.Function):
    """x and its gradient, each off by up to e of itself."""

    @staticmethod
    def forward(ctx, x, e, gen):
        ctx.e, ctx.gen = e, gen
        return x * (1 + e * signs(x, gen))

    @staticmethod
    def backward(ctx, g):
        return g * (1 + ctx.e * signs(g, ctx.gen)), None, None


def signs(x, gen):
    return torch.randint(0, 2, x.shape, generator=gen).to(x.dtype) * 2 - 1


def rule64(q, k, v, g, b, state, lengths, dim, reverse, scale, logits, off=0.0, gen=None):
    """The recurrence; every tensor in 64 bits -> (y, last)."""
    o = (lambda t: Off.apply(t, off, gen)) if off else lambda t: t
    dim %= q.dim()
    O, T, W = math.prod(q.shape[:dim]), q.shape[dim], math.prod(q.shape[dim + 1:-2])
    place = lambda t, tail: t.reshape(O, T, W, *t.shape[t.dim() - tail:])
    group = v.shape[-2] // q.shape[-2]
    q, k = (place(t.repeat_interleave(group, -2), 2) for t in (q, k))
    v, g, b = place(v, 2), place(g, 1), place(b, 1)
    hv, dk, dv = v.shape[3], q.shape[-1], v.shape[-1]
    a = o(torch.sigmoid(g) if logits else torch.exp(g))
    beta = o(torch.sigmoid(b) if logits else b)
    ys, lasts = [], []
    state = torch.zeros(O, W, hv, dk, dv, dtype=torch.float64) if state is None else state.reshape(O, W, hv, dk, dv)
    for i in range(O):
        n = T if lengths is None else max(0, min(T, int(lengths.reshape(-1)[i])))
        S, rows = state[i], [torch.zeros(W, hv, dv, dtype=torch.float64)] * T
        for t in range(n - 1, -1, -1) if reverse else range(n):
            S = S * a[i, t][..., None, None]
            u = o(beta[i, t][..., None] * (v[i, t] - (k[i, t][..., None, :] @ S)[..., 0, :]))
            S = o(S + k[i, t][..., None] * u[..., None, :])
            rows[t] = scale * (q[i, t][..., None, :] @ S)[..., 0, :]
        ys.append(torch.stack(rows) if T else torch.zeros(0, W, hv, dv, dtype=torch.float64))
        lasts.append(S)
    return ys, lasts


def recurrence(s, train, off=0.0, seed=0):
    """-> {name: 64 bits} for a case's data"""
    gen = torch.Generator().manual_seed(seed)
    leaves = {n: s[n].double().requires_grad_(train) for n in NAMES + ["state"] if s[n] is not None}
    behind = s["behind"]   # (places that hold NaN where a sequence has ended: nothing may come of them)
    args = {n: leaves[n] if n == "state" else torch.where(behind[(...,) + (None,) * (leaves[n].dim() - behind.dim())], 0.0, leaves[n]) for n in leaves}
    ys, lasts = rule64(*(args.get(n) for n in NAMES + ["state"]), s["lengths"], s["dim"], s["reverse"], s["scale"], s["logits"], off, gen)
    y = torch.stack(ys).reshape(s["v"].shape) if ys else torch.zeros(s["v"].shape, dtype=torch.float64)
    last = torch.stack(lasts).reshape(s["glast"].shape) if lasts else torch.zeros(s["glast"].shape, dtype=torch.float64)
    out = {"y": y.detach(), "last": last.detach()}
    if train:
        gy = torch.where(behind[(...,) + (None,) * (y.dim() - behind.dim())], 0.0, s["gy"].double())
        loss = (y * gy).sum() + ((last * s["glast"].double()).sum() if s["use_last"] else 0.0)
        grads = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True) if loss.requires_grad else [None] * len(leaves)
        out |= {"g" + n: torch.zeros_like(leaves[n]) if t is None else t for n, t in zip(leaves, grads)}
    return out


def bounds(s, train):
    """-> {name: (value, bound)}"""
    ref = recurrence(s, train)
    # (roundings of 32-bit numbers, and of what 16-bit tensors keep)
    wide = {k: t for k, t in ref.items() if k in ("last", "gstate") or s["q"].dtype == torch.float32}
    out = {}
    for off, names in ((2.0 ** -21, set(wide)), (2.0 ** -16, set(ref) - set(wide))):
        if not names:
            continue
        moved = {k: 0.0 for k in names}
        for seed in range(3):
            r = recurrence(s, train, off, seed + 1)
            for k in names:
                if ref[k].numel():
                    moved[k] = max(moved[k], float((r[k] - ref[k]).abs().max()))
        for k in names:
            out[k] = ref[k], 16 * moved[k] + off * (float(ref[k].abs().max()) if ref[k].numel() else 0.0)
    return out


def check(got, ref, bound, name):
    got = got.detach()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    info = torch.finfo(got.dtype)
    off = (got.double().cpu() - ref).abs() - (info.eps / 2 * (ref.abs() + bound) + bound + info.smallest_normal * info.eps)
    assert not torch.isnan(off).any(), name
    assert off.numel() == 0 or float(off.max()) <= 0, (name, float(off.max()), bound)


def data(lead, hk, hv, dk, dv, dtype, dim=-3, reverse=False, lengths=None, state=False, gates=None, logits=True, scale=None, use_last=True, seed=0,
         nan=True):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=gen)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True).clamp_min(1e-3)
    gates = dtype if gates is None else gates
    dim = len(lead) + 2 + dim if dim < 0 else dim
    s = dict(q=unit(rnd(*lead, hk, dk)).to(dtype), k=(0.99 * unit(rnd(*lead, hk, dk))).to(dtype), v=rnd(*lead, hv, dv).to(dtype))
    g, b = rnd(*lead, hv) * 2 + 2, rnd(*lead, hv)
    s["g"], s["b"] = (g.to(gates), b.to(gates)) if logits else ((-torch.nn.functional.softplus(-g)).to(gates), torch.sigmoid(b).to(gates))
    rest = [n for i, n in enumerate(lead) if i != dim]
    s["state"] = rnd(*rest, hv, dk, dv) if state else None
    s["gy"], s["glast"] = rnd(*lead, hv, dv).to(dtype), rnd(*rest, hv, dk, dv)
    s["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32).reshape(lead[:dim])
    behind = torch.zeros(*lead, dtype=torch.bool)
    if lengths is not None:
        at = torch.arange(lead[dim]).reshape([-1 if i == dim else 1 for i in range(len(lead))])
        behind = (at >= s["lengths"].reshape([lead[i] if i < dim else 1 for i in range(len(lead))])).expand(*lead)
        if nan:
            for n in NAMES + ["gy"]:
                s[n][behind] = float("nan")
    s.update(behind=behind, dim=dim, reverse=reverse, scale=dk ** -0.5 if scale is None else scale, logits=logits, use_last=use_last)
    return s


def run(s, train=True, leaves=None):
    names = [n for n in NAMES + ["state"] if s[n] is not None]
    v = leaves or {n: s[n].cuda().requires_grad_(train) for n in names}
    lengths = None if s["lengths"] is None else s["lengths"].cuda()
    y, last = pcb().gated_delta(*(v.get(n) for n in NAMES + ["state"]), lengths, s["dim"], s["reverse"], s["scale"], s["logits"])
    out = {"y": y, "last": last}
    if train:
        outs, grads = ([y, last], [s["gy"].cuda(), s["glast"].cuda()]) if s["use_last"] else ([y], [s["gy"].cuda()])
        out |= dict(zip(["g" + n for n in names], torch.autograd.grad(outs, [v[n] for n in names], grads)))
    return out


def compare(s, train=True):
    got, ref = run(s, train), bounds(s, train)
    assert set(got) == set(ref)
    for k, (value, bound) in ref.items():
        check(got[k], value, bound, k)
    if s["lengths"] is not None:
        behind = s["behind"].cuda()
        for k in set(got) & {"y", "gq", "gk", "gv", "gg", "gb"}:
            assert not got[k][behind].any(), k
    return got


# (dimensions before the heads, heads of keys, of values, channels of keys, of values) and what else
CASES = {
    "one step": ((1, 1), 1, 1, 4, 3, {}),
    "one channel": ((2, 5), 1, 2, 1, 1, dict(state=True)),
    "no steps": ((2, 0), 2, 2, 16, 16, dict(state=True)),
    "no sequences": ((0, 9), 2, 2, 16, 16, {}),
    "two steps, one state": ((3, 2), 2, 2, 32, 32, dict(state=True)),
    "a chunk less one": ((2, 63), 2, 2, 32, 32, dict(state=True)),
    "a chunk": ((2, 64), 3, 3, 24, 40, {}),
    "a chunk and one": ((2, 65), 1, 1, 33, 20, dict(state=True, reverse=True)),
    "odd sizes": ((2, 130), 2, 2, 13, 7, dict(state=True)),
    "40 channels": ((2, 100), 3, 3, 40, 40, dict(reverse=True)),
    "64 channels": ((2, 150), 2, 2, 64, 64, dict(state=True)),
    "65 channels": ((1, 70), 1, 1, 65, 33, dict(state=True)),
    "128 channels": ((1, 130), 2, 2, 128, 128, dict(state=True)),
    "more values": ((1, 90), 2, 2, 16, 128, {}),
    "more keys": ((1, 90), 1, 1, 128, 16, dict(state=True)),
    "shared, 32": ((2, 100), 2, 6, 32, 24, dict(state=True)),
    "shared, 64": ((2, 100), 1, 2, 64, 64, {}),
    "shared, 128": ((1, 100), 2, 4, 128, 72, dict(state=True)),
    "lengths": ((6, 140), 2, 2, 32, 32, dict(lengths=[0, 1, 64, 65, 140, 999], state=True)),
    "lengths, reversed, shared": ((4, 90), 1, 2, 48, 48, dict(lengths=[-3, 1, 70, 90], reverse=True, state=True)),
    "down the columns": ((2, 70, 5), 2, 2, 16, 16, dict(dim=1, state=True)),
    "along the rows of columns": ((2, 3, 66, 2), 2, 4, 24, 16, dict(dim=2, reverse=True)),
    "columns with lengths": ((3, 40, 4), 2, 2, 32, 32, dict(dim=1, lengths=[40, 0, 17], state=True)),
    "first dimension": ((50, 3), 2, 2, 16, 16, dict(dim=0, state=True)),
    "gates of 32 bits": ((2, 80), 2, 2, 32, 32, dict(gates=torch.float32)),
    "gates themselves": ((2, 80), 2, 2, 32, 32, dict(logits=False, gates=torch.float32, state=True)),
    "last state unused": ((2, 80), 2, 2, 32, 32, dict(use_last=False, scale=1.0)),
    "segments": ((1, 1300), 1, 1, 32, 32, dict(state=True)),
    "segments, shared, reversed": ((1, 1100), 1, 2, 64, 40, dict(reverse=True, lengths=[1030], state=True)),
    "segments, 128": ((1, 900), 1, 1, 128, 128, dict(state=True)),
}


def case(name, dtype, **more):
    *sizes, options = CASES[name]
    return data(*sizes, dtype, **{**options, **more})


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", CASES)
def test_against_the_recurrence(name, dtype):
    compare(case(name, dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lead,more", [((2, 0), {}), ((3, 1), {}), ((2, 7), dict(reverse=True)), ((2, 16), dict(lengths=[3, 16])), ((2, 17), {}),
                                       ((3, 75), dict(lengths=[75, 0, 9])), ((1, 1500), {}), ((2, 6, 5), dict(dim=1))], ids=str)
@pytest.mark.parametrize("sizes", [(2, 4, 40, 36), (1, 1, 128, 128), (3, 3, 17, 5)], ids=str)
def test_without_gradients(sizes, lead, more, dtype):
    """Few steps go one after another, more in chunks: the same rule, and near the pass that keeps states for its gradients."""
    s = data(lead, *sizes, dtype, state=True, **more)
    compare(s, train=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("value", ["-inf", "min", "some"])
@pytest.mark.parametrize("T", [5, 130])
def test_gates_that_forget_everything(T, value, dtype):
    """Decays of 0: what was before is gone, as if sequences began there; also all of them, and with gates of the type's lowest value."""
    s = data((2, T), 2, 2, 32, 24, dtype, state=True)
    lowest = float("-inf") if value != "min" else torch.finfo(dtype).min
    where = torch.rand(s["g"].shape, generator=torch.Generator().manual_seed(1)) < (0.2 if value == "some" else 1.1)
    s["g"][where] = lowest
    for logits in (True, False):
        if not logits:
            s["g"], s["b"] = -s["g"].abs(), torch.sigmoid(s["b"].double()).to(dtype)
        s["logits"] = logits
        got = compare(s)
        assert not got["gg"].cpu()[where].any()
        compare(s, train=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gates_at_their_ends(dtype):
    """Logits far out: nothing fades and nothing is written, all is replaced."""
    s = data((2, 100), 2, 2, 16, 16, dtype, state=True)
    s["g"][0], s["b"][0, 50:] = 1e4, -1e4
    s["b"][1, :, 0], s["b"][1, :, 1] = 1e4, float("-inf")
    got = compare(s)
    assert not got["gv"][1, :, 1].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T", [9, 200])
def test_keys_and_queries_of_zeros(T, dtype):
    """Rows of padding: a key of 0 writes nothing, and nothing but the decay happens."""
    s = data((2, T), 2, 2, 32, 32, dtype, state=True)
    s["k"][0], s["q"][1], s["v"][1, T // 2:] = 0, 0, 0
    compare(s)
    compare(s, train=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_what_is_not_finite_stays_in_its_chain(dtype):
    s = data((3, 90), 2, 2, 32, 32, dtype, state=True)
    base = run(s)
    s["v"][1, 40, 0, 3], s["k"][2, 5, 1, 0] = float("nan"), float("inf")
    got = run(s)
    for k in got:
        fine = torch.ones(got[k].shape, dtype=torch.bool)
        if k in ("last", "gstate"):
            fine[1, 0] = fine[2, 1] = False
        else:
            fine[1, :, 0] = fine[2, :, 1] = False
        assert torch.equal(got[k].cpu()[fine], base[k].cpu()[fine]), k
    assert torch.equal(got["y"][1, :40].cpu(), base["y"][1, :40].cpu()) or got["y"][1, :40].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", ["a chunk and one", "shared, 64", "down the columns", "128 channels"])
@pytest.mark.parametrize("how", ["slices", "heads first", "unaligned"])
def test_where_tensors_lie(how, name, dtype):
    """Slices of one projection, tensors with their heads ahead of the steps, rows off any alignment: the dense tensors' results."""
    s = case(name, dtype)
    dense, few = run(s), run(s, train=False)
    names = [n for n in NAMES + ["state"] if s[n] is not None]
    v = {n: s[n].cuda() for n in names}
    if how == "slices":
        flat = [v[n].flatten(-2) if n in "qkv" else v[n] for n in NAMES]
        parts = torch.cat(flat, -1).split([t.shape[-1] for t in flat], -1)
        v.update({n: p.unflatten(-1, s[n].shape[-2:]) if n in "qkv" else p for n, p in zip(NAMES, parts)})
    elif how == "heads first":
        for n in NAMES:
            to = -3 if n in "qkv" else -2
            h = s[n].dim() - (2 if n in "qkv" else 1)
            v[n] = v[n].movedim(h, 1).contiguous().movedim(1, h)
    else:
        for n in NAMES:
            store = torch.empty(v[n].numel() + 1, device="cuda", dtype=dtype)
            store[1:] = v[n].flatten()
            v[n] = store[1:].view(v[n].shape)
    got = run(s, leaves={n: t.detach().requires_grad_() for n, t in v.items()})
    for k in dense:
        assert torch.equal(got[k], dense[k]), k
    got = run(s, train=False, leaves={n: t.detach() for n, t in v.items()})
    for k in few:
        assert torch.equal(got[k], few[k]), k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_broadcast_keys_get_the_sum_of_their_gradients(dtype):
    """One key and one gate for all value heads by expand: autograd sums what the kernels give each."""
    s = data((2, 70), 3, 3, 32, 16, dtype, state=True)
    for n in ("k", "g"):
        s[n] = s[n][:, :, :1].expand(s[n].shape).clone()
    whole = run(s)
    v = {n: s[n].cuda().requires_grad_() for n in NAMES + ["state"]}
    one = {n: s[n][:, :, :1].cuda().requires_grad_() for n in ("k", "g")}
    y, last = pcb().gated_delta(v["q"], one["k"].expand(s["k"].shape), v["v"], one["g"].expand(s["g"].shape), v["b"], v["state"])
    # (the state's gradient is asked for in both: what lies between is kept in as many bits)
    got = torch.autograd.grad([y, last], [*one.values(), v["state"]], [s["gy"].cuda(), s["glast"].cuda()])
    for n, t in zip(one, got):
        assert torch.equal(t, whole["g" + n].sum(2, keepdim=True)), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_offsets_past_32_bits(dtype):
    """The second sequence lies 2^31 + 64 elements behind the first, and so do gates and steps."""
    T, h, d, far = 70, 2, 32, (1 << 31) + 64
    s = data((2, T), h, h, d, d, dtype)
    dense, few = run(s, train=False), None
    store = torch.empty(far + T * h * d, device="cuda", dtype=dtype)
    v = {n: s[n].cuda() for n in NAMES}
    for n in ("q", "v", "g"):
        tail = (h * d, d, 1) if n != "g" else (h, 1)
        far_view = store.as_strided(s[n].shape, (far, *tail))
        far_view.copy_(v[n])
        got = run(s, train=False, leaves={**v, n: far_view})
        for k in dense:
            assert torch.equal(got[k], dense[k]), (n, k)
    # steps far apart: one sequence of three
    s = data((1, 3), h, h, d, d, dtype)
    dense = run(s, train=False)
    del store
    store = torch.empty(2 * far + h * d, device="cuda", dtype=dtype)
    far_view = store.as_strided(s["k"].shape, (0, far, d, 1))
    far_view.copy_(s["k"].cuda())
    v = {n: s[n].cuda() for n in NAMES}
    for train in (False, True):   # (step by step, and in a chunk)
        ref = run(s, train)
        got = run(s, train, leaves={n: (far_view if n == "k" else v[n]).detach().requires_grad_(train) for n in NAMES})
        for k in ref:
            assert torch.equal(got[k], ref[k]), k


@pytest.mark.parametrize("name", ["a chunk and one", "shared, 32", "lengths, reversed, shared"])
def test_gradients_are_differences(name):
    """Along random directions in 32 bits: (f(x + h v) - f(x - h v)) / 2h is off by h^2 of the third derivative, which two widths show, and by the
    roundings of both values, 2^-18 of the sum of magnitudes."""
    s = case(name, torch.float32, nan=False)
    grads = run(s)
    live = ~s["behind"]
    gen = torch.Generator().manual_seed(5)
    for n in [n for n in NAMES + ["state"] if s[n] is not None]:
        v = torch.randn(s[n].shape, generator=gen)
        v /= v.abs().max()

        def along(h):
            rs = [run({**s, n: s[n] + e * h * v}, train=False) for e in (1, -1)]
            pick = lambda r: [(r["y"].double().cpu() * s["gy"].double())[live], r["last"].double().cpu() * s["glast"].double()]
            f = [sum(float(t.sum()) for t in pick(r)) for r in rs]
            return (f[0] - f[1]) / (2 * h), 2.0 ** -18 * sum(float(t.abs().sum()) for t in pick(rs[0])) / h

        (a, ra), (b, rb) = along(2.0 ** -6), along(2.0 ** -5)
        slope = float((grads["g" + n].double().cpu() * v.double()).sum())
        assert abs(slope - a) <= abs(b - a) + ra + rb, (n, slope, a, b, ra)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1), (2, 6, 40, 36), (3, 3, 128, 128), (8, 16, 64, 64), (1, 2, 17, 5)], ids=str)
@pytest.mark.parametrize("streams", [0, 1, 70])
def test_step(streams, sizes, dtype):
    """One step: in place and into another state; a call of one step gives the same bits."""
    s = data((streams, 1), *sizes, dtype, state=True)
    v = {n: s[n][:, 0].cuda() for n in NAMES}
    old = s["state"].cuda()
    to = torch.full_like(old, float("nan"))
    y, new = pcb().gated_delta_step(*v.values(), old, to)
    assert new is to and torch.equal(old.cpu(), s["state"])
    ref = bounds(s, train=False)
    check(y[:, None], *ref["y"], "y"), check(new, *ref["last"], "last")
    version = old._version
    y2, new2 = pcb().gated_delta_step(*v.values(), old)
    assert new2 is old and old._version > version and torch.equal(y2, y) and torch.equal(old, to)
    with torch.no_grad():
        y3, last = pcb().gated_delta(*(s[n].cuda() for n in NAMES), s["state"].cuda())
    assert torch.equal(y3[:, 0], y) and torch.equal(last, to)


def test_step_where_tensors_lie_and_refusals():
    s = data((5, 1), 2, 4, 24, 40, torch.bfloat16, state=True)
    v = {n: s[n][:, 0].cuda() for n in NAMES}
    y, new = pcb().gated_delta_step(*v.values(), s["state"].cuda())
    wide = torch.cat([t.flatten(1) for t in v.values()], -1)
    parts = wide.split([t.flatten(1).shape[1] for t in v.values()], -1)
    sliced = [p.unflatten(-1, v[n].shape[1:]) if n in "qkv" else p for n, p in zip(NAMES, parts)]
    y2, new2 = pcb().gated_delta_step(*sliced, s["state"].cuda())
    assert torch.equal(y, y2) and torch.equal(new, new2)
    state = s["state"].cuda()
    store = torch.zeros(2 * state.numel(), device="cuda")
    half = state.numel() // 2
    with pytest.raises(ValueError, match="overlap"):
        pcb().gated_delta_step(*v.values(), store[:state.numel()].view(state.shape), store[half:half + state.numel()].view(state.shape))
    with pytest.raises(ValueError, match="dense"):
        pcb().gated_delta_step(*v.values(), state.transpose(-1, -2).contiguous().transpose(-1, -2))
    with pytest.raises(RuntimeError, match="no gradient"):
        pcb().gated_delta_step(v["q"].clone().requires_grad_(), *list(v.values())[1:], state)
    with torch.no_grad():
        pcb().gated_delta_step(v["q"].clone().requires_grad_(), *list(v.values())[1:], state)
    with torch.inference_mode():
        pcb().gated_delta_step(*v.values(), torch.zeros_like(state))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_pieces_and_steps_continue_a_state(dtype):
    """A sequence in pieces, with and without what gradients need, and its end in single steps: the recurrence's results for the whole."""
    s = data((2, 300), 2, 4, 32, 48, dtype, state=True)
    ref = bounds(s, train=False)
    v = {n: s[n].cuda() for n in NAMES}
    h, ys = s["state"].cuda(), []
    for a, b, grad in ((0, 1, False), (1, 9, False), (9, 150, True), (150, 150, False), (150, 297, False)):
        y, h = pcb().gated_delta(*(v[n][:, a:b].clone().requires_grad_(grad) for n in NAMES), h)
        h = h.detach()
        ys.append(y.detach())
    for t in range(297, 300):
        y, same = pcb().gated_delta_step(*(v[n][:, t] for n in NAMES), h)
        assert same is h
        ys.append(y[:, None])
    # (each piece's roundings as in one pass)
    check(torch.cat(ys, 1), ref["y"][0], 2 * ref["y"][1], "y")
    check(h, ref["last"][0], 2 * ref["last"][1], "last")


def test_gradients_that_nothing_asks_for():
    for dtype in (torch.float32, torch.bfloat16):
        s = case("shared, 64", dtype, state=True)
        whole = run(s)
        v = {n: s[n].cuda().requires_grad_() for n in NAMES + ["state"]}
        outs = pcb().gated_delta(*v.values())
        for n in v:
            (got,) = torch.autograd.grad(outs, [v[n]], [s["gy"].cuda(), s["glast"].cuda()], retain_graph=True)
            # (with the gradient of a state more of what lies between is kept: at most both roundings apart)
            assert torch.equal(got, whole["g" + n]) or (dtype != torch.float32 and n != "state"), n
            step = torch.finfo(dtype).eps * whole["g" + n].abs().float() + 2.0 ** -12 * whole["g" + n].abs().max().float()
            assert float(((got.float() - whole["g" + n].float()).abs() - step).max()) <= 0, n
        only_last = torch.autograd.grad(outs[1], [v["k"], v["q"]], s["glast"].cuda(), retain_graph=True, allow_unused=True)
        assert only_last[0].any() and (only_last[1] is None or not only_last[1].any())


def test_function_form_module_trace_checkpoint_and_no_second_derivative():
    from torch.utils.checkpoint import checkpoint

    s = data((2, 150), 2, 2, 32, 20, torch.float32, state=True, lengths=[150, 31], reverse=True)
    base = run(s)
    v = [s[n].cuda().requires_grad_() for n in NAMES + ["state"]]
    more = (s["lengths"].cuda(), 1, True, s["scale"], True)
    grads = [s["gy"].cuda(), s["glast"].cuda()]
    for out in (pcb().GatedDeltaFunction.apply(*v, *more), pcb().GatedDelta(dim=1, reverse=True)(*v, more[0]),
                checkpoint(lambda *t: pcb().gated_delta(*t, *more), *v, use_reentrant=False)):
        for k, t in zip(("y", "last", "gq", "gk", "gv", "gg", "gb", "gstate"), (*out, *torch.autograd.grad(out, v, grads))):
            assert torch.equal(t, base[k]), k
    f = lambda a: pcb().gated_delta(a, a, a, a[..., 0], a[..., 1])[0]
    x, other = torch.randn(2, 9, 2, 8, device="cuda"), torch.randn(3, 100, 2, 8, device="cuda") * 0.3
    traced = torch.jit.trace(f, (x,), check_trace=False)
    torch.testing.assert_close(traced(other), f(other), rtol=1e-4, atol=1e-4)   # (a trace's form keeps states: another order of products)
    with pytest.raises((RuntimeError, TypeError, ValueError)):
        traced(other.double())
    y, last = pcb().gated_delta(*v)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum() + last.sum(), v[0], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x[None])


def test_saved_tensor_changed_in_place_is_noticed():
    s = case("a chunk", torch.float32)
    v = {n: s[n].cuda().requires_grad_() for n in NAMES}
    k = v["k"] * 1.0
    y, _ = pcb().gated_delta(v["q"], k, v["v"], v["g"], v["b"])
    k.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("name", ["segments", "shared, 128", "lengths"])
def test_results_are_the_same_on_any_stream_and_every_time(name):
    s = case(name, torch.bfloat16)
    base, few = run(s), run(s, train=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, few2 = run(s), run(s, train=False)
    side.synchronize()
    for k in base:
        assert torch.equal(base[k], again[k]), k
    for k in few:
        assert torch.equal(few[k], few2[k]), k


def layer(x, h, state=None):
    """Queries, keys, values and gates of one projection x [B, T, 3 h d + 2 h], as a layer has them."""
    d = (x.shape[-1] - 2 * h) // (3 * h)
    q, k, v, gates = x.split([h * d, h * d, h * d, 2 * h], -1)
    q, k, v = (t.unflatten(-1, (h, d)) for t in (q, k, v))
    q, k = pcb().head_rotary(q, k, kind="l2")
    return pcb().gated_delta(q, k, v, gates[..., :h], gates[..., h:], state)


def test_two_streams_at_once():
    """Both operators on two streams, under way together, forward and backward: bitwise what each is by itself."""
    xs = [torch.randn(2, 1500, 3 * 2 * 32 + 4, device="cuda").bfloat16().requires_grad_() for _ in range(2)]
    gy = torch.randn(2, 1500, 2, 32, device="cuda").bfloat16()

    def f(x):
        y, last = layer(x, 2)
        with torch.no_grad():
            few = layer(x[:, :5], 2, last)
        return [y.detach(), last.detach(), *few, *torch.autograd.grad(y, [x], gy)]

    alone = [f(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    results = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(f(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in results[i]:
            for a, b in zip(r, alone[i]):
                assert torch.equal(a, b)


def test_captured_passes_replay():
    """Two graphs that stand beside one another, of a whole pass and of one token, replayed with eager work between: every replay is the eager
    result on the same inputs."""
    x = torch.randn(1, 1500, 3 * 2 * 32 + 4, device="cuda").bfloat16().requires_grad_()
    gy = torch.randn(1, 1500, 2, 32, device="cuda").bfloat16()
    h = torch.randn(1, 2, 32, 32, device="cuda")
    to = torch.empty_like(h)

    def whole():
        y, last = layer(x, 2, h)
        return [y.detach(), last.detach(), *torch.autograd.grad(y, [x], gy)]

    def token():
        with torch.no_grad():
            t = x[:, 0]
            q, k, v = t[:, :192].unflatten(-1, (3, 2, 32)).unbind(1)
            q, k = pcb().head_rotary(q, k, positions=torch.full((1, 1), 7, device="cuda", dtype=torch.int32), kind="l2")
            return list(pcb().gated_delta_step(q, k, v, t[:, 192:194], t[:, 194:], h, to))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        whole(), token()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for f in (whole, token):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = f()
        graphs.append((graph, f, res))
    for seed in range(4):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            h.copy_(torch.randn_like(h))
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in res] for _, _, res in graphs]
        for (_, f, _), res in zip(graphs, got):
            for a, b in zip(res, f()):
                assert torch.equal(a, b)


@pytest.mark.parametrize("op", ["rotary", "delta"])
def test_capture_beside_an_eager_graph_is_refused(op):
    """A backward pass under capture whose gradients would go to accumulators of the default stream raises, and leaves the process as it was;
    with the eager output gone the same capture works."""
    q, k, v = (torch.randn(2, 80, 2, 32, device="cuda").requires_grad_() for _ in range(3))
    g = torch.randn(2, 80, 2, device="cuda").requires_grad_()
    w = torch.ones(32, device="cuda").requires_grad_()
    gy = torch.randn(2, 80, 2, 32, device="cuda")

    def forward():
        if op == "rotary":
            return pcb().head_rotary(q, weight=w, kind="rms"), [q, w]
        return pcb().gated_delta(q, k, v, g, g)[0], [q, k, v, g]

    def step():
        y, leaves = forward()
        return torch.autograd.grad(y, leaves, gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    eager = forward()
    with pytest.raises(RuntimeError, match="drop that output first"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    ref = torch.autograd.grad(*eager, gy)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for _ in range(3):
        for t in res:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, ref):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_as_a_layer(dtype):
    """A layer as a model has it: norm, one projection, queries and keys normed and turned, the rule down a sequence, gated residual; gradients of all of
    it against plain operations in 64 bits; then the same sequence token by token.

    Each tensor between the operators is rounded once in 16 bits (2^-9): results agree to a few times 2^-8 of their norm; in 32 bits to a few
    hundred times 2^-24, which a projection's sums and the rule's chunks leave."""
    torch.manual_seed(0)
    B, T, h, d = 2, 90, 2, 32
    C = h * d
    leaf = lambda *s, mean=0.0, std=1.0: (torch.randn(*s) * std + mean).to(dtype)
    p = {"x": leaf(B, T, C), "w1": leaf(C, mean=1.0, std=0.1), "proj": leaf(3 * C + 2 * h, C, std=C ** -0.5), "wq": leaf(d, mean=1.0, std=0.1),
         "wk": leaf(d, mean=0.5, std=0.05), "w2": leaf(C, mean=1.0, std=0.1), "scale": leaf(C, mean=0.5, std=0.1)}
    go = leaf(B, T, C)
    v = {n: t.cuda().requires_grad_() for n, t in p.items()}

    def parts(z, proj):
        y = torch.nn.functional.linear(z, proj)
        q, k, val, gates = y.split([C, C, C, 2 * h], -1)
        return *(t.unflatten(-1, (h, d)) for t in (q, k, val)), gates[..., :h], gates[..., h:]

    def ours(x, positions, state, step=False):
        q, k, val, g, b = parts(pcb().channel_norm(x, v["w1"]), v["proj"])
        q, k = pcb().head_rotary(q, k, v["wq"], v["wk"], positions, kind="l2")
        y, state = (pcb().gated_delta_step if step else pcb().gated_delta)(q, k, val, g, b, state)
        return pcb().gated_residual(x, y.flatten(-2), v["w2"], scale=v["scale"], kind="rms"), state

    out, last = ours(v["x"], None, None)
    grads = torch.autograd.grad(out, list(v.values()), go.cuda())

    r = {n: t.double().requires_grad_() for n, t in p.items()}
    rms = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    l2 = lambda t, w: t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() * w
    q, k, val, g, b = parts(rms(r["x"], r["w1"]), r["proj"])
    t = torch.arange(T, dtype=torch.float64)[:, None] * 1e4 ** -(torch.arange(d // 2, dtype=torch.float64) / (d // 2))
    turn = lambda z: torch.cat([z[..., :d // 2] * t.cos()[:, None] - z[..., d // 2:] * t.sin()[:, None],
                                z[..., d // 2:] * t.cos()[:, None] + z[..., :d // 2] * t.sin()[:, None]], -1)
    ys, lasts = rule64(turn(l2(q, r["wq"])), turn(l2(k, r["wk"])), val, g, b, None, None, 1, False, d ** -0.5, True)
    y = torch.stack(ys).reshape(B, T, C)
    rout = r["x"] + r["scale"] * rms(y, r["w2"])
    rgrads = torch.autograd.grad(rout, list(r.values()), go.double())
    most = 2 ** -6 if dtype != torch.float32 else 2 ** -16
    for name, a, c in zip(["out", "last", *v], [out, last, *grads], [rout, torch.stack(lasts).reshape(last.shape), *rgrads]):
        err = (a.detach().double().cpu() - c.detach()).norm() / c.detach().norm()
        assert err <= most, (name, float(err))
    with torch.no_grad():
        whole, state = ours(v["x"][:, :80], None, None)
        rows = [whole]
        for at in range(80, T):
            row, state = ours(v["x"][:, at], torch.full((1,), at, device="cuda", dtype=torch.int32), state, step=True)
            rows.append(row[:, None])
    err = (torch.cat(rows, 1).double().cpu() - rout.detach()).norm() / rout.detach().norm()
    assert err <= most, float(err)
    err = (state.double().cpu() - torch.stack(lasts).detach().reshape(state.shape)).norm() / torch.stack(lasts).detach().norm()
    assert err <= most, float(err)
