"""head_rotary against its formula in 64 bits, element by element.

Bounds, with U = 2^-24 for each operation in 32 bits and half a step of the result's type for its one rounding: a row's sum of squares is d / lanes products
one after another and some exchanges, its root, reciprocal and three products a few more: (d + 16) U relative for the norm; an angle is
off by 2^-53 of itself for each of four roundings, its sine and cosine by that, 2^-29 of their series and 2 U; a rotation adds two
products.  Sums over rows for the weights: as many additions as a group of lanes has rows, 256 groups, 16 of their sums and 6 exchanges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def pcb():
    import pyramidconvblock_amd

    return pyramidconvblock_amd


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, ref, bound, name):
    got = got.detach()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps   # (half a step of the smallest numbers)
    off = (got.double().cpu() - ref).abs() - (half_step(got.dtype) * (ref.abs() + bound) + bound + tiny)
    assert not torch.isnan(off).any(), name
    assert off.numel() == 0 or float(off.max()) <= 0, (name, float(off.max()), float(bound.max()))


def sections_of(d, axes):
    return [d // 2 // axes + (a < d // 2 % axes) for a in range(axes)]


def angles(lead, positions, axes, sections, frequencies, base):
    """-> angles [lead..., P] and how far they may be off."""
    if positions is None:
        grid = torch.meshgrid(*[torch.arange(n, dtype=torch.float64) for n in lead[-axes:]], indexing="ij")
        pos = torch.stack(grid, -1)
    else:
        pos = positions.double()
    pos = pos.expand(*lead, axes)
    parts, at = [], 0
    for a, n in enumerate(sections):
        f = base ** -(torch.arange(n, dtype=torch.float64) / max(n, 1)) if frequencies is None else frequencies[at:at + n].double()
        parts.append(pos[..., a:a + 1] * f)
        at += n
    t = torch.cat(parts, -1)
    return t, 4 * 2.0 ** -53 * t.abs() + 2.0 ** -29 + 2 * U


def split(y, P, neighbours):
    if neighbours:
        return y[..., 0:2 * P:2], y[..., 1:2 * P:2], y[..., 2 * P:]
    return y[..., :P], y[..., P:2 * P], y[..., 2 * P:]


def joined(a, b, rest, neighbours):
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if neighbours else torch.cat([a, b], -1), rest], -1)


def turned(x, slack, t, dt, neighbours, back=False):
    """x's pairs by t[..., None, :], and the bound: `slack` is x's own."""
    P, t, dt = t.shape[-1], t[..., None, :], dt[..., None, :]
    c, s = t.cos(), t.sin() * (-1 if back else 1)
    a, b, rest = split(x, P, neighbours)
    da, db, drest = split(slack, P, neighbours)
    m = (a.abs() + b.abs()) * (dt + 3 * U)
    return (joined(a * c - b * s, b * c + a * s, rest, neighbours),
            joined(da * c.abs() + db * s.abs() + m, db * c.abs() + da * s.abs() + m, drest, neighbours))


def norm_of(x, kind, eps):
    """-> (r, x r) in 64 bits"""
    if kind == "none":
        return torch.ones_like(x[..., :1]), x
    sq = x.square()
    r = ((sq.mean(-1, keepdim=True) if kind == "rms" else sq.sum(-1, keepdim=True)) + eps).rsqrt()
    return r, x * r


def reference(x, w, gy, t, dt, kind, eps, neighbours):
    """-> {name: (value, bound)} of one of q and k"""
    d, w64 = x.shape[-1], 1.0 if w is None else w.double()
    x = x.double()
    c = (d + 16) * U if kind != "none" else 0.0
    r, n = norm_of(x, kind, eps)
    out = {"y": turned(n * w64, (n * w64).abs() * c, t, dt, neighbours)}
    if gy is None:
        return out
    g, dg = turned(gy.double(), torch.zeros_like(x), t, dt, neighbours, back=True)
    if kind == "none":
        out["gx"] = (g, dg)
        return out
    u, du = g * w64, dg * (w64 if w is None else w64.abs()) + 2 * U * (g * w64).abs()
    part = 1.0 / d if kind == "rms" else 1.0
    dot = (u * n).sum(-1, keepdim=True) * part
    ddot = ((du + 3 * c * u.abs()) * n.abs()).sum(-1, keepdim=True) * part
    out["gx"] = (r * (u - n * dot), r * (du + n.abs() * ddot + 3 * c * (u.abs() + (n * dot).abs())))
    if w is not None:
        rows = x.numel() // d
        terms = g * n
        adds = 300 + rows / 64
        out["gw"] = (terms.reshape(-1, d).sum(0), ((dg + c * g.abs()) * n.abs() + adds * U * terms.abs()).reshape(-1, d).sum(0))
    return out


# (dimensions before the heads, heads of q and k (0: none), d, kind, weights, axes, sections, neighbours, positions, own frequencies)
CASES = {
    "one": ((1,), 1, 1, 2, "rms", True, 1, None, False, None, False),
    "one channel": ((3,), 2, 0, 1, "l2", True, 1, None, False, None, False),
    "no tokens": ((0, 4), 3, 2, 16, "rms", True, 1, None, False, None, False),
    "no heads of k": ((5,), 3, 0, 16, "none", False, 1, None, True, None, False),
    "odd d": ((2, 7), 3, 1, 13, "rms", True, 1, None, False, None, False),
    "odd d, neighbours": ((2, 7), 3, 1, 27, "l2", False, 1, (5,), True, None, False),
    "rows and columns": ((2, 9, 11), 5, 5, 40, "rms", True, 2, None, True, None, False),
    "frames, rows, columns": ((2, 3, 5, 7), 8, 4, 64, "rms", True, 3, None, False, None, False),
    "uneven sections": ((3, 4, 6), 2, 2, 32, "l2", True, 3, (7, 0, 4), False, None, False),
    "nothing turned": ((6, 5), 2, 1, 24, "rms", True, 1, (0,), False, None, False),
    "part of a head": ((700,), 9, 9, 128, "none", False, 1, (16,), False, None, False),
    "given": ((3, 50), 4, 2, 48, "l2", False, 1, None, True, (torch.int32, 1, 1000), False),
    "far": ((2, 60), 3, 1, 64, "none", False, 1, None, False, (torch.int64, 2, 1 << 20), False),
    "farthest": ((2, 60), 1, 3, 64, "rms", False, 1, None, False, (torch.int64, 1, (1 << 31) - 1), False),
    "between": ((4, 6, 7), 2, 2, 56, "rms", True, 2, None, True, (torch.float32, 2, 100), True),
    "all positions": ((2, 9, 11), 5, 5, 40, "rms", True, 2, None, False, (torch.int32, 3, 300), True),
    "256 channels": ((3, 100), 2, 1, 256, "rms", True, 1, None, False, None, False),
    "255 channels": ((2, 40), 2, 1, 255, "l2", True, 1, None, True, None, False),
    "many rows": ((2, 61, 67), 7, 3, 36, "rms", True, 2, None, False, None, False),
    "many heads": ((5,), 300, 7, 8, "rms", True, 1, None, False, None, False),
}


def data(case, dtype, seed=0):
    lead, hq, hk, d, kind, weights, axes, sections, neighbours, positions, own = CASES[case]
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s, mean=0.0: (torch.randn(*s, generator=gen) + mean).to(dtype)
    s = {n: rnd(*lead, h, d) if h else None for n, h in (("q", hq), ("k", hk))}
    s.update({"g" + n: rnd(*lead, h, d) if h else None for n, h in (("q", hq), ("k", hk))})
    s["weight"] = rnd(d, mean=1.0) if weights else None
    s["key_weight"] = rnd(d, mean=1.0) if weights and hk else None
    sections = sections_of(d, axes) if sections is None else list(sections)
    s["positions"] = None
    if positions is not None:
        kind_of, dims, far = positions
        p = torch.randint(-far // 2 if far <= 1 << 20 else 0, far, (*lead[len(lead) - dims:], axes), generator=gen)
        s["positions"] = p.to(kind_of) if kind_of != torch.float32 else p.float() / 16
    s["frequencies"] = torch.rand(sum(sections), generator=gen) * 2 if own else None
    s["more"] = dict(axes=axes, sections=sections, kind=kind, neighbours=neighbours, base=1e4, eps=1e-6)
    return s


def run(s, train=True, leaves=None):
    names = [n for n in ("q", "k", "weight", "key_weight") if s[n] is not None]
    v = leaves or {n: s[n].cuda().requires_grad_(train) for n in names}
    cuda = lambda t: None if t is None else t.cuda()
    out = pcb().head_rotary(v["q"], v.get("k"), v.get("weight"), v.get("key_weight"), cuda(s["positions"]), frequencies=cuda(s["frequencies"]), **s["more"])
    outs = list(out) if isinstance(out, tuple) else [out]
    grads = torch.autograd.grad(outs, [v[n] for n in names], [cuda(s["g" + n]) for n in ("q", "k") if s[n] is not None]) if train else []
    return dict(zip(["yq", "yk"], outs)) | dict(zip(["g" + n for n in names], grads))


def expected(s, train=True):
    m = s["more"]
    t, dt = angles(s["q"].shape[:-2], s["positions"], m["axes"], m["sections"], s["frequencies"], m["base"])
    ref = {}
    for n, w in (("q", "weight"), ("k", "key_weight")):
        if s[n] is None:
            continue
        r = reference(s[n], s[w], s["g" + n] if train else None, t, dt, m["kind"], m["eps"], m["neighbours"])
        ref["y" + n] = r["y"]
        if train:
            ref["g" + n] = r["gx"]
            if s[w] is not None:
                ref["g" + w] = r["gw"]
    return ref


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", CASES)
def test_against_the_formula(case, dtype):
    s = data(case, dtype)
    got, ref = run(s), expected(s)
    assert set(got) == set(ref)
    for k, (value, bound) in ref.items():
        check(got[k], value, bound, k)
    plain = run(s, train=False)
    for k in plain:
        assert torch.equal(plain[k], got[k]), k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", ["rows and columns", "odd d", "part of a head", "given"])
@pytest.mark.parametrize("how", ["slices", "transposed", "unaligned", "expanded"])
def test_where_tensors_lie(how, case, dtype):
    """Slices of a fused projection, heads ahead of tokens, rows off any alignment, one head for all of them."""
    s = data(case, dtype)
    dense = run(s)
    v = {n: s[n].cuda() for n in ("q", "k", "weight", "key_weight") if s[n] is not None}
    if how == "slices":
        wide = torch.cat([v["q"].flatten(-2), v["k"].flatten(-2)], -1)
        v["q"], v["k"] = (t.unflatten(-1, (-1, s["q"].shape[-1])) for t in wide.split([v["q"].flatten(-2).shape[-1], v["k"].flatten(-2).shape[-1]], -1))
    elif how == "transposed":
        for n in ("q", "k"):
            v[n] = v[n].movedim(-2, 0).contiguous().movedim(0, -2)
    elif how == "unaligned":
        for n in v:
            store = torch.empty(v[n].numel() + 1, device="cuda", dtype=dtype)
            store[1:] = v[n].flatten()
            v[n] = store[1:].view(v[n].shape)
    else:
        for n in ("q", "k"):
            s[n] = s[n][..., :1, :].expand(s[n].shape).clone()
        dense = run(s)
        v.update({n: s[n][..., :1, :].cuda().expand(s[n].shape) for n in ("q", "k")})
    got = run(s, leaves={n: t.detach().requires_grad_() for n, t in v.items()})
    for k in dense:
        assert torch.equal(got[k], dense[k]), k


def test_a_head_that_all_share_gets_the_sum_of_their_gradients():
    s = data("given", torch.float32)
    lead, h, d = s["q"].shape[:-2], s["q"].shape[-2], s["q"].shape[-1]
    one = s["q"][..., :1, :].cuda().requires_grad_()
    y = pcb().head_rotary(one.expand(*lead, h, d), positions=s["positions"].cuda(), **s["more"])
    (g,) = torch.autograd.grad(y, [one], s["gq"].cuda())
    s["q"], s["k"] = s["q"][..., :1, :].expand(*lead, h, d), None
    value, bound = expected(s)["gq"]
    check(g, value.sum(-2, keepdim=True), (bound + 2 * h * U * value.abs()).sum(-2, keepdim=True), "g")


@pytest.mark.parametrize("case", ["rows and columns", "uneven sections", "given"])
def test_gradients_are_differences(case):
    """Along random directions: (f(x + h v) - f(x - h v)) / 2h is off by h^2 of the third derivative, which two widths show, and by the roundings
    of both values, 64 U of the sum of magnitudes."""
    s = data(case, torch.float32)
    names = [n for n in ("q", "k", "weight", "key_weight") if s[n] is not None]
    grads = run(s)
    outs = [n for n in ("q", "k") if s[n] is not None]
    gen = torch.Generator().manual_seed(5)
    for n in names:
        v = torch.randn(s[n].shape, generator=gen)
        v /= v.abs().max()

        def along(h):
            r = [run({**s, n: s[n] + e * h * v}, train=False) for e in (1, -1)]
            f = [sum(float((x["y" + o].double().cpu() * s["g" + o].double()).sum()) for o in outs) for x in r]
            size = sum(float((r[0]["y" + o].double().cpu() * s["g" + o].double()).abs().sum()) for o in outs)
            return (f[0] - f[1]) / (2 * h), 64 * U * size / h

        (a, ra), (b, rb) = along(2.0 ** -6), along(2.0 ** -5)
        slope = float((grads["g" + n].double().cpu() * v.double()).sum())
        assert abs(slope - a) <= abs(b - a) + ra + rb, (n, slope, a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_of_zeros_infinities_and_nan_stay_among_themselves(dtype):
    """A row of zeros is 0 and its gradient finite; what is not finite in one row is in no other."""
    s = data("rows and columns", dtype)
    s["q"][0, 1, 2, 3], s["q"][1, 3, 4, 0, 5], s["k"][0, 0, 0, 1] = 0, float("nan"), float("inf")
    got = run(s)
    assert not got["yq"][0, 1, 2, 3].any() and got["gq"][0, 1, 2, 3].isfinite().all()
    for n, bad in (("q", (1, 3, 4, 0)), ("k", (0, 0, 0, 1))):
        for k in ("y" + n, "g" + n):
            fine = torch.ones(s[n].shape[:-1], dtype=torch.bool)
            fine[bad] = False
            assert got[k].cpu()[fine].isfinite().all(), k
            assert not got[k].cpu()[bad].isfinite().any() or n == "k", k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_offsets_past_32_bits(dtype):
    """The second batch element lies 2^31 + 64 elements behind the first."""
    d, T, far = 32, 5, (1 << 31) + 64
    store = torch.empty(far + T * 2 * d, device="cuda", dtype=dtype)
    q = store.as_strided((2, T, 2, d), (far, 2 * d, d, 1))
    x = torch.randn(2, T, 2, d, device="cuda").to(dtype)
    q.copy_(x)
    assert torch.equal(pcb().head_rotary(q, kind="l2"), pcb().head_rotary(x, kind="l2"))


def test_gradients_that_nothing_asks_for():
    """One output, one leaf: the others' work is left out and the results stay what they are."""
    s = data("rows and columns", torch.bfloat16)
    whole = run(s)
    v = {n: s[n].cuda().requires_grad_() for n in ("q", "k", "weight", "key_weight")}
    y, yk = pcb().head_rotary(*v.values(), **s["more"])
    for n, out, g in (("q", y, "gq"), ("weight", y, "gq"), ("k", yk, "gk"), ("key_weight", yk, "gk")):
        (got,) = torch.autograd.grad(out, [v[n]], s[g].cuda(), retain_graph=True)
        assert torch.equal(got, whole["g" + n]), n
    zero = torch.autograd.grad(yk, [v["q"], v["weight"]], s["gk"].cuda(), retain_graph=True, allow_unused=True)
    assert all(t is None or not t.any() for t in zero)
    none = torch.zeros(3, 0, 8, device="cuda").requires_grad_()
    w = torch.ones(8, device="cuda").requires_grad_()
    out = pcb().head_rotary(none, weight=w, kind="rms")
    (g,) = torch.autograd.grad(out, [w], torch.zeros_like(out))
    assert not g.any()


def test_function_form_module_trace_and_no_second_derivative():
    s = data("rows and columns", torch.float32)
    m = s["more"]
    base = run(s)
    v = [s[n].cuda().requires_grad_() for n in ("q", "k", "weight", "key_weight")]
    out = pcb().HeadRotaryFunction.apply(*v, None, None, m["axes"], tuple(m["sections"]), m["base"], 1, m["neighbours"], m["eps"])
    grads = torch.autograd.grad(out, v, [s["gq"].cuda(), s["gk"].cuda()])
    for k, t in zip(("yq", "yk", "gq", "gk", "gweight", "gkey_weight"), (*out, *grads)):
        assert torch.equal(t, base[k]), k
    layer = pcb().HeadRotary(40, axes=2, neighbours=True).cuda()
    with torch.no_grad():
        layer.weight.copy_(v[2]), layer.key_weight.copy_(v[3])
    for a, b in zip(layer(v[0], v[1]), out):
        assert torch.equal(a, b)
    assert torch.equal(layer(v[0]), out[0])
    w = v[2].detach()
    f = lambda a: pcb().head_rotary(a, weight=w, kind="rms", axes=2)
    other = torch.randn(5, 4, 3, 2, 40, device="cuda")
    assert torch.equal(torch.jit.trace(f, (v[0].detach(),), check_trace=False)(other), f(other))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(f(v[0]).sum(), v[0], create_graph=True)
    from torch.utils.checkpoint import checkpoint

    gy = s["gq"].cuda()
    (plain,), (again,) = (torch.autograd.grad(y, [v[0]], gy) for y in (f(v[0]), checkpoint(f, v[0], use_reentrant=False)))
    assert torch.equal(plain, again)


def test_streams():
    """Passes on two streams, under way together: bitwise what each is by itself."""
    sets = [data("frames, rows, columns", torch.bfloat16, seed) for seed in (1, 2)]
    on = [{n: s[n].cuda().requires_grad_() for n in ("q", "k", "weight", "key_weight")} for s in sets]
    alone = [run(s, leaves=v) for s, v in zip(sets, on)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    results = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(run(sets[i], leaves=on[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in results[i]:
            for k in r:
                assert torch.equal(r[k], alone[i][k]), k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("nothing", [dict(tokens=0), dict(heads=(0, 0)), dict(heads=(0, 2))], ids=str)
def test_library_writes_the_gradients_of_weights_without_rows(nothing, dtype):
    """From C: zeros into each gradient that is asked for, and no other memory."""
    import ctypes

    from pyramidconvblock_amd import _lib

    L, d = _lib.lib(), 24
    c = _lib.Rotary()
    x, w = torch.ones(5, 2, d, device="cuda", dtype=dtype), torch.ones(2, d, device="cuda", dtype=dtype)
    c.tokens, c.d, c.axes, c.kind, c.dtype, c.eps, c.base = nothing.get("tokens", 5), d, 1, 1, _lib.dtype_code(dtype), 1e-6, 1e4
    c.x[:], c.heads[:], c.sections[:], c.grid[:] = (x.data_ptr(),) * 2, nothing.get("heads", (2, 2)), (4, 0, 0), (5, 0, 0)
    c.xt[:], c.xh[:], c.weight[:] = (2 * d, 2 * d), (d, d), (w[0].data_ptr(), w[1].data_ptr())
    gw = torch.full((4, d), float("nan"), device="cuda", dtype=dtype)
    work = torch.empty(L.pdw_rotary_bwd_workspace_bytes(d), device="cuda", dtype=torch.uint8)
    two = lambda a, b: (ctypes.c_void_p * 2)(a, b)
    gys, gxs = two(x.data_ptr(), x.data_ptr()), two(None, None)
    for rows in ((0, 2), (0, None), (None, 2)):
        gw.fill_(float("nan"))
        to = two(*(None if r is None else gw[r].data_ptr() for r in rows))
        assert L.pdw_rotary_bwd(ctypes.addressof(c), *(ctypes.addressof(a) for a in (gys, gxs, to)), work.data_ptr(), work.numel(),
                                torch.cuda.current_stream().cuda_stream) == 0, L.pdw_last_error()
        for r in range(4):
            if r not in rows:
                assert gw[r].isnan().all(), (rows, r)
            elif r == 0 or c.tokens == 0 or c.heads[1] == 0:
                assert not gw[r].any() and not gw[r].isnan().any(), (rows, r)
