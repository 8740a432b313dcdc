"""channel_norm and gated_residual against the formulas in 64 bits, on identically rounded inputs, forward and backward.

Bounds, element by element: half a step of the type for the one rounding of a result, and for what happens in 32 bits before it
u = 2^-24 a rounding, times how many there are.  A sum over C channels is at most 32 additions in a lane and 8 exchanges, the rest of a
formula some ten operations more: 64 u of the sum of the magnitudes that go into it.  A sum over N rows is, in a lane, N / 1024 rows or one,
and at most 40 additions from there to the result.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6


def pcb():
    import pyramidconvblock_amd

    return pyramidconvblock_amd


def rnd(gen, *shape, dtype=torch.float32, mean=0.0, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float64) * std + mean).to(dtype)


def check(got, ref, slack, what):
    """|got - ref| <= half a step + slack, everywhere"""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    dtype = got.dtype
    got = got.detach().double().cpu()
    bound = torch.finfo(dtype).eps / 2 * (ref.abs() + slack) + slack + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - ref).abs() / bound).nan_to_num(9e9).max()):.2f} of the bound"


def norm64(v, w, b, kind):
    """-> (norm, n, r, a bound on the error of n in 32 bits)"""
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1 / (c.square().mean(-1, keepdim=True) + EPS).sqrt() if kind != "none" else torch.ones_like(c[..., :1])
    n = c * r
    dn = 64 * U * (r * v.abs().amax(-1, keepdim=True) + n.abs()) if kind != "none" else torch.zeros_like(n)
    y = n * w if w is not None else n
    return (y + b if b is not None else y), n, r, dn


def norm_bwd64(t, n, r, dn, w, kind, dt=0.0):
    """Gradient of a norm's input from its output's, t known to dt; -> (gradient, bound on its error)"""
    w = 1.0 if w is None else w
    u, du = t * w, dt * abs(w) if not isinstance(dt, float) else 0.0
    if kind == "none":
        return u, du + 8 * U * u.abs()
    mean = lambda v: v.mean(-1, keepdim=True)
    m1, m0 = mean(u * n), mean(u) if kind == "layer" else 0.0
    g = r * (u - m0 - n * m1)
    mag = u.abs() + mean(u.abs()) + n.abs() * mean((u * n).abs())
    err = 64 * U * mag + dn * mean((u * n).abs()) + n.abs() * mean(u.abs() * dn)
    if not isinstance(du, float):
        err = err + du + mean(du) + n.abs() * mean(du * n.abs())
    return g, r * err * (1 + 64 * U) + 64 * U * g.abs()


def rows_slack(terms, dterms):
    """Bound for a sum over all rows of `terms`, known to dterms."""
    N = terms[..., 0].numel()
    over = tuple(range(terms.dim() - 1))
    return terms.abs().sum(over) * (48 + N / 1024) * U + dterms.sum(over)


SHAPES = [(1, 1), (1, 128), (5, 3), (3, 7), (2, 3, 8), (17, 9), (4, 31), (33, 64), (2, 7, 65), (3, 5, 7, 200), (9, 257), (5, 520),
          (3, 1025), (7, 1152), (2, 1999), (3, 2049), (2, 4100), (2, 8191), (2, 8192), (4096, 16), (2500, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,affine", [("rms", "w"), ("layer", "wb"), ("layer", ""), ("rms", "wb")])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm(shape, kind, affine, dtype):
    gen = torch.Generator().manual_seed(sum(shape) + len(kind) + len(affine))
    C = shape[-1]
    x, gy = rnd(gen, *shape, dtype=dtype, mean=0.5), rnd(gen, *shape, dtype=dtype)
    w = rnd(gen, C, dtype=dtype, mean=1.0, std=0.3) if "w" in affine else None
    b = rnd(gen, C, dtype=dtype) if "b" in affine else None
    dev = lambda t: None if t is None else t.cuda().requires_grad_()
    xd, wd, bd = dev(x), dev(w), dev(b)
    y = pcb().channel_norm(xd, wd, bd, kind=kind, eps=EPS)
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = dict(zip(["x"] + ["w"] * (w is not None) + ["b"] * (b is not None), torch.autograd.grad(y, leaves, gy.cuda())))
    f = lambda t: None if t is None else t.double()
    ry, n, r, dn = norm64(f(x), f(w), f(b), kind)
    aw = 1.0 if w is None else f(w).abs()
    check(y, ry, dn * aw + 8 * U * ry.abs(), "y")
    gx, dgx = norm_bwd64(f(gy), n, r, dn, f(w), kind)
    check(grads["x"], gx, dgx, "gx")
    over = tuple(range(len(shape) - 1))
    if w is not None:
        check(grads["w"], (f(gy) * n).sum(over), rows_slack(f(gy) * n, f(gy).abs() * dn), "gw")
    if b is not None:
        check(grads["b"], f(gy).sum(over), rows_slack(f(gy), 0 * f(gy)), "gb")


def residual64(d, act, kind, next_kind, image):
    """The formulas and their errors' bounds from double tensors; -> dict of (value, bound)"""
    x, y, gate, scale, w, b, nw, nb, go, gn = (d.get(k) for k in ("x", "y", "gate", "scale", "w", "b", "nw", "nb", "go", "gn"))
    t, n, r, dn = norm64(y, w, b, kind)
    aw = 1.0 if w is None else w.abs()
    dt = dn * aw + 8 * U * (t.abs() + (0.0 if b is None else b.abs()))
    g = gate
    if gate is not None and image:
        g = gate.reshape(gate.shape[0], *[1] * (x.dim() - 2), gate.shape[1])
    if g is None:
        a, slope = torch.ones_like(x), torch.zeros_like(x)
    else:
        q = torch.sigmoid(g)
        a, slope = {"none": (g, torch.ones_like(g)), "sigmoid": (q, q * (1 - q)), "silu": (g * q, q * (1 + g * (1 - q)))}[act]
        a, slope = a.expand_as(x), slope.expand_as(x)
    da = 8 * U * a.abs()
    s = torch.ones(x.shape[-1], dtype=torch.float64) if scale is None else scale
    f = a * s
    df = da * s.abs() + 2 * U * f.abs()
    out = x + f * t
    dout = df * t.abs() + f.abs() * dt + 8 * U * (x.abs() + (f * t).abs())
    res = {"out": (out, dout)}
    gtot, dg = go, torch.zeros_like(go)
    if next_kind != "none":
        z, n2, r2, dn2 = norm64(out, nw, nb, next_kind)
        # an error of out moves the norm by at most r2 times itself and, through mean and deviation, by its mean twice
        mean = lambda v: v.mean(-1, keepdim=True)
        dn2f = dn2 + r2 * (dout + mean(dout)) + n2.abs() * r2 * mean(dout * n2.abs()) * 1.01
        anw = 1.0 if nw is None else nw.abs()
        res["next"] = (z, dn2f * anw + 8 * U * (z.abs() + (0.0 if nb is None else nb.abs())))
        # backward: out is made again, with at most the same error as before; it moves n2 and 1 / deviation in the same way
        moved = r2 * mean(dout * n2.abs()) * 1.01
        dn2b = dn2 + r2 * (dout + mean(dout)) + n2.abs() * moved
        gv, dgv = norm_bwd64(gn, n2, r2, dn2b, nw, next_kind)
        dgv = (dgv + gv.abs() * moved) * (1 + moved)
        gtot, dg = go + gv, dgv + 4 * U * (go.abs() + gv.abs())
        res["gx"] = (gtot, dg)
        over = tuple(range(x.dim() - 1))
        if nw is not None:
            res["gnw"] = ((gn * n2).sum(over), rows_slack(gn * n2, gn.abs() * dn2b))
        if nb is not None:
            res["gnb"] = (gn.sum(over), rows_slack(gn, 0 * gn))
    else:
        res["gx"] = (go, torch.zeros_like(go))
    over = tuple(range(x.dim() - 1))
    tt = gtot * f
    dtt = dg * f.abs() + gtot.abs() * df
    res["gy"] = norm_bwd64(tt, n, r, dn, w, kind, dt=dtt + 4 * U * tt.abs())
    if g is not None:
        ggf = gtot * s * slope * t
        dggf = (dg * (s * slope * t).abs() + gtot.abs() * s.abs() * (slope.abs() * dt + 16 * U * (slope.abs() + q.expand_as(x)) * (t.abs() + dt))
                + 8 * U * ggf.abs())
        if image:
            # as the kernel forms it: slope * scale * (w * sum(g n) + b * sum(g))
            mid = tuple(range(1, x.dim() - 1))
            P = max(x[0, ..., 0].numel(), 1)
            wt = (gtot * n).abs() * aw + (gtot.abs() * b.abs() if b is not None else 0.0)
            ref, bound = ggf, dggf + wt * (s * slope).abs() * (64 + P / 64) * U
            if mid:
                ref, bound = ref.sum(mid), bound.sum(mid)
            res["ggate"] = (ref, bound)
        else:
            res["ggate"] = (ggf, dggf)
    u, du = gtot * a, dg * a.abs() + gtot.abs() * da
    sum1 = rows_slack(u * n, du * n.abs() + u.abs() * dn)
    sum0 = rows_slack(u, du)
    ab = 0.0 if b is None else b.abs()
    if scale is not None:
        res["gscale"] = ((u * t).sum(over), sum1 * aw + sum0 * ab + 8 * U * ((u * n).sum(over).abs() * aw + u.sum(over).abs() * ab))
    if w is not None:
        res["gw"] = (s * (u * n).sum(over), s.abs() * sum1)
    if b is not None:
        res["gb"] = (s * u.sum(over), s.abs() * sum0)
    return res


def run_residual(d, act, kind, next_kind, dtype, gate=None):
    """The kernels' results by the same names; d: CPU tensors of `dtype`."""
    names = ["x", "y", "gate", "scale", "w", "b", "nw", "nb"]
    v = {k: d[k].cuda().requires_grad_() for k in names if d.get(k) is not None}
    if gate is not None:
        v["gate"] = gate
    out = pcb().gated_residual(v["x"], v["y"], v.get("w"), v.get("b"), v.get("gate"), v.get("scale"), kind, act, v.get("nw"), v.get("nb"),
                               next_kind, EPS)
    outs = [out] if next_kind == "none" else list(out)
    have = [k for k in names if k in v]
    grads = torch.autograd.grad(outs, [v[k] for k in have], [d["go"].cuda()] + [d["gn"].cuda()] * (next_kind != "none"))
    rename = {"x": "gx", "y": "gy", "gate": "ggate", "scale": "gscale", "w": "gw", "b": "gb", "nw": "gnw", "nb": "gnb"}
    res = {rename[k]: g for k, g in zip(have, grads)}
    res["out"] = outs[0]
    if next_kind != "none":
        res["next"] = outs[1]
    return res


def residual_data(shape, dtype, gate, scale, affine, next_affine, seed=0):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]
    d = {"x": rnd(gen, *shape, dtype=dtype, mean=0.3), "y": rnd(gen, *shape, dtype=dtype), "go": rnd(gen, *shape, dtype=dtype),
         "gn": rnd(gen, *shape, dtype=dtype)}
    if gate == "full":
        d["gate"] = rnd(gen, *shape, dtype=dtype)
    if gate == "image":
        d["gate"] = rnd(gen, shape[0], C, dtype=dtype)
    if scale:
        d["scale"] = rnd(gen, C, dtype=dtype, mean=0.3, std=0.1)
    for k, on in (("w", "w" in affine), ("b", "b" in affine), ("nw", "w" in next_affine), ("nb", "b" in next_affine)):
        if on:
            d[k] = rnd(gen, C, dtype=dtype, mean=1.0 if "w" in k else 0.0, std=0.3)
    return d


def doubles(d):
    return {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in d.items()}


# gate, activation, kind, affine, next, its affine, scale
FORMS = [("none", "none", "none", "", "none", "", False), ("none", "none", "rms", "w", "none", "", True),
         ("image", "none", "layer", "wb", "rms", "w", True), ("image", "silu", "none", "", "layer", "wb", True),
         ("image", "sigmoid", "rms", "wb", "none", "", False), ("full", "silu", "layer", "wb", "rms", "w", True),
         ("full", "none", "rms", "w", "layer", "wb", False), ("full", "sigmoid", "none", "wb", "layer", "", True)]
RESIDUAL_SHAPES = [(1, 1, 1), (1, 5, 8), (2, 3, 7), (3, 5, 9), (2, 4, 4, 64), (5, 1, 72), (3, 7, 9, 200), (2, 19, 201), (2, 3, 520),
                   (2, 3, 1152), (2, 2, 1601), (1, 3, 4096), (2, 1, 8192), (2, 1031, 48), (3000, 2, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(v) for v in f))
@pytest.mark.parametrize("shape", RESIDUAL_SHAPES, ids=str)
def test_residual(shape, form, dtype):
    gate, act, kind, affine, next_kind, next_affine, scale = form
    d = residual_data(shape, dtype, gate, scale, affine, next_affine)
    got = run_residual(d, act, kind, next_kind, dtype)
    ref = residual64(doubles(d), act, kind, next_kind, gate == "image")
    assert set(got) == set(ref)
    for k, (value, bound) in ref.items():
        check(got[k], value, bound, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gate_from_a_slice_and_tensors_at_odd_addresses(dtype):
    """The gate as a slice of a wider projection (read where it lies), everything else at storage offsets that are no multiple of
    16 bytes: bitwise the result of dense aligned tensors."""
    d = residual_data((2, 5, 7, 48), dtype, "full", True, "wb", "wb")
    base = run_residual(d, "silu", "layer", "rms", dtype)
    wide = torch.randn(2, 5, 7, 150, device="cuda").to(dtype)
    wide[..., 51:99] = d["gate"].cuda()
    wide.requires_grad_()
    names = ["x", "y", "scale", "w", "b", "nw", "nb"]
    v = {}
    for k in names:
        store = torch.empty(d[k].numel() + 3, dtype=dtype, device="cuda")
        v[k] = store[3:].view(d[k].shape).copy_(d[k]).requires_grad_()
        assert v[k].data_ptr() % 16 != 0
    out = pcb().gated_residual(v["x"], v["y"], v["w"], v["b"], wide[..., 51:99], v["scale"], "layer", "silu", v["nw"], v["nb"], "rms", EPS)
    grads = torch.autograd.grad(out, [wide] + [v[k] for k in names], [d["go"].cuda(), d["gn"].cuda()])
    assert torch.equal(out[0], base["out"]) and torch.equal(out[1], base["next"])
    assert torch.equal(grads[0][..., 51:99], base["ggate"]) and not grads[0][..., :51].any() and not grads[0][..., 99:].any()
    for g, k in zip(grads[1:], ["gx", "gy", "gscale", "gw", "gb", "gnw", "gnb"]):
        assert torch.equal(g, base[k]), k


def test_gradients_against_differences():
    """Directional differences of the formula in 64 bits against the kernels' gradients.  With steps of h = 1e-4 the quotient is off by
    h^2 / 6 of a third derivative of order one and 1e-16 / h of the loss, a gradient's product with a direction by 1e-5 of the
    products' magnitudes (the bounds above at these sizes)."""
    shape, act, kind, next_kind = (2, 3, 3, 24), "silu", "layer", "rms"
    d = residual_data(shape, torch.float32, "image", True, "wb", "w")
    got = run_residual(d, act, kind, next_kind, torch.float32)
    dd = doubles(d)

    def loss(v):
        r = residual64(v, act, kind, next_kind, True)
        return float((r["out"][0] * dd["go"]).sum() + (r["next"][0] * dd["gn"]).sum())

    gen = torch.Generator().manual_seed(5)
    for k, g in (("x", "gx"), ("y", "gy"), ("gate", "ggate"), ("scale", "gscale"), ("w", "gw"), ("b", "gb"), ("nw", "gnw")):
        direction = torch.randn(dd[k].shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        quotient = (loss({**dd, k: dd[k] + h * direction}) - loss({**dd, k: dd[k] - h * direction})) / (2 * h)
        prods = got[g].double().cpu() * direction
        assert abs(quotient - float(prods.sum())) <= 1e-5 * float(prods.abs().sum()) + 1e-5, k


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 values: the last rows are bitwise those of a call on them alone; the weights' gradients are theirs, since
    every other row's is zero."""
    N, C, last = (1 << 31) // 4096 + 1000, 4096, 64
    x = torch.zeros(N, C, device="cuda", dtype=torch.bfloat16)
    gy = torch.zeros_like(x)
    gen = torch.Generator().manual_seed(2)
    xl, gl = rnd(gen, last, C, dtype=torch.bfloat16).cuda(), rnd(gen, last, C, dtype=torch.bfloat16).cuda()
    x[-last:], gy[-last:] = xl, gl
    w, b = rnd(gen, C, dtype=torch.bfloat16, mean=1.0, std=0.2).cuda().requires_grad_(), rnd(gen, C, dtype=torch.bfloat16).cuda().requires_grad_()
    assert x.numel() > 1 << 31
    x.requires_grad_(), xl.requires_grad_()
    y, yl = pcb().channel_norm(x, w, b, kind="layer"), pcb().channel_norm(xl, w, b, kind="layer")
    assert torch.equal(y[-last:], yl) and torch.equal(y[0], b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], gy)
    gxl, gwl, gbl = torch.autograd.grad(yl, [xl, w, b], gl)
    assert torch.equal(gx[-last:], gxl) and not gx[:-last].any()
    n = norm64(xl.detach().double().cpu(), None, None, "layer")
    check(gw, (gl.double().cpu() * n[1]).sum(0), rows_slack(gl.double().cpu() * n[1], gl.double().cpu().abs() * n[3]), "gw")
    check(gb, gl.double().cpu().sum(0), rows_slack(gl.double().cpu(), 0 * gl.double().cpu()), "gb")
    del y, gx
    out = pcb().gated_residual(x, x, w, b, scale=w, kind="layer")
    outl = pcb().gated_residual(xl, xl, w, b, scale=w, kind="layer")
    assert torch.equal(out[-last:], outl)


def test_constant_rows_and_large_offsets():
    """Rows without variance: the layer norm is its bias exactly as far as the mean is exact; rows far from zero keep their variance
    (it is taken from centred values)."""
    x = torch.full((3, 64), 2.5)
    x[1] = 0
    b = torch.randn(64)
    y = pcb().channel_norm(x.cuda(), None, b.cuda(), kind="layer", eps=EPS)
    check(y, b.double().expand(3, 64), torch.zeros(3, 64, dtype=torch.float64), "bias")
    y = pcb().channel_norm(torch.zeros(2, 100, device="cuda"), kind="rms")
    assert not y.any()
    gen = torch.Generator().manual_seed(1)
    far = (rnd(gen, 4, 256, std=1.0) + 4096.0)
    ref, n, r, dn = norm64(far.double(), None, None, "layer")
    got = pcb().channel_norm(far.cuda(), kind="layer", eps=EPS)
    check(got, ref, dn, "far from zero")
    assert float(dn.max()) < 0.05   # (a difference of squares would have lost everything: 4096^2 u is the variance itself)


def test_nonfinite_rows_stay_to_themselves():
    x = torch.randn(40, 72, device="cuda")
    ref = pcb().channel_norm(x, kind="rms")
    x2 = x.clone()
    x2[7, 3], x2[20, 71] = float("nan"), float("inf")
    got = pcb().channel_norm(x2, kind="rms")
    rows = torch.ones(40, dtype=torch.bool)
    rows[[7, 20]] = False
    assert torch.equal(got[rows], ref[rows]) and got[7].isnan().all()


def test_only_some_gradients_and_only_one_output():
    """Each leaf's gradient by itself is bitwise what it is among all; an output without a gradient counts as zero."""
    for gate in ("image", "full"):
        d = residual_data((2, 6, 40), torch.float32, gate, True, "wb", "wb")
        base = run_residual(d, "sigmoid", "layer", "layer", torch.float32)
        names = {"x": "gx", "y": "gy", "gate": "ggate", "scale": "gscale", "w": "gw", "b": "gb", "nw": "gnw", "nb": "gnb"}
        for k in names:
            v = {n: d[n].cuda() for n in names}
            v[k].requires_grad_()
            out = pcb().gated_residual(v["x"], v["y"], v["w"], v["b"], v["gate"], v["scale"], "layer", "sigmoid", v["nw"], v["nb"],
                                       "layer", EPS)
            (g,) = torch.autograd.grad(out, [v[k]], [d["go"].cuda(), d["gn"].cuda()])
            assert torch.equal(g, base[names[k]]), (gate, k)
        zero = torch.zeros_like(d["go"])
        for which in (0, 1):
            z = dict(d)
            z["go" if which else "gn"] = zero
            ref = run_residual(z, "sigmoid", "layer", "layer", torch.float32)
            v = {n: d[n].cuda().requires_grad_() for n in names}
            out = pcb().gated_residual(v["x"], v["y"], v["w"], v["b"], v["gate"], v["scale"], "layer", "sigmoid", v["nw"], v["nb"],
                                       "layer", EPS)
            grads = torch.autograd.grad(out[which], list(v.values()), d["gn" if which else "go"].cuda(), allow_unused=True)
            for n, g in zip(names, grads):
                assert torch.equal(g, ref[names[n]]), (gate, which, n)


def test_no_rows():
    for shape in ((0, 16), (2, 0, 16), (0, 3, 16)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(16, device="cuda", requires_grad=True)
        y = pcb().channel_norm(x, w, w, kind="layer")
        y.sum().backward()
        assert y.shape == shape and x.grad.shape == shape and not w.grad.any()
        gate = torch.ones(shape[0], 16, device="cuda", requires_grad=True)
        out, nxt = pcb().gated_residual(x, x, w, w, gate, w, "rms", "silu", w, w, "layer")
        w.grad = None
        (out.sum() + nxt.sum()).backward()
        assert out.shape == nxt.shape == shape and not w.grad.any() and not gate.grad.any() and w.grad.isfinite().all()


def test_composition_is_the_separate_calls():
    """out is bitwise the call without a next norm; next is within a rounding of out of the norm of the stored out."""
    d = residual_data((2, 9, 9, 96), torch.bfloat16, "image", True, "w", "w")
    both = run_residual(d, "none", "rms", "rms", torch.bfloat16)
    alone = pcb().gated_residual(d["x"].cuda(), d["y"].cuda(), d["w"].cuda(), None, d["gate"].cuda(), d["scale"].cuda(), "rms", eps=EPS)
    assert torch.equal(both["out"], alone)
    z = pcb().channel_norm(alone, d["nw"].cuda(), kind="rms", eps=EPS)
    # out is stored to half a step; the norm moves by that, its own mean square by as much again, and is rounded once itself
    assert ((z.double() - both["next"].double()).abs() <= 4 * torch.finfo(torch.bfloat16).eps * (z.double().abs() + 1e-3)).all()


def test_other_stream_and_repeatability():
    d = residual_data((8, 50, 128), torch.bfloat16, "image", True, "wb", "w")
    base = run_residual(d, "silu", "layer", "rms", torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run_residual(d, "silu", "layer", "rms", torch.bfloat16)
    side.synchronize()
    for k in base:
        assert torch.equal(base[k], again[k]), k


def test_no_second_derivative_and_function_form():
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(pcb().channel_norm(x, w).sum(), x, create_graph=True)
    out, nxt = pcb().gated_residual(x, x * 2, w, scale=w, kind="rms", next_weight=w, next_kind="layer")
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out.sum() + nxt.sum(), x, create_graph=True)
    # the form that a trace records gives the same
    y = pcb().channel_norm(x, w, w, kind="layer")
    f = pcb().ChannelNormFunction.apply(x, w, w, 2, 1e-6)
    g = torch.randn_like(y)
    assert torch.equal(y, f)
    for a, b in zip(torch.autograd.grad(y, [x, w], g), torch.autograd.grad(f, [x, w], g)):
        assert torch.equal(a, b)
    gate = torch.randn(4, 16, device="cuda", requires_grad=True)
    pair = pcb().gated_residual(x, x, w, w, gate, w, "layer", "silu", w, None, "rms")
    pair_f = pcb().GatedResidualFunction.apply(x, x, gate, w, w, w, w, None, 2, 2, 1, 1e-6)
    gn = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(pair, [x, w, gate], [g, gn]), torch.autograd.grad(pair_f, [x, w, gate], [g, gn])):
        assert torch.equal(a, b)


def test_checkpointed_and_transformed_calls():
    """Under activation checkpointing the same bits; forward-mode derivatives and batching are refused, not left out."""
    from torch.utils.checkpoint import checkpoint

    x, gate = torch.randn(3, 5, 24, device="cuda", requires_grad=True), torch.randn(3, 24, device="cuda", requires_grad=True)
    w = torch.rand(24, device="cuda", requires_grad=True)

    def f(x, gate, w):
        z = pcb().channel_norm(x, w, kind="layer")
        y, last = pcb().gated_scan(z, z * 2)
        out, nxt = pcb().gated_residual(x, y, w, gate=gate, kind="rms", activation="silu", next_weight=w, next_kind="layer")
        return out.sum() + nxt.square().sum() + last.sum()

    plain = torch.autograd.grad(f(x, gate, w), [x, gate, w])
    kept = torch.autograd.grad(checkpoint(f, x, gate, w, use_reentrant=False), [x, gate, w])
    for a, b in zip(plain, kept):
        assert torch.equal(a, b)
    for call in (lambda t: pcb().channel_norm(t), lambda t: pcb().gated_residual(t, t, kind="rms"), lambda t: pcb().gated_scan(t, t)[0]):
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x.detach(),), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x.detach()[None])


def test_saved_tensor_changed_in_place_is_noticed():
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    y = torch.randn(4, 16, device="cuda", requires_grad=True)
    b = y * 1.0
    out = pcb().gated_residual(x, b, kind="rms")
    b.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_captured_step_replays():
    """Forward and backward of norm -> residual with its next norm in a graph: every replay, with eager work between, is the eager
    result on the same inputs."""
    dtype = torch.bfloat16
    gen = torch.Generator().manual_seed(3)
    C = 128
    x = rnd(gen, 4, 14, 14, C, dtype=dtype).cuda().requires_grad_()
    gate = rnd(gen, 4, C, dtype=dtype).cuda().requires_grad_()
    params = [rnd(gen, C, dtype=dtype, mean=1.0, std=0.1).cuda().requires_grad_() for _ in range(4)]
    go, gn = rnd(gen, 4, 14, 14, C, dtype=dtype).cuda(), rnd(gen, 4, 14, 14, C, dtype=dtype).cuda()

    def step():
        z = pcb().channel_norm(x, params[0])
        out, nxt = pcb().gated_residual(x, z * 2, params[1], gate=gate, scale=params[2], kind="layer", activation="silu",
                                        next_weight=params[3], next_kind="rms")
        return [out.detach(), nxt.detach(), *torch.autograd.grad([out, nxt], [x, gate, *params], [go, gn])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in range(4):
        g2 = torch.Generator().manual_seed(100 + seed)
        with torch.no_grad():
            x.copy_(rnd(g2, *x.shape, dtype=dtype))
            gate.copy_(rnd(g2, *gate.shape, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in res]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("gated", [False, True])
def test_stack_of_blocks(gated):
    """ResidualConvStack: bitwise its own steps called one by one, and gradients for every parameter."""
    torch.manual_seed(0)
    stack = pcb().ResidualConvStack(64, depth=2, kernel_size=7, init_scale=0.5).to(torch.bfloat16).cuda()
    x = torch.randn(2, 16, 16, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    gate = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16) if gated else None
    out, z = stack(x, gate)
    (out.float().square().mean() + z.float().square().mean()).backward()
    for name, p in stack.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.abs().sum() > 0, name
    assert x.grad.isfinite().all()
    with torch.no_grad():
        h, n = x, pcb().channel_norm(x, stack.norms[0].weight)
        for i in range(2):
            r = stack.residuals[i]
            h, n = pcb().gated_residual(h, stack.blocks[i](n), r.weight, None, None if gate is None else gate[i], r.scale, "rms",
                                        next_weight=stack.norms[i + 1].weight, next_kind="rms")
        eager = stack(x.detach(), gate)
    assert torch.equal(eager[0], h) and torch.equal(eager[1], n)
