"""gated_scan and gated_scan_step against the recurrence step by step in 64 bits, on identically rounded inputs.

Bounds, element by element: half a step of the type for the one rounding of a result, and before it what 32 bits lose, u = 2^-24 a
rounding.  a and 1 - a are good to 4 u.  A step's h is off by a times what the last one was off by and some roundings of a h and m x;
composed in pieces a state takes at most as many roundings again for its place in lanes, wavefronts and segments (each a product
and a sum): 16 u (a |h| + m |x|) a step.  The bounds run through the same recurrence.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def pcb():
    import pyramidconvblock_amd

    return pyramidconvblock_amd


def check(got, ref, slack, what):
    """|got - ref| <= half a step + slack, everywhere"""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    dtype = got.dtype
    got = got.detach().double().cpu()
    bound = torch.finfo(dtype).eps / 2 * (ref.abs() + slack) + slack + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - ref).abs() / bound).nan_to_num(9e9).max()):.2f} of the bound"


def reference(x, g, state, lengths, dim, reverse, gy=None, glast=None):
    """Double tensors -> dict of (value, bound); dim >= 0."""
    x, g = x.movedim(dim, 0), g.movedim(dim, 0)
    T = x.shape[0]
    a, m = torch.sigmoid(g), torch.sigmoid(-g)
    h = state.clone() if state is not None else torch.zeros(x.shape[1:], dtype=torch.float64)
    lens = torch.full(x.shape[1:], T) if lengths is None else lengths.long().clamp(0, T).reshape(
        lengths.shape + (1,) * (x.dim() - 1 - lengths.dim())).expand(x.shape[1:])
    eh = torch.zeros_like(h)
    y, ey, hp, ehp = (torch.zeros_like(x) for _ in range(4))
    order = range(T - 1, -1, -1) if reverse else range(T)
    for t in order:
        on = t < lens
        hp[t], ehp[t] = h, eh
        xt = torch.where(on, x[t], 0.0)
        e = a[t] * eh + 16 * U * (a[t] * h.abs() + m[t] * xt.abs())
        h, eh = torch.where(on, a[t] * h + m[t] * xt, h), torch.where(on, e, eh)
        y[t], ey[t] = torch.where(on, h, 0.0), torch.where(on, eh, 0.0)
    res = {"y": (y.movedim(0, dim), ey.movedim(0, dim)), "last": (h, eh)}
    if gy is None:
        return res
    gy = gy.movedim(dim, 0)
    e, ee = glast.clone(), torch.zeros_like(glast)
    gx, ex, gg, eg = (torch.zeros_like(x) for _ in range(4))
    for t in reversed(order):
        on = t < lens
        xt = torch.where(on, x[t], 0.0)
        d = torch.where(on, gy[t], 0.0) + e
        # (what the sum's terms lose counts, not what is left of it)
        mag = torch.where(on, gy[t], 0.0).abs() + e.abs()
        ed = ee + 2 * U * mag
        s = a[t] * m[t]
        gx[t], ex[t] = torch.where(on, d * m[t], 0.0), torch.where(on, ed * m[t] + 16 * U * m[t] * mag, 0.0)
        gg[t] = torch.where(on, d * (hp[t] - xt) * s, 0.0)
        eg[t] = torch.where(on, (ed * (hp[t] - xt).abs() + d.abs() * ehp[t] + 16 * U * mag * (hp[t].abs() + xt.abs())) * s, 0.0)
        e, ee = torch.where(on, a[t] * d, e), torch.where(on, a[t] * ed + 16 * U * a[t] * mag, ee)
    return {**res, "gx": (gx.movedim(0, dim), ex.movedim(0, dim)), "gg": (gg.movedim(0, dim), eg.movedim(0, dim)), "gstate": (e, ee)}


def data(shape, dim, dtype, state=True, lengths=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s, mean=0.0, std=1.0, dt=dtype: (torch.randn(*s, generator=gen, dtype=torch.float64) * std + mean).to(dt)
    carried = shape[:dim] + shape[dim + 1:]
    d = {"x": rnd(*shape), "g": rnd(*shape, mean=2.0, std=2.0), "gy": rnd(*shape), "glast": rnd(*carried, dt=torch.float32),
         "state": rnd(*carried, dt=torch.float32) if state else None, "lengths": None}
    if lengths:
        T = shape[dim]
        n = torch.randint(0, T + 1, shape[:dim], generator=gen, dtype=torch.int32).reshape(-1)
        edge = torch.tensor([0, T, 1, max(T - 1, 0)], dtype=torch.int32)[:n.numel()]
        n[:edge.numel()] = edge
        d["lengths"] = n.reshape(shape[:dim])
    return d


def run(d, dim, reverse, packed=False):
    cuda = lambda t: None if t is None else t.cuda()
    x, g, state, lengths = (cuda(d[k]) for k in ("x", "g", "state", "lengths"))
    leaves = [torch.cat([x, g], -1)] if packed else [x, g]
    leaves += [state] if state is not None else []
    for t in leaves:
        t.requires_grad_()
    y, last = pcb().gated_scan(leaves[0], None if packed else g, state, lengths, dim, reverse)
    grads = list(torch.autograd.grad([y, last], leaves, [cuda(d["gy"]), cuda(d["glast"])]))
    if packed:
        grads[:1] = grads[0].chunk(2, -1)
    res = {"y": y, "last": last, "gx": grads[0], "gg": grads[1]}
    if state is not None:
        res["gstate"] = grads[2]
    return res


def compare(d, got, dim, reverse):
    f = lambda t: None if t is None else t.double()
    ref = reference(f(d["x"]), f(d["g"]), f(d["state"]), d["lengths"], dim, reverse, f(d["gy"]), f(d["glast"]))
    for k, v in got.items():
        check(v, *ref[k], k)


# chains of one step to several tiles and segments; channels that fill strips and that do not; axes before, between and behind others
SHAPES = [((1, 1, 1), 1), ((2, 1, 8), 1), ((3, 2, 3), 1), ((2, 5, 64), 1), ((1, 33, 5), 1), ((4, 16, 66), 1), ((2, 65, 130), 1),
          ((2, 129, 20), 1), ((1, 257, 67), 1), ((3, 600, 24), 1), ((1, 3001, 65), 1), ((2, 1500, 2), 1), ((1, 5000, 1), 1), ((17, 9), 0), ((300, 7), 0),
          ((2, 9, 11, 24), 1), ((2, 9, 11, 24), 2), ((2, 3, 40, 5, 6), 2), ((300, 40, 16), 1), ((130, 300, 130), 1),
          ((32, 2100, 100), 1), ((20, 1500, 200), 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shape,dim", SHAPES, ids=str)
def test_scan(shape, dim, reverse, dtype):
    d = data(shape, dim, dtype, state=sum(shape) % 2 == 0, lengths=False)
    compare(d, run(d, dim, reverse), dim, reverse)


# many chains: a lane has six, seven or eight steps of a tile, so that the last tile is nearly full; at the ends of such tiles, before and behind
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("batch,channels,steps", [(210, 5, t) for t in (12, 13, 15, 28, 33, 49, 57, 96, 129, 193, 225, 257, 385, 449, 513, 769, 897, 1793)]
                         + [(130, 20, t) for t in (33, 49, 57, 65, 97, 113, 129, 192, 224, 257, 384, 449, 785)])
def test_many_chains(batch, channels, steps, reverse, dtype):
    d = data((batch, steps, channels), 1, dtype, lengths=True, seed=steps)
    compare(d, run(d, 1, reverse), 1, reverse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shape,dim", [((6, 40, 24), 1), ((5, 300, 10), 1), ((4, 2000, 70), 1), ((3, 4, 50, 8), 2), ((3, 50, 4, 8), 1), ((6, 3, 2), 1), ((33, 1300, 98), 1)],
                         ids=str)
def test_lengths_leave_the_rest_alone(shape, dim, reverse, dtype):
    """Lengths of 0, 1, T - 1, T and between, what lies behind them NaN and infinities in x, g and gy: not read, and 0 in results."""
    d = data(shape, dim, dtype, lengths=True)
    lens = d["lengths"].long().reshape(d["lengths"].shape + (1,) * (len(shape) - dim))
    pos = torch.arange(shape[dim]).reshape((-1,) + (1,) * (len(shape) - dim - 1))
    off = (pos >= lens).expand(shape)
    dirty = dict(d)
    for k, v in (("x", float("nan")), ("g", float("inf")), ("gy", float("-inf"))):
        dirty[k] = torch.where(off, torch.tensor(v, dtype=dtype), d[k])
    got = run(dirty, dim, reverse)
    for k in ("y", "gx", "gg"):
        assert not got[k][off.cuda()].any(), k
    compare(d, got, dim, reverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,dim", [((2, 70, 24), 1), ((2, 9, 11, 10), 1), ((2, 9, 11, 10), 2), ((1, 1000, 64), 1), ((2, 2, 3), 1)], ids=str)
def test_halves_of_one_tensor(shape, dim, dtype):
    """x and g in one tensor: bitwise the separate tensors' results, and one gradient for both."""
    d = data(shape, dim, dtype, lengths=True)
    a, b = run(d, dim, True), run(d, dim, True, packed=True)
    for k in ("y", "last", "gstate"):
        assert torch.equal(a[k], b[k]), k
    for k in ("gx", "gg"):
        assert torch.equal(a[k], b[k]), k


def test_slices_transposes_and_odd_addresses():
    d = data((3, 80, 24), 1, torch.bfloat16)
    base = run(d, 1, False)
    wide = torch.randn(3, 80, 101, device="cuda").bfloat16()
    wide[..., 5:29], wide[..., 60:84] = d["x"].cuda(), d["g"].cuda()
    wide.requires_grad_()
    state = d["state"].cuda().requires_grad_()
    y, last = pcb().gated_scan(wide[..., 5:29], wide[..., 60:84], state)
    gw, gs = torch.autograd.grad([y, last], [wide, state], [d["gy"].cuda(), d["glast"].cuda()])
    assert torch.equal(y, base["y"]) and torch.equal(last, base["last"]) and torch.equal(gs, base["gstate"])
    assert torch.equal(gw[..., 5:29], base["gx"]) and torch.equal(gw[..., 60:84], base["gg"])
    # time first in memory, channels first in memory: strides that are read as they are, and ones that are not
    for perm, back in (((1, 0, 2), (1, 0, 2)), ((2, 0, 1), (1, 2, 0))):
        x = d["x"].permute(*perm).contiguous().cuda().permute(*back).requires_grad_()
        g = d["g"].permute(*perm).contiguous().cuda().permute(*back)
        assert x.shape == (3, 80, 24) and not x.is_contiguous()
        y, last = pcb().gated_scan(x, g, d["state"].cuda())
        (gx,) = torch.autograd.grad([y, last], [x], [d["gy"].cuda(), d["glast"].cuda()])
        assert torch.equal(y, base["y"]) and torch.equal(gx, base["gx"])
    # a broadcast x and a broadcast gradient
    x = d["x"][:1, :, :1].cuda().requires_grad_()
    y, last = pcb().gated_scan(x.expand(3, 80, 24), d["g"].cuda())
    y2, _ = pcb().gated_scan(x.expand(3, 80, 24).contiguous(), d["g"].cuda())
    assert torch.equal(y, y2)
    y.sum().backward()
    assert x.grad.shape == x.shape and x.grad.isfinite().all()


@pytest.mark.parametrize("shape,dim,expand", [((3, 4, 50, 8), 2, (0,)), ((3, 4, 50, 8), 2, (1,)), ((3, 4, 50, 8), 2, (0, 1)), ((3, 50, 4, 5, 8), 1, (3,)),
                                              ((3, 50, 4, 5, 8), 1, (2,)), ((3, 50, 4, 8), 1, (1,)), ((3, 50, 4, 8), 1, (0, 2))], ids=str)
def test_expanded_dimensions(shape, dim, expand):
    """Inputs that repeat along some dimensions (strides of zero): bitwise the results of their dense copies, gradients summed."""
    d = data(shape, dim, torch.float32)
    index = tuple(slice(0, 1) if i in expand else slice(None) for i in range(len(shape)))
    small = d["x"][index].cuda().requires_grad_()
    g, state, gy, glast = (d[k].cuda() for k in ("g", "state", "gy", "glast"))
    y, last = pcb().gated_scan(small.expand(shape), g, state, dim=dim)
    (gs,) = torch.autograd.grad([y, last], [small], [gy, glast])
    dense = small.detach().expand(shape).contiguous().requires_grad_()
    y2, last2 = pcb().gated_scan(dense, g, state, dim=dim)
    (gd,) = torch.autograd.grad([y2, last2], [dense], [gy, glast])
    assert torch.equal(y, y2) and torch.equal(last, last2)
    assert torch.equal(gs, gd.sum(expand, keepdim=True))


def test_saved_tensors_that_come_back_in_another_layout():
    """Saved-tensor hooks that move tensors to the host and back lay strided ones out anew: the gradients stay as they are."""
    d = data((2, 40, 6, 8), 1, torch.float32)
    wide = torch.cat([d["x"], d["g"]], -1).cuda().requires_grad_()
    turned = d["x"].transpose(1, 2).contiguous().cuda().transpose(1, 2)   # the other way round: dense in no order of its own

    def grads(hooks):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.cuda()) if hooks else torch.enable_grad():
            y, last = pcb().gated_scan(wide, dim=1)
            z, _ = pcb().gated_scan(turned.requires_grad_(), wide[..., 8:], dim=1)
            x = d["x"].cuda().requires_grad_()
            v, _ = pcb().gated_scan(x, d["g"].cuda(), dim=1)
        return torch.autograd.grad([y, z, v], [wide, turned, x], [d["gy"].cuda()] * 3)

    for a, b in zip(grads(False), grads(True)):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """More than 2^31 values, and a step of more than 2^21 values between positions: the results of dense small tensors (the second bitwise;
    the first is cut otherwise, so its states differ by up to 64 u of the largest, as many roundings as a state has on its way; two
    results of bfloat16 that are each half a step, 2^-8 of the value, off the state they round differ by up to 2^-7 of it more)."""
    O, T, C = 3, 360000, 2000
    x = torch.zeros(O, T, C, device="cuda", dtype=torch.bfloat16)
    g = torch.full_like(x, 2.0)
    gen = torch.Generator().manual_seed(4)
    xl = torch.randn(1, T, 8, generator=gen).bfloat16().cuda()
    x[2:, :, -8:] = xl
    assert x.numel() > 1 << 31
    x.requires_grad_()
    y, last = pcb().gated_scan(x, g)
    a = xl.clone().requires_grad_()
    yl, lastl = pcb().gated_scan(a, g[2:, :, -8:])
    assert ((y[2:, :, -8:].float() - yl.float()).abs() <= 2.0 ** -7 * yl.float().abs() + 64 * U * 5).all()
    assert ((last[2:, -8:] - lastl).abs() <= 64 * U * 5).all() and not y[:2].any()
    gy = torch.zeros_like(x)
    gy[2:, :, -8:] = xl
    (gx,), (gl,) = torch.autograd.grad(y, [x], gy), torch.autograd.grad(yl, [a], xl)
    assert ((gx[2:, :, -8:].float() - gl.float()).abs() <= 2.0 ** -7 * gl.float().abs() + 64 * U * 5).all() and not gx[:2].any()
    del x, g, y, gy, gx, last

    wide = torch.empty(1, 700, 3 << 20, device="cuda", dtype=torch.bfloat16)
    d = data((1, 700, 8), 1, torch.bfloat16)
    base = run(d, 1, True)
    x, g = wide[..., 5:13], wide[..., -9:-1]
    x.copy_(d["x"]), g.copy_(d["g"])
    x, g, state = x.detach().requires_grad_(), g.detach().requires_grad_(), d["state"].cuda().requires_grad_()
    assert x.stride(1) > 1 << 21
    y, last = pcb().gated_scan(x, g, state, reverse=True)
    grads = torch.autograd.grad([y, last], [x, g, state], [d["gy"].cuda(), d["glast"].cuda()])
    for t, k in zip((y, last, *grads), ("y", "last", "gx", "gg", "gstate")):
        assert torch.equal(t, base[k]), k


def test_extreme_gates():
    """a = 1 holds the state, a = 0 takes the input, exactly, and their gradients are finite."""
    x = torch.randn(2, 200, 16)
    state = torch.randn(2, 16)
    for v, want in ((float("inf"), None), (200.0, None), (float("-inf"), "x"), (-200.0, "x")):
        g = torch.full_like(x, v).cuda().requires_grad_()
        xd = x.cuda().requires_grad_()
        y, last = pcb().gated_scan(xd, g, state.cuda())
        assert torch.equal(y.cpu(), x if want else state[:, None].expand(2, 200, 16)), v
        gx, gg = torch.autograd.grad([y], [xd, g], torch.ones_like(y))
        assert torch.equal(gx, torch.ones_like(gx) if want else torch.zeros_like(gx)) and gg.isfinite().all(), v


def test_channels_do_not_mix():
    d = data((2, 300, 70), 1, torch.float32)
    base = run(d, 1, False)
    d["x"][1, 100, 33] = float("nan")
    got = run(d, 1, False)
    same = torch.ones(2, 70, dtype=torch.bool)
    same[1, 33] = False
    for k in ("y", "gx", "gg"):
        assert torch.equal(got[k].movedim(1, 2)[same], base[k].movedim(1, 2)[same]), k
    assert torch.equal(got["y"][:, :100], base["y"][:, :100]) and got["y"][1, 100:, 33].isnan().all()


def test_no_steps_and_no_chains():
    state = torch.randn(3, 8, device="cuda", requires_grad=True)
    x = torch.empty(3, 0, 8, device="cuda", requires_grad=True)
    y, last = pcb().gated_scan(x, x, state)
    assert y.shape == (3, 0, 8) and torch.equal(last, state)
    g = torch.randn_like(last)
    gs, gx = torch.autograd.grad(last, [state, x], g)
    assert torch.equal(gs, g) and gx.shape == x.shape
    y, last = pcb().gated_scan(x, x)
    assert not last.any()
    for shape in ((0, 5, 8), (2, 5, 0)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y, last = pcb().gated_scan(x, x)
        (y.sum() + last.sum()).backward()
        assert y.shape == shape and x.grad.shape == shape


def test_lengths_out_of_range_are_limited():
    d = data((3, 50, 8), 1, torch.float32)
    d["lengths"] = torch.tensor([-5, 1 << 30, 50], dtype=torch.int32)
    got = run(d, 1, False)
    d["lengths"] = torch.tensor([0, 50, 50], dtype=torch.int32)
    for k, v in run(d, 1, False).items():
        assert torch.equal(v, got[k]), k


def test_gradients_against_differences():
    """Directional differences of the recurrence in 64 bits against the kernels' gradients: h^2 / 6 of a third derivative of order ten
    (h = 1e-4) and 1e-16 / h of the loss, a gradient's product with a direction by 1e-5 of the products' magnitudes."""
    d = data((2, 40, 6), 1, torch.float32)
    got = run(d, 1, True)
    dd = {k: v.double() for k, v in d.items() if v is not None}

    def loss(v):
        r = reference(v["x"], v["g"], v["state"], None, 1, True)
        return float((r["y"][0] * dd["gy"]).sum() + (r["last"][0] * dd["glast"]).sum())

    gen = torch.Generator().manual_seed(5)
    for k, g in (("x", "gx"), ("g", "gg"), ("state", "gstate")):
        direction = torch.randn(dd[k].shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        quotient = (loss({**dd, k: dd[k] + h * direction}) - loss({**dd, k: dd[k] - h * direction})) / (2 * h)
        prods = got[g].double().cpu() * direction
        assert abs(quotient - float(prods.sum())) <= 1e-5 * float(prods.abs().sum()) + 1e-5, k


def test_only_some_gradients_and_only_one_output():
    d = data((2, 400, 40), 1, torch.float32)
    base = run(d, 1, False)
    names = {"x": "gx", "g": "gg", "state": "gstate"}
    for k in names:
        v = {n: d[n].cuda() for n in names}
        v[k].requires_grad_()
        out = pcb().gated_scan(v["x"], v["g"], v["state"])
        (g,) = torch.autograd.grad(out, [v[k]], [d["gy"].cuda(), d["glast"].cuda()])
        assert torch.equal(g, base[names[k]]), k
    for which in (0, 1):
        z = dict(d)
        z["glast" if which == 0 else "gy"] = torch.zeros_like(d["glast" if which == 0 else "gy"])
        ref = run(z, 1, False)
        v = {n: d[n].cuda().requires_grad_() for n in names}
        out = pcb().gated_scan(v["x"], v["g"], v["state"])
        grads = torch.autograd.grad(out[which], list(v.values()), d["gy" if which == 0 else "glast"].cuda())
        for n, g in zip(names, grads):
            assert torch.equal(g, ref[names[n]]), (which, n)


def test_pieces_of_a_sequence():
    """A sequence in pieces, each from the state that the one before left, and token by token: the whole, within both bounds."""
    d = data((2, 700, 48), 1, torch.float32)
    f = lambda t: t.double()
    ref = reference(f(d["x"]), f(d["g"]), f(d["state"]), None, 1, False)
    x, g, h = d["x"].cuda(), d["g"].cuda(), d["state"].cuda()
    ys = []
    for a, b in ((0, 1), (1, 301), (301, 698)):
        y, h = pcb().gated_scan(x[:, a:b], g[:, a:b], h)
        ys.append(y)
    for t in (698, 699):
        y, h2 = pcb().gated_scan_step(x[:, t], g[:, t], h)
        assert h2 is h
        ys.append(y[:, None])
    check(torch.cat(ys, 1), *ref["y"], "y")
    check(h, *ref["last"], "last")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 130), (256, 1152), (2, 3, 36), (0, 8), (4, 0)], ids=str)
def test_step(shape, dtype):
    gen = torch.Generator().manual_seed(sum(shape))
    x, g = torch.randn(*shape, generator=gen).to(dtype), (torch.randn(*shape, generator=gen) * 2 + 2).to(dtype)
    h = torch.randn(*shape, generator=gen)
    a, m = torch.sigmoid(g.double()), torch.sigmoid(-g.double())
    ref = a * h.double() + m * x.double()
    slack = 16 * U * (a * h.double().abs() + m * x.double().abs())
    old = h.cuda()
    to = torch.full_like(old, float("nan"))
    y, new = pcb().gated_scan_step(x.cuda(), g.cuda(), old, to)
    assert new is to and torch.equal(old.cpu(), h)
    check(y, ref, slack, "y"), check(new, ref, slack, "state")
    version = old._version
    y2, new2 = pcb().gated_scan_step(torch.cat([x, g], -1).cuda(), None, old)
    assert new2 is old and old._version > version and torch.equal(y2, y) and torch.equal(old, to)


def test_step_refuses_gradients_and_overlap():
    x = torch.randn(4, 8, device="cuda")
    store = torch.zeros(80, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        pcb().gated_scan_step(x, x, store[:32].view(4, 8), store[16:48].view(4, 8))
    with pytest.raises(RuntimeError, match="no gradient"):
        pcb().gated_scan_step(x.clone().requires_grad_(), x, store[:32].view(4, 8))
    with torch.no_grad():
        pcb().gated_scan_step(x.clone().requires_grad_(), x, store[:32].view(4, 8))
    with torch.inference_mode():
        h = torch.zeros(4, 8, device="cuda")
        pcb().gated_scan_step(x, x, h)


def test_function_form_and_no_second_derivative():
    d = data((2, 300, 20), 1, torch.float32, lengths=True)
    base = run(d, 1, True)
    v = [d[k].cuda().requires_grad_() for k in ("x", "g", "state")]
    out = pcb().GatedScanFunction.apply(*v, d["lengths"].cuda(), 1, True)
    grads = torch.autograd.grad(out, v, [d["gy"].cuda(), d["glast"].cuda()])
    for k, t in zip(("y", "last", "gx", "gg", "gstate"), (*out, *grads)):
        assert torch.equal(t, base[k]), k
    y, last = pcb().GatedScan(dim=1)(v[0], v[1])
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum() + last.sum(), v[0], create_graph=True)


def test_trace_records_the_function_form():
    x, g = torch.randn(2, 9, 8, device="cuda"), torch.randn(2, 9, 8, device="cuda")
    traced = torch.jit.trace(lambda a, b: pcb().gated_scan(a, b)[0], (x, g), check_trace=False)
    x2 = torch.randn_like(x)
    assert torch.equal(traced(x2, g), pcb().gated_scan(x2, g)[0])


def test_other_stream_and_repeatability():
    d = data((2, 3000, 64), 1, torch.bfloat16)
    base = run(d, 1, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(d, 1, False)
    side.synchronize()
    for k in base:
        assert torch.equal(base[k], again[k]), k


def test_two_streams_at_once():
    """Passes on two streams, under way together, forward and backward of all three operators: bitwise what each is by itself."""
    dt = torch.bfloat16
    sets = [[torch.randn(2, 2500, 96, device="cuda").to(dt).requires_grad_() for _ in range(3)] for _ in range(2)]
    w = torch.rand(96, device="cuda").to(dt)

    def f(x, g, gate):
        z = pcb().channel_norm(x, w, kind="layer")
        y, last = pcb().gated_scan(z, g)
        out, nxt = pcb().gated_residual(x, y, w, gate=gate, kind="rms", activation="sigmoid", next_weight=w, next_kind="rms")
        return [out.detach(), nxt.detach(), last.detach(), *torch.autograd.grad([out, nxt], [x, g, gate], [z.detach(), y.detach()])]

    alone = [f(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    results = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(f(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in results[i]:
            for a, b in zip(r, alone[i]):
                assert torch.equal(a, b)


def test_captured_passes_replay():
    """Two graphs, one of a long chain cut into segments and one of steps, replayed with eager work between: every replay is the
    eager result on the same inputs."""
    x = torch.randn(1, 3000, 64, device="cuda").bfloat16().requires_grad_()
    g = (torch.randn(1, 3000, 64, device="cuda") + 2).bfloat16().requires_grad_()
    gy = torch.randn(1, 3000, 64, device="cuda").bfloat16()
    h = torch.randn(1, 64, device="cuda")
    to = torch.empty_like(h)

    def step():
        y, last = pcb().gated_scan(x, g, h)
        return [y.detach(), last.detach(), *torch.autograd.grad(y, [x, g], gy)]

    def token():
        return list(pcb().gated_scan_step(x.detach()[:, 0], g.detach()[:, 0], h, to))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), token()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for f in (step, token):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, f, f()))
        graphs[-1] = (graph, f, graphs[-1][2])
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


@pytest.mark.parametrize("op", ["scan", "norm", "residual"])
def test_capture_beside_an_eager_graph_is_refused(op):
    """A backward pass under capture whose gradients would go to accumulators of the default stream raises, and leaves the process as it was;
    with the eager output gone the same capture works."""
    x, g = (torch.randn(2, 40, 64, device="cuda").requires_grad_() for _ in range(2))
    w = torch.ones(64, device="cuda").requires_grad_()
    gy = torch.randn(2, 40, 64, device="cuda")

    def forward():
        if op == "scan":
            return pcb().gated_scan(x, g)[0], [x, g]
        if op == "norm":
            return pcb().channel_norm(x, w), [x, w]
        return pcb().gated_residual(x, g, w, kind="rms"), [x, g, w]

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
            if t.data_ptr() != gy.data_ptr():   # (the gradient of a residual's x is gy itself)
                t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, ref):
            assert torch.equal(a, b)


def test_norm_scan_residual_as_a_block():
    """A block around the recurrence as a model has it: norm, one projection for values, decays and gate, the scan down an image's
    columns, gated residual with the next norm; gradients for all of it against the same in plain 64-bit operations.

    The projection's result is rounded to bfloat16 in both; from there each tensor between the operators is rounded once (2^-9), so
    results agree to a few times 2^-8 of their largest."""
    torch.manual_seed(0)
    B, H, W, C = 2, 12, 10, 32
    dt = torch.bfloat16
    leaf = lambda *s, mean=0.0, std=1.0: (torch.randn(*s) * std + mean).to(dt)
    p = {"x": leaf(B, H, W, C), "w1": leaf(C, mean=1.0, std=0.1), "proj": leaf(3 * C, C, std=C ** -0.5), "w2": leaf(C, mean=1.0, std=0.1),
         "scale": leaf(C, mean=0.5, std=0.1), "w3": leaf(C, mean=1.0, std=0.1)}
    go, gn = leaf(B, H, W, C), leaf(B, H, W, C)
    v = {k: t.cuda().requires_grad_() for k, t in p.items()}
    z = pcb().channel_norm(v["x"], v["w1"])
    q = torch.nn.functional.linear(z, v["proj"])
    y, _ = pcb().gated_scan(q[..., :2 * C], dim=1, reverse=True)
    out, nxt = pcb().gated_residual(v["x"], y, v["w2"], gate=q[..., 2 * C:], scale=v["scale"], kind="rms", activation="silu",
                                    next_weight=v["w3"], next_kind="layer")
    grads = torch.autograd.grad([out, nxt], list(v.values()), [go.cuda(), gn.cuda()])

    r = {k: t.double().requires_grad_() for k, t in p.items()}
    rms = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    q = torch.nn.functional.linear(rms(r["x"], r["w1"]), r["proj"])
    x, g, gate = q.chunk(3, -1)
    h, ys = torch.zeros(B, W, C, dtype=torch.float64), [None] * H
    for t in range(H - 1, -1, -1):
        a = torch.sigmoid(g[:, t])
        h = a * h + (1 - a) * x[:, t]
        ys[t] = h
    rout = r["x"] + r["scale"] * gate * torch.sigmoid(gate) * rms(torch.stack(ys, 1), r["w2"])
    c = rout - rout.mean(-1, keepdim=True)
    rnxt = c / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt() * r["w3"]
    rgrads = torch.autograd.grad([rout, rnxt], list(r.values()), [go.double(), gn.double()])
    for name, a, b in zip(["out", "next", *v], [out, nxt, *grads], [rout, rnxt, *rgrads]):
        err = (a.detach().double().cpu() - b.detach()).norm() / b.detach().norm()
        assert err <= 2 ** -6, (name, float(err))
