"""channel_norm, gated_residual and gated_scan where their ranges end.  References and bounds are those of test_gpu_norm.py and
test_gpu_scan.py: 64 bits, element by element."""
import pytest
import torch
from test_gpu_norm import (EPS, check, doubles, norm64, norm_bwd64, pcb, residual64, residual_data, rnd, rows_slack,
                           run_residual)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# Gates far from zero.  Below -87 the kernels take silu and its slope for 0: there both are under 88 e^-87 < 2^-118, times factors
# under 2^10 and sums of fewer than 2^8 terms: under 2^-100 in every result.
LOW = [-1.0, -20.0, -86.0, -87.5, -88.0, -90.0, -110.0, -200.0, -1e4, -1e30, -1e36, "min"]


def extreme_gates(shape, dtype, high, seed):
    info = torch.finfo(dtype)
    values = torch.tensor([max(info.min if v == "min" else v, info.min) for v in LOW] + high, dtype=torch.float64)
    gen = torch.Generator().manual_seed(seed)
    return values[torch.randint(0, len(values), shape, generator=gen)].to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("gate", ["image", "full"])
@pytest.mark.parametrize("next_kind", ["none", "rms"])
@pytest.mark.parametrize("shape", [(3, 5, 40), (2, 7, 9), (2, 3, 1152)], ids=str)
def test_extreme_gates(shape, next_kind, gate, act, dtype):
    """Gates down to the type's lowest value, as masks leave them, and large ones: a silu of 0 and not of -4, and no gradient."""
    d = residual_data(shape, dtype, gate, True, "w", "w" if next_kind != "none" else "")
    # (a next norm squares the sum; in float16 it has to stay in range itself)
    high = [30.0, 100.0] + ([1e30] if next_kind == "none" and dtype != torch.float16 else [])
    d["gate"] = extreme_gates(d["gate"].shape, dtype, high, 7)
    got = run_residual(d, act, "rms", next_kind, dtype)
    ref = residual64(doubles(d), act, "rms", next_kind, gate == "image")
    assert set(got) == set(ref)
    for k, (value, bound) in ref.items():
        check(got[k], value, bound + 2.0 ** -100, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", ["min", "-inf"])
@pytest.mark.parametrize("gate", ["image", "full"])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_a_masked_branch_adds_nothing(act, gate, value, dtype):
    d = residual_data((2, 9, 72), dtype, gate, True, "wb", "")
    d["gate"] = torch.full_like(d["gate"], torch.finfo(dtype).min if value == "min" else float("-inf"))
    got = run_residual(d, act, "layer", "none", dtype)
    if dtype == torch.float16 and value == "min":   # (of a float16 gate too: its lowest value is below -87)
        assert float(d["gate"].max()) < -87
    assert torch.equal(got["out"].detach().cpu(), d["x"])
    for k in ("gy", "ggate", "gscale", "gw", "gb"):
        assert not got[k].any(), k


@pytest.mark.parametrize("eps", [0.0, 1e-44])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("value", [1e-18, 1.1e-19, 1e-19, 1e-20, 1e-21])
def test_tiny_rows_without_an_eps(value, kind, eps):
    """Rows of +-v whose variance is subnormal: +-1, as far as the square is one of the type's numbers (2^-149 apart: v^2, the sum of 64 of them, exact
    from there, and its 64th part are each off by half of that at most, and so the result by half of 1.5 * 2^-149 / v^2 and
    some roundings; eps adds 1e-44 / v^2 / 2), and finite gradients of rows that are not tiny beside them."""
    x = torch.full((3, 64), value)
    x[:, ::2] *= -1
    x[2] = torch.randn(64)
    xd = x.cuda().requires_grad_()
    y = pcb().channel_norm(xd, kind=kind, eps=eps)
    off = 0.75 * 2.0 ** -149 / value ** 2 + eps / value ** 2 / 2 + 16 * U
    assert float((y[:2].detach().cpu() - x[:2].sign()).abs().max()) <= off
    (g,) = torch.autograd.grad(y, [xd], torch.randn(3, 64, device="cuda"))
    assert g[2].isfinite().all()


# Calls in which a row group goes through several rows (its next row's loads under way, its column sums carried along), with a last one that is
# not full.  A lane's sum is as many additions as its group has rows, at most N / 512 + 1 (the backward aims at 512 workgroups or more), one or a few
# for segments and 24 for lanes, wavefronts and the sum over segments; rows_slack's 48 + N / 1024 holds that up to N = 24 * 1024 rows
# of a whole workgroup, and any N of groups of which a workgroup has two or more.
def backward_rows(N, C, dtype):
    """Rows of a group in the backward, at most, from the segments that the workspace is made for."""
    from pyramidconvblock_amd import _lib

    segments = _lib.lib().pdw_norm_bwd_workspace_bytes(N, C, _lib.dtype_code(dtype)) // (2 * C * 4)
    pieces = -(-C // (4 if dtype == torch.float32 else 8))
    groups = 1 if pieces > 64 else 512 // max(8, 1 << (pieces - 1).bit_length())
    return -(-N // segments) / groups


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,affine", [("rms", "w"), ("layer", "wb")])
@pytest.mark.parametrize("shape", [(65573 * 2, 24), (20011, 200), (20011, 201), (9001, 520), (4207, 1152), (2101, 5000)], ids=str)
def test_norm_of_several_rows_a_group(shape, kind, affine, dtype):
    N, C = shape
    assert backward_rows(N, C, dtype) > 1
    gen = torch.Generator().manual_seed(N)
    x, gy = rnd(gen, N, C, dtype=dtype, mean=0.5), rnd(gen, N, C, dtype=dtype)
    w = rnd(gen, C, dtype=dtype, mean=1.0, std=0.3)
    b = rnd(gen, C, dtype=dtype) if "b" in affine else None
    leaves = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    y = pcb().channel_norm(*leaves, kind=kind, eps=EPS)
    grads = torch.autograd.grad(y, leaves, gy.cuda())
    f = lambda t: None if t is None else t.double()
    ry, n, r, dn = norm64(f(x), f(w), f(b), kind)
    check(y, ry, dn * f(w).abs() + 8 * U * ry.abs(), "y")
    check(grads[0], *norm_bwd64(f(gy), n, r, dn, f(w), kind), "gx")
    check(grads[1], (f(gy) * n).sum(0), rows_slack(f(gy) * n, f(gy).abs() * dn), "gw")
    if b is not None:
        check(grads[2], f(gy).sum(0), rows_slack(f(gy), 0 * f(gy)), "gb")


ROWS_FORMS = [("none", "none", "rms", "w", "none", "", True), ("image", "silu", "layer", "wb", "rms", "w", True),
              ("image", "sigmoid", "none", "", "none", "", True), ("full", "silu", "layer", "wb", "rms", "w", True),
              ("full", "none", "rms", "w", "none", "", False), ("none", "none", "none", "", "layer", "wb", True)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("form", ROWS_FORMS, ids=lambda f: "-".join(str(v) for v in f))
@pytest.mark.parametrize("shape", [(2, 40011, 24), (3, 7001, 201), (3, 3001, 520), (40, 99, 1152), (2, 1051, 5000)], ids=str)
def test_residual_of_several_rows_a_group(shape, form, dtype):
    gate, act, kind, affine, next_kind, next_affine, scale = form
    assert backward_rows(shape[0] * shape[1], shape[2], dtype) > 1
    d = residual_data(shape, dtype, gate, scale, affine, next_affine, seed=3)
    got = run_residual(d, act, kind, next_kind, dtype)
    ref = residual64(doubles(d), act, kind, next_kind, gate == "image")
    assert set(got) == set(ref)
    for k, (value, bound) in ref.items():
        check(got[k], value, bound, k)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,W,C", [(2, 9, 5, 8), (1, 40, 3, 33), (2, 300, 4, 16), (70, 20, 6, 64)])
def test_halves_in_rows_that_overlap(B, T, W, C, dtype, reverse):
    """Sliding windows over the channels as x and g in one tensor: each half's rows lie side by side, the gradient's do not.  Bitwise
    the results of a copy without overlap, and the gradients summed where windows share an element."""
    gen = torch.Generator().manual_seed(W)
    base = rnd(gen, B, T, (W + 1) * C, dtype=dtype).cuda().requires_grad_()
    gy, glast = rnd(gen, B, T, W, C, dtype=dtype).cuda(), rnd(gen, B, W, C).cuda()
    windows = base.unfold(-1, 2 * C, C)
    assert windows.shape == (B, T, W, 2 * C) and windows.stride()[-2:] == (C, 1)
    dense = windows.detach().contiguous().requires_grad_()
    got, ref = (pcb().gated_scan(t, dim=1, reverse=reverse) for t in (windows, dense))
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    leaf = windows.detach().as_strided(windows.shape, windows.stride()).requires_grad_()
    (gl,) = torch.autograd.grad(pcb().gated_scan(leaf, dim=1, reverse=reverse), [leaf], [gy, glast])
    (gd,) = torch.autograd.grad(ref, [dense], [gy, glast])
    assert torch.equal(gl, gd)
    (gb,) = torch.autograd.grad(got, [base], [gy, glast])
    summed = torch.zeros_like(base)
    for w in range(W):
        summed[..., w * C:(w + 2) * C] += gd[:, :, w]
    # two addends at most, in whichever order: one rounding
    assert torch.equal(gb, summed)


def test_channels_up_to_the_last_32_bit_number():
    """2^31 - 1 channels, the last of which a lane of the last strip shares with the lane before it: the last ones are bitwise what they are in a
    call by themselves, the others what zeros give."""
    C, T, last = (1 << 31) - 1, 2, 45
    gen = torch.Generator().manual_seed(14)
    data = [rnd(gen, T, last, dtype=torch.bfloat16).cuda() for _ in range(3)] + [rnd(gen, last).cuda()]
    wide = [torch.zeros(T, C, device="cuda", dtype=torch.bfloat16) for _ in range(3)] + [torch.zeros(C, device="cuda")]
    for a, b in zip(wide, data):
        a[..., -last:] = b

    def call(x, g, gy, state):
        x, g, state = (t.requires_grad_() for t in (x, g, state))
        y, end = pcb().gated_scan(x, g, state, dim=0)
        return [y.detach(), end.detach(), *torch.autograd.grad(y, [x, g, state], gy)]

    for a, b in zip(call(*wide), call(*data)):
        assert torch.equal(a[..., -last:], b) and int(torch.count_nonzero(a)) == int(torch.count_nonzero(b))


def test_more_images_than_one_launch_holds():
    """A gate row for each of so many images that the workgroups times their threads pass 2^32, in the forward (256 threads), the backward (512) and
    the sums over rows (1024): HIP would cut the grid without an error.
    The last images are bitwise what they are in a call by themselves, the column sums within their bound."""
    B, P, C, last = (1 << 24) + 3, 2, 8, 37
    gen = torch.Generator().manual_seed(11)
    x = torch.zeros(B, P, C, device="cuda", dtype=torch.bfloat16)
    y, go, gate = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(B, C, device="cuda", dtype=torch.bfloat16)
    d = {k: rnd(gen, last, P, C, dtype=torch.bfloat16).cuda() for k in ("x", "y", "go")}
    d["gate"] = rnd(gen, last, C, dtype=torch.bfloat16).cuda()
    w = rnd(gen, C, dtype=torch.bfloat16, mean=1.0, std=0.2).cuda().requires_grad_()
    for big, k in ((x, "x"), (y, "y"), (go, "go"), (gate, "gate")):
        big[-last:] = d[k]

    def call(x, y, gate, go):
        x, y, gate = (t.requires_grad_() for t in (x, y, gate))
        out, nxt = pcb().gated_residual(x, y, w, gate=gate, kind="rms", activation="silu", next_kind="layer")
        return [out, nxt, *torch.autograd.grad([out, nxt], [x, y, gate, w], [go, go])]

    many, few = call(x, y, gate, go), call(d["x"], d["y"], d["gate"], d["go"])
    for a, b in zip(many[:-1], few[:-1]):
        assert torch.equal(a[-last:], b) and not a[:-last].any()
    # the weight's gradient: zeros and the same terms in another order, each sum within 64 u of the terms' magnitudes and rounded once
    f = lambda t: t.detach().double().cpu()
    out, _, gx, *_ = few
    n = norm64(f(d["y"]), None, None, "rms")[1]
    q = f(d["gate"])[:, None]
    terms = (f(gx) * n * q * torch.sigmoid(q)).abs().sum((0, 1))
    # (gx itself is rounded to bfloat16 in `terms` alone: they only scale the bound, by 1 + 2^-8)
    assert ((f(many[-1]) - f(few[-1])).abs() <= 2.0 ** -7 * f(few[-1]).abs() + 2 * 64 * U * 1.01 * terms).all()


def test_more_chains_than_one_launch_holds():
    """So many chains and tokens that the workgroups times their threads pass 2^32: the last ones are bitwise what they are in a call by themselves."""
    B, T, last = (1 << 24) + 5, 3, 33   # of one channel: a workgroup of 256 threads each
    gen = torch.Generator().manual_seed(12)
    x, g = torch.zeros(B, T, 1, device="cuda", dtype=torch.bfloat16), torch.zeros(B, T, 1, device="cuda", dtype=torch.bfloat16)
    gy = torch.zeros_like(x)
    xl, gl, gyl = (rnd(gen, last, T, 1, dtype=torch.bfloat16).cuda() for _ in range(3))
    x[-last:], g[-last:], gy[-last:] = xl, gl, gyl

    def call(x, g, gy):
        x, g = x.requires_grad_(), g.requires_grad_()
        y, state = pcb().gated_scan(x, g)
        return [y, state, *torch.autograd.grad(y, [x, g], gy)]

    for a, b in zip(call(x, g, gy), call(xl, gl, gyl)):
        assert torch.equal(a[-last:], b) and not a[:-last].any()


def test_more_tokens_than_one_launch_holds():
    B, C, last = (1 << 30) + 7, 5, 100   # of an odd number of channels: a thread a value
    gen = torch.Generator().manual_seed(13)
    x, state = torch.zeros(B, C, device="cuda", dtype=torch.bfloat16), torch.zeros(B, C, device="cuda")
    xl, hl = rnd(gen, last, C, dtype=torch.bfloat16).cuda(), rnd(gen, last, C).cuda()
    x[-last:], state[-last:] = xl, hl
    y, h = pcb().gated_scan_step(x, x, state)
    yl, hl = pcb().gated_scan_step(xl, xl, hl)
    assert torch.equal(y[-last:], yl) and torch.equal(h[-last:], hl)
    assert not y[:-last].any() and not h[:-last].any()


@pytest.mark.parametrize("op", ["scan", "norm", "residual"])
def test_capture_asks_only_for_the_gradients_that_are_wanted(op):
    """A captured backward pass that wants x's gradient alone, beside an eager graph of the other leaf, whose accumulator works on the default
    stream: nothing is handed to that one, so the capture goes through, and its replays are the eager result."""
    x, other, w = torch.randn(2, 40, 64, device="cuda"), torch.randn(2, 40, 64, device="cuda"), torch.ones(64, device="cuda")
    gy = torch.randn(2, 40, 64, device="cuda")
    x.requires_grad_(), other.requires_grad_(), w.requires_grad_()
    unrelated = torch.randn(2, 40, 64, device="cuda")

    def forward(x):
        if op == "scan":
            return pcb().gated_scan(x, other)[0]
        if op == "norm":
            return pcb().channel_norm(x, w)
        return pcb().gated_residual(x, other, w, kind="rms", next_weight=w, next_kind="layer")[1]

    def step():
        return torch.autograd.grad(forward(x), [x], gy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    eager = forward(unrelated)   # keeps the accumulators of `other` and `w`, not of x
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for _ in range(3):
        res.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = res.clone()
        assert torch.equal(got, step())
    assert eager.requires_grad


def test_a_replayed_trace_checks_its_tensors():
    """A trace calls the function forms again with the tensors that it is given: with ones that fit the results of the plain calls, with others a
    refusal."""
    x, w = torch.randn(3, 7, 24, device="cuda"), torch.rand(24, device="cuda")
    calls = {"norm": lambda t: pcb().channel_norm(t, w, kind="layer"),
             "residual": lambda t: pcb().gated_residual(t, t * 2, w, scale=w, kind="rms", next_kind="layer")[1],
             "scan": lambda t: pcb().gated_scan(t, t * 2, dim=-2)[0], "halves": lambda t: pcb().gated_scan(t, dim=-2)[0]}
    for name, f in calls.items():
        traced = torch.jit.trace(f, (x,), check_trace=False)
        other = torch.randn(5, 9, 24, device="cuda")
        assert torch.equal(traced(other), f(other)), name
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            traced(other.double())
        if name in ("norm", "residual"):
            with pytest.raises((RuntimeError, TypeError, ValueError)):
                traced(torch.randn(5, 9, 40, device="cuda"))
