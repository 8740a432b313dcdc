"""gated_delta where a workgroup goes through many chunks, in one run and in segments, with more workgroups than the chip has places for; and with keys
that repeat.  Against the recurrence in 64 bits (on the GPU, all chains at once), with the bounds of test_gpu_delta.py: the recurrence again, off by
2^-16 (32-bit results: 2^-21) at every step, and 16 times the most that an element of the same step of the sequence moved in two such runs.

The chains' operands are under way 4, 3 and 2 chunks ahead with up to 32, 64 and 128 channels of keys: runs here are longer than twice that."""
import ctypes

import pytest
import torch
from test_gpu_delta import DTYPES, NAMES, check, compare, data, run

AHEAD = {32: 4, 64: 3, 128: 2}
# (dimensions before the heads, heads of keys, of values, channels of keys, of values), whether in segments, and what else
CASES = {
    "32": ((1, 620, 300), 2, 2, 17, 5, False, dict(dim=1, state=True)),
    "32, reversed, lengths": ((3, 610, 50), 1, 2, 32, 20, False, dict(dim=1, lengths=[610, 577, 130], reverse=True)),
    "64": ((2, 500, 75), 2, 2, 33, 9, False, dict(dim=1, state=True)),
    "128": ((1, 500, 130), 1, 2, 65, 5, False, dict(dim=1, state=True)),
    "32, segments": ((1, 1590, 48), 2, 2, 17, 5, True, dict(dim=1, state=True)),
    "64, segments": ((2, 1290, 16), 1, 2, 33, 9, True, dict(dim=1, state=True, reverse=True, lengths=[1290, 1001])),
    "128, segments": ((1, 1290, 10), 2, 2, 65, 70, True, dict(dim=1, state=True)),
}


def padded(dk):
    return 32 if dk <= 32 else 64 if dk <= 64 else 128


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", CASES)
def test_the_cases_are_long_runs(name, dtype):
    """(Without a GPU.)  How many segments a call is cut into shows in the size of its workspace: a map of DK x DK in three planes and a shift of DK x dvp for each
    chain's segments but one, and 64 x dvp for each chunk."""
    from pyramidconvblock_amd import _lib

    (O, T, W), hk, hv, dk, dv, segments, _ = CASES[name]
    c = _lib.Delta()
    for n, v in dict(q=1, k=1, v=1, g=1, b=1, O=O, T=T, W=W, Hk=hk, Hv=hv, dk=dk, dv=dv, scale=1.0, dtype=_lib.dtype_code(dtype)).items():
        setattr(c, n, v)
    got = _lib.lib().pdw_delta_workspace_bytes(ctypes.addressof(c), 0, 1)
    chains, chunks, DK, dvp = O * W * hv, (T + 63) // 64, padded(dk), (dv + 31) // 32 * 32
    whole = lambda n: (n + 255) // 256 * 256
    size = lambda s: whole(chains * (s - 1) * DK * DK * 3 * 2) + whole(chains * (s - 1) * DK * dvp * 4) + whole(chains * chunks * 64 * dvp * 4)
    (n,) = [s for s in range(1, 65) if size(s) == got]
    assert (n > 1) == segments and -(-chunks // n) > 2 * AHEAD[DK], (n, chunks)


class Off(torch.autograd.Function):
    """x and its gradient, each off by up to e of itself."""

    @staticmethod
    def forward(ctx, x, e, gen):
        ctx.e, ctx.gen = e, gen
        return x * (1 + e * Off.signs(x, gen))

    @staticmethod
    def backward(ctx, g):
        return g * (1 + ctx.e * Off.signs(g, ctx.gen)), None, None

    @staticmethod
    def signs(x, gen):
        return torch.empty_like(x).uniform_(-1, 1, generator=gen).sign()


def reference(s, off=0.0, seed=0):
    """-> {name: 64 bits on the CPU}"""
    gen = torch.Generator("cuda").manual_seed(seed)
    o = (lambda t: Off.apply(t, off, gen)) if off else lambda t: t
    leaves = {n: s[n].cuda().double().requires_grad_() for n in NAMES + ["state"] if s[n] is not None}
    O, T, W, hk, dk = s["q"].shape
    hv, dv = s["v"].shape[-2:]
    n = torch.full((O,), T, device="cuda") if s["lengths"] is None else s["lengths"].cuda().long()
    at = torch.arange(T, device="cuda").expand(O, T)
    valid = at < n[:, None]
    step = torch.where(valid, n[:, None] - 1 - at, at) if s["reverse"] else at
    # [T, O, W, heads, ..] in the order of the rule (and back: the order is its own inverse)
    turn = lambda t: t.gather(1, step.reshape(O, T, *[1] * (t.dim() - 2)).expand(t.shape))
    rows = {k: turn(leaves[k]).transpose(0, 1) for k in NAMES}
    q, k = (rows[m].repeat_interleave(hv // hk, -2) for m in "qk")
    there = valid.t()[:, :, None, None]
    a = torch.where(there, o(torch.sigmoid(rows["g"])), 1.0)
    beta = torch.where(there, o(torch.sigmoid(rows["b"])), 0.0)
    S = leaves["state"] if "state" in leaves else torch.zeros(O, W, hv, dk, dv, dtype=torch.float64, device="cuda")
    ys = []
    for t in range(T):
        S = S * a[t][..., None, None]
        u = o(beta[t][..., None] * (rows["v"][t] - (k[t][..., :, None] * S).sum(-2)))
        S = o(S + k[t][..., :, None] * u[..., None, :])
        ys.append((q[t][..., :, None] * S).sum(-2))
    y = turn((torch.where(there[..., None], torch.stack(ys), 0.0) * s["scale"]).transpose(0, 1))
    out = {"y": y, "last": S}
    grads = torch.autograd.grad([y, S], list(leaves.values()), [s["gy"].cuda().double(), s["glast"].cuda().double()])
    out |= {"g" + m: t for m, t in zip(leaves, grads)}
    return {m: t.detach().cpu() for m, t in out.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", CASES)
def test_long_runs(name, dtype):
    lead, hk, hv, dk, dv, _, options = CASES[name]
    s = data(lead, hk, hv, dk, dv, dtype, nan=False, **options)
    ref, off, bound = reference(s), 2.0 ** -16, {}
    for seed in (1, 2):
        r = reference(s, off, seed)
        for k in ref:   # (what such small steps move goes with their size)
            less = 2.0 ** -5 if k in ("last", "gstate") or dtype == torch.float32 else 1.0
            # (gg at a step is a sum over the steps behind it in its chunk, of terms that cancel: it is as far off as the largest of them, not as it is large)
            most = lambda t: t.abs().amax(list(range({"last": 1, "gstate": 1, "gg": 0}.get(k, 2), t.dim())), keepdim=True)
            bound[k] = torch.maximum(bound.get(k, torch.zeros(())), less * (16 * most(r[k] - ref[k]) + off * most(ref[k])))
    for train in (True, False):
        got = run(s, train)
        for k in got:
            check(got[k], ref[k], bound[k], (k, train))
    if s["lengths"] is not None:
        for k in ("y", "gq", "gk", "gv", "gg", "gb"):
            assert k not in got or not got[k][s["behind"].cuda()].any(), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("how", ["same", "two in turn", "signs"])
def test_keys_that_repeat(how, d, dtype):
    """Hardly any decay, nearly everything replaced: the triangular system's entries are all near 1 (powers of it grow as binomials, and cancel)."""
    s = data((2, 150), 2, 2, d, 24, dtype, state=True)
    t = torch.arange(150)
    s["k"] = s["k"][:, t % 2 if how == "two in turn" else 0 * t]
    if how == "signs":
        s["k"] = s["k"] * torch.where(t % 3 == 0, -1, 1).to(dtype)[:, None, None]
    s["g"][:], s["b"][:, :, 0], s["b"][:, :, 1] = 9.0, 8.0, 2.0
    compare(s)
    compare(s, train=False)
