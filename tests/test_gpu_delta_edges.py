"""gated_delta where values are not finite: what such a value may reach."""
import pytest
import torch
from test_gpu_delta import DTYPES, NAMES, data, run

pytestmark = pytest.mark.gpu

CHUNK = 64
SIZES = {
    "32": ((2, 150), 2, 2, 32, 24, {}),
    "32, reversed, lengths": ((2, 150), 2, 2, 20, 40, dict(reverse=True, lengths=[150, 131])),
    "64": ((2, 150), 2, 2, 64, 64, {}),
    "64, shared, down the columns": ((2, 150, 2), 1, 2, 48, 72, dict(dim=1)),
    "128": ((2, 150), 1, 1, 128, 128, dict(reverse=True)),
    "segments": ((1, 1300), 1, 1, 32, 32, {}),
}


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("value", ["nan", "inf"])
@pytest.mark.parametrize("name", SIZES)
def test_what_is_not_finite_reaches_no_step_before_it(name, value, dtype):
    """As step by step: from the bad step on y and the last state are NaN, of its channel of v or (k, g, b) of its head; every other result is the
    bits that it was.  In the gradients a bad v leaves the chunks before its own as they were."""
    lead, *heads, options = SIZES[name]
    s = data(lead, *heads, dtype, state=True, nan=False, **options)
    base, few = run(s), run(s, train=False)
    T, row = lead[s["dim"]], len(lead) - 1   # (the last row of each axis but the sequence's)
    n = T if s["lengths"] is None else int(s["lengths"].reshape(-1)[-1])
    at = lambda t, i: t[tuple(i if d == s["dim"] else -1 for d in range(row + 1))]
    for place in [i for i in (0, 5, 16, 33, 47, 62, 63, 64, 79, 100, 127, 128, n - 1, T // 2) if i < n]:
        step = n - 1 - place if s["reverse"] else place
        order = list(range(n - 1, -1, -1) if s["reverse"] else range(n))
        for what in ("v", "k", "g", "b"):
            if value == "inf" and what in "gb":
                continue   # (gates at their ends are gates)
            bad = {**s, what: s[what].clone()}
            at(bad[what], step)[(-1, 3) if what in "vk" else -1] = float(value)
            spoiled = s["v"].shape[-2] // s["q"].shape[-2] if what == "k" else 1   # (value heads of the last key head)
            for train, ref in ((True, base), (False, few)):
                got = run(bad, train)
                y, last = got["y"].detach().cpu(), got["last"].detach().cpu()
                mine = torch.zeros(y.shape, dtype=torch.bool)
                for i in order[place:]:
                    at(mine, i)[(-1, 3) if what == "v" else slice(-spoiled, None)] = True
                ends = torch.zeros(last.shape, dtype=torch.bool)
                ends[(-1,) * (row) + ((-1, slice(None), 3) if what == "v" else (slice(-spoiled, None),))] = True
                for k, t, m in (("y", y, mine), ("last", last, ends)):
                    assert t[m].isnan().all(), (what, place, train, k)
                    assert torch.equal(t[~m], ref[k].detach().cpu()[~m]), (what, place, train, k)
                if train and what == "v":
                    for k in ("gq", "gk", "gv", "gg", "gb"):
                        for i in order[:place // CHUNK * CHUNK]:
                            assert torch.equal(at(got[k], i), at(base[k], i)), (k, place, i)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_a_state_that_is_not_finite(dtype):
    s = data((2, 90), 2, 2, 32, 32, dtype, state=True)
    for train in (True, False):
        base = run(s, train)
        got = run({**s, "state": s["state"].index_put((torch.tensor(1), torch.tensor(0), torch.tensor(7), torch.tensor(3)), torch.tensor(float("nan")))}, train)
        for k in ("y", "last"):
            mine = torch.zeros(got[k].shape, dtype=torch.bool)
            mine[(1, slice(None), 0, 3) if k == "y" else (1, 0, slice(None), 3)] = True
            assert got[k].cpu()[mine].isnan().all() and torch.equal(got[k].cpu()[~mine], base[k].cpu()[~mine])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_bad_steps_are_where_the_form_step_by_step_has_them(dtype):
    """16 steps: in chunks (for gradients) and one after another (without)."""
    for n in NAMES:
        s = data((2, 16), 2, 4, 24, 40, dtype, state=True)
        s[n][1, 9, 1] = float("nan")
        chunks, steps = run(s), run(s, train=False)
        for k in ("y", "last"):
            assert torch.equal(chunks[k].isnan(), steps[k].isnan()), (n, k)
        assert chunks["y"].isnan().any() and not chunks["y"][:, :9].isnan().any(), n
