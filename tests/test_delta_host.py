"""What head_rotary, gated_delta and gated_delta_step refuse, and the library's answers to arguments, without a GPU."""
import ctypes

import pytest
import torch


def pcb():
    import pyramidconvblock_amd

    return pyramidconvblock_amd


def lib():
    from pyramidconvblock_amd import _lib

    return _lib.lib()


def refused(error, match, call, *args, **kw):
    with pytest.raises(error, match=match):
        call(*args, **kw)


def test_rotary_refusals():
    f = pcb().head_rotary
    q, k, w = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8), torch.ones(8)
    refused(RuntimeError, "no CPU path", f, q, k)
    refused(ValueError, "kind", f, q, kind="batch")
    refused(TypeError, "q has to be", f, None)
    refused(TypeError, "Tensor", f, [1.0])
    refused(TypeError, "float32/float16/bfloat16", f, q.double())
    refused(TypeError, "float32/float16/bfloat16", f, q.int())
    refused(TypeError, "k is", f, q, k.half())
    refused(ValueError, "alike but for their heads", f, q, k[:1])
    refused(ValueError, "alike but for their heads", f, q, k[..., :4])
    refused(ValueError, "alike but for their heads", f, q, k[0])
    refused(ValueError, "1 <= d <= 256", f, torch.zeros(2, 1, 257))
    refused(ValueError, "1 <= d <= 256", f, torch.zeros(2, 1, 0))
    refused(ValueError, "1 <= d <= 256", f, torch.zeros(8))
    refused(ValueError, "65536 heads", f, torch.zeros(1).expand(1, 65537, 1))
    refused(ValueError, "1, 2 or 3", f, q, axes=0)
    refused(ValueError, "1, 2 or 3", f, q, axes=4)
    refused(ValueError, "are the grid", f, q, axes=3)
    refused(ValueError, "are the grid", f, torch.zeros(4, 8))
    refused(TypeError, "tuple of 2", f, q, axes=2, sections=(2,))
    refused(ValueError, "5 pairs", f, q, sections=(5,))
    refused(ValueError, "section 0 has -1", f, q, axes=2, sections=(-1, 2))
    refused(ValueError, "section 0 has 9", f, q, sections=(9,))
    refused(TypeError, None, f, q, sections=("a",))
    refused(ValueError, "base", f, q, base=0.0)
    refused(ValueError, "base", f, q, base=float("nan"))
    refused(ValueError, "eps", f, q, eps=-1e-6)
    refused(ValueError, "weight without a norm", f, q, weight=w)
    refused(ValueError, "key_weight without k", f, q, key_weight=w, kind="rms")
    refused(ValueError, "weight has to be", f, q, weight=torch.ones(7), kind="rms")
    refused(ValueError, "key_weight has to be", f, q, k, key_weight=torch.ones(4, 8), kind="l2")
    refused(TypeError, "weight is", f, q, weight=w.half(), kind="rms")
    refused(TypeError, "positions are", f, q, positions=torch.zeros(5, 1, dtype=torch.float64))
    refused(ValueError, "positions have to be", f, q, positions=torch.zeros(4, 1))
    refused(ValueError, "positions have to be", f, q, positions=torch.zeros(5, 2))
    refused(ValueError, "positions have to be", f, q, positions=torch.zeros(2, 1, 1))
    refused(ValueError, "positions have to be", f, q, positions=torch.tensor(1.0))
    refused(RuntimeError, "positions have no gradient", f, q, positions=torch.zeros(5, 1).requires_grad_())
    refused(TypeError, "frequencies are", f, q, frequencies=torch.zeros(4, dtype=torch.float64))
    refused(ValueError, "frequencies have to be", f, q, frequencies=torch.zeros(3))
    refused(RuntimeError, "frequencies have no gradient", f, q, frequencies=torch.zeros(4).requires_grad_())
    refused(ValueError, "kind", pcb().HeadRotary, 8, kind="layer")


def delta_data(T=5, hk=2, hv=4, dk=8, dv=6):
    return [torch.zeros(2, T, hk, dk), torch.zeros(2, T, hk, dk), torch.zeros(2, T, hv, dv), torch.zeros(2, T, hv), torch.zeros(2, T, hv)]


def test_delta_refusals():
    f = pcb().gated_delta
    t = delta_data()

    def but(**other):
        return [other.get(n, x) for n, x in zip("qkvgb", t)]

    refused(RuntimeError, "no CPU path", f, *t)
    for n in "qkvgb":
        refused(TypeError, f"{n} has to be", f, *but(**{n: None}))
        refused(TypeError, "Tensor", f, *but(**{n: [1.0]}))
    refused(TypeError, "float32/float16/bfloat16", f, *(x.double() for x in t))
    refused(TypeError, "k is", f, *but(k=t[1].half()))
    refused(TypeError, "v is", f, *but(v=t[2].half()))
    refused(TypeError, "g is", f, *but(g=t[3].half()))
    refused(TypeError, "b is", f, *(x.half() for x in t[:4]), t[4])
    refused(ValueError, "one shape", f, *but(k=t[1][..., :4]))
    refused(ValueError, "one shape", f, *but(k=t[1][:, :4]))
    refused(ValueError, "alike but for heads", f, *but(v=t[2][:, :4]))
    refused(ValueError, "alike but for heads", f, *but(v=t[2][0]))
    refused(ValueError, "multiple", f, *but(v=torch.zeros(2, 5, 3, 6)))
    refused(ValueError, "multiple", f, *but(v=torch.zeros(2, 5, 0, 6)))
    refused(ValueError, "g has to be", f, *but(g=t[3][..., :2]))
    refused(ValueError, "b has to be", f, *but(b=t[4][:1]))
    refused(ValueError, "1 to 128", f, *delta_data(dk=129))
    refused(ValueError, "1 to 128", f, *delta_data(dv=129))
    refused(ValueError, "1 to 128", f, *delta_data(dk=0))
    refused(ValueError, "channels", f, *(x[0, 0] for x in t), dim=0)
    refused(IndexError, "dim 4", f, *t, dim=4)
    refused(IndexError, f"dim {(1 << 32) + 1}", f, *t, dim=(1 << 32) + 1)
    refused(OverflowError, "too large", f, *t, dim=1 << 70)
    for dim in (2, 3, -1, -2):
        refused(ValueError, "any dimension but", f, *t, dim=dim)
    refused(ValueError, "state has to be", f, *t, state=torch.zeros(2, 4, 6, 8))
    refused(ValueError, "state has to be", f, *t, state=torch.zeros(1, 4, 8, 6))
    refused(TypeError, "state is float32", f, *t, state=torch.zeros(2, 4, 8, 6).half())
    refused(TypeError, "lengths is int32", f, *t, lengths=torch.zeros(2, dtype=torch.int64))
    refused(ValueError, "lengths has to be", f, *t, lengths=torch.zeros(3, dtype=torch.int32))
    refused(ValueError, "lengths has to be", f, *t, lengths=torch.zeros(2, 1, dtype=torch.int32))
    refused(TypeError, None, f, *t, scale="a")
    refused(TypeError, None, f, *t, dim=1.5)
    one = torch.zeros(1)
    many = [one.expand(1 << 16, 2, 1 << 16, 1, 1)] * 3 + [one.expand(1 << 16, 2, 1 << 16, 1)] * 2
    refused(ValueError, "2\\^31 - 1", f, *many, dim=1)


def test_step_refusals():
    f = pcb().gated_delta_step
    t = [x[:, 0] for x in delta_data()]
    h = torch.zeros(2, 4, 8, 6)
    refused(RuntimeError, "no CPU path", f, *t, h)
    refused(TypeError, "state has to be", f, *t)
    refused(TypeError, "the state is float32", f, *t, h.half())
    refused(TypeError, "the state is float32", f, *t, h, h.half())
    refused(ValueError, "the state has to be dense", f, *t, h[:1])
    refused(ValueError, "the state has to be dense", f, *t, h.transpose(-1, -2))
    refused(ValueError, "the state has to be dense", f, *t, h, torch.zeros(2, 4, 6, 8))
    refused(ValueError, "multiple", f, t[0], t[1], torch.zeros(2, 3, 6), *t[3:], h)
    store = torch.zeros(2 * h.numel())
    half = h.numel() // 2
    refused(ValueError, "overlaps", f, *t, store[:h.numel()].view(h.shape), store[half:half + h.numel()].view(h.shape))
    refused(ValueError, "overlaps", f, *t[:3], store[:8].view(2, 4), t[4], h, store[:h.numel()].view(h.shape))
    refused(RuntimeError, "no CPU path", f, *t, store[:h.numel()].view(h.shape), store[h.numel():].view(h.shape))


def test_function_forms_refuse_the_same():
    """The Function forms are public, and a trace's replays call them with whatever tensors they are given: as many checks, before any launch."""
    rotary, delta = pcb().HeadRotaryFunction.apply, pcb().GatedDeltaFunction.apply
    q = torch.zeros(2, 5, 4, 8)
    more = (1, (4,), 1e4, 1, False, 1e-6)
    refused(RuntimeError, "no CPU path", rotary, q, None, None, None, None, None, *more)
    refused(ValueError, "alike", rotary, q, q[:1], None, None, None, None, *more)
    refused(ValueError, "weight has to be", rotary, q, None, torch.ones(7), None, None, None, *more)
    refused(ValueError, "positions have to be", rotary, q, None, None, None, torch.zeros(4, 1), None, *more)
    refused(ValueError, "code", rotary, q, None, None, None, None, None, 1, (4,), 1e4, 3, False, 1e-6)
    t = delta_data()
    refused(RuntimeError, "no CPU path", delta, *t, None, None, 1, False, 1.0, True)
    refused(ValueError, "one shape", delta, t[0], t[1][:1], *t[2:], None, None, 1, False, 1.0, True)
    refused(ValueError, "any dimension but", delta, *t, None, None, 2, False, 1.0, True)
    refused(ValueError, "state has to be", delta, *t, torch.zeros(2), None, 1, False, 1.0, True)


def test_modules_have_the_parameters_they_name():
    layer = pcb().HeadRotary(16, axes=2)
    assert set(dict(layer.named_parameters())) == {"weight", "key_weight"} and layer.sections == (4, 4)
    assert pcb().HeadRotary(26, axes=3).sections == (5, 4, 4)
    for m in (pcb().HeadRotary(16, kind="none"), pcb().HeadRotary(16, kind="l2", weights=False), pcb().GatedDelta(dim=1)):
        assert list(m.parameters()) == []
    assert "axes=2" in repr(layer) and "'rms'" in repr(layer) and "reverse=True" in repr(pcb().GatedDelta(reverse=True))


def rotary_call(**other):
    from pyramidconvblock_amd import _lib

    c = _lib.Rotary()
    fields = dict(tokens=10, d=8, axes=1, kind=1, position_type=0, dtype=0, eps=1e-6, base=1e4, neighbours=0, positions=None, frequencies=None)
    lists = dict(x=(1, 1), heads=(4, 2), sections=(4, 0, 0), grid=(10, 0, 0), xt=(32, 16), xh=(8, 8), weight=(None, None))
    for n, v in {**fields, **other}.items():
        if n not in lists:
            setattr(c, n, v)
    for n, v in {**lists, **{n: v for n, v in other.items() if n in lists}}.items():
        getattr(c, n)[:] = v
    return c


def test_library_refuses_rotary_calls_before_any_launch():
    L = lib()
    two = (ctypes.c_void_p * 2)(1, 1)
    bad = (dict(d=0), dict(d=257), dict(axes=0), dict(axes=4), dict(tokens=-1), dict(heads=(-1, 2)), dict(heads=(65537, 1)), dict(kind=3), dict(kind=-1),
           dict(dtype=3), dict(position_type=4), dict(position_type=-1), dict(position_type=1), dict(sections=(5, 0, 0)), dict(sections=(-1, 0, 0)),
           dict(sections=(1 << 30, 0, 0)), dict(grid=(0, 0, 0)), dict(x=(None, 1)))
    for other in bad:
        c = rotary_call(**other)
        assert L.pdw_rotary_fwd(ctypes.addressof(c), ctypes.addressof(two), None) == 1, other
        assert b"pdw_rotary_fwd" in L.pdw_last_error(), other
        assert L.pdw_rotary_bwd(ctypes.addressof(c), ctypes.addressof(two), ctypes.addressof(two), ctypes.addressof(two), 1, 1 << 30, None) == 1, other
    assert L.pdw_rotary_fwd(None, ctypes.addressof(two), None) == 1 and b"null" in L.pdw_last_error()
    c = rotary_call()
    assert L.pdw_rotary_fwd(ctypes.addressof(c), None, None) == 1
    assert L.pdw_rotary_bwd(ctypes.addressof(c), None, ctypes.addressof(two), ctypes.addressof(two), None, 0, None) == 1
    need = L.pdw_rotary_bwd_workspace_bytes(8)
    assert need >= 2 * 8 * 4 and L.pdw_rotary_bwd_workspace_bytes(0) == 0 and L.pdw_rotary_bwd_workspace_bytes(257) == 0
    for work, size in ((None, 0), (None, need), (1, need - 1)):
        assert L.pdw_rotary_bwd(ctypes.addressof(c), *[ctypes.addressof(two)] * 3, work, size, None) == 1
        assert b"workspace" in L.pdw_last_error()
    for nothing in (dict(tokens=0, x=(None, None)), dict(heads=(0, 0))):
        c = rotary_call(**nothing)
        assert L.pdw_rotary_fwd(ctypes.addressof(c), ctypes.addressof(two), None) == 0, nothing


def test_library_refuses_weights_without_a_norm():
    L = lib()
    one, none = (ctypes.c_void_p * 2)(1, None), (ctypes.c_void_p * 2)()
    for weight in ((1, None), (None, 1)):
        for tokens in (10, 0):
            c = rotary_call(kind=0, weight=weight, tokens=tokens)
            assert L.pdw_rotary_fwd(ctypes.addressof(c), ctypes.addressof(one), None) == 1 and b"without a norm" in L.pdw_last_error()
            assert L.pdw_rotary_bwd(ctypes.addressof(c), *[ctypes.addressof(one)] * 2, ctypes.addressof(none), None, 0, None) == 1
            assert b"without a norm" in L.pdw_last_error()
    for gweight in (one, (ctypes.c_void_p * 2)(None, 1)):
        c = rotary_call(kind=0)
        assert L.pdw_rotary_bwd(ctypes.addressof(c), *[ctypes.addressof(one)] * 2, ctypes.addressof(gweight), 1, 1 << 30, None) == 1
        assert b"without a norm" in L.pdw_last_error()


def delta_call(**other):
    from pyramidconvblock_amd import _lib

    c = _lib.Delta()
    fields = dict(q=1, k=1, v=1, g=1, b=1, h0=None, lengths=None, O=2, T=100, W=3, Hk=2, Hv=4, dk=16, dv=24, reverse=0, logits=1, gates_f32=0, scale=1.0,
                  dtype=2)
    for n, v in {**fields, **other}.items():
        setattr(c, n, v)
    return c


def test_library_refuses_key_heads_without_value_heads():
    """(The gradients of q and k would have elements that no launch writes.)"""
    L, c = lib(), delta_call(Hv=0, Hk=2)
    assert L.pdw_delta_fwd(ctypes.addressof(c), 1, None, None, None, 0, None) == 1 and b"value heads" in L.pdw_last_error()
    assert L.pdw_delta_bwd(ctypes.addressof(c), 1, None, 1, 1, 1, 1, 1, 1, None, None, 0, None) == 1
    assert L.pdw_delta_step(ctypes.addressof(c), 1, 1, None) == 1


def test_library_refuses_delta_calls_before_any_launch():
    L = lib()
    fwd = lambda c, y=1, states=None, ws=None, n=0: L.pdw_delta_fwd(ctypes.addressof(c), y, None, states, ws, n, None)
    bwd = lambda c, gy=1, states=1, ws=None, n=0: L.pdw_delta_bwd(ctypes.addressof(c), gy, None, states, 1, 1, 1, 1, 1, None, ws, n, None)
    step = lambda c, y=1, last=1: L.pdw_delta_step(ctypes.addressof(c), y, last, None)
    bad = (dict(O=-1), dict(T=-1), dict(W=-1), dict(Hk=-1), dict(Hv=-1), dict(T=1 << 31), dict(T=(1 << 31) - 1), dict(dk=0), dict(dk=129), dict(dv=0),
           dict(dv=129), dict(Hk=0), dict(Hk=3), dict(dtype=5), dict(dtype=-1), dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(b=None),
           dict(O=1 << 16, W=1 << 16), dict(O=1 << 20, W=1 << 10, Hv=1 << 10, Hk=1))
    for other in bad:
        c = delta_call(**other)
        for call in (fwd, bwd, step):
            assert call(c) == 1, other
            assert b"pdw_delta_" in L.pdw_last_error(), other
        assert L.pdw_delta_states_bytes(ctypes.addressof(c)) == 0 and L.pdw_delta_workspace_bytes(ctypes.addressof(c), 0, 0) == 0, other
    assert L.pdw_delta_fwd(None, 1, None, None, None, 0, None) == 1 and b"null" in L.pdw_last_error()
    c = delta_call()
    need = L.pdw_delta_workspace_bytes(ctypes.addressof(c), 0, 0)
    kept = L.pdw_delta_workspace_bytes(ctypes.addressof(c), 0, 1)
    back = L.pdw_delta_workspace_bytes(ctypes.addressof(c), 1, 1)
    assert 0 < kept < need and back > 0 and L.pdw_delta_states_bytes(ctypes.addressof(c)) > 0
    for work, n in ((None, 0), (None, need), (1, need - 1)):
        assert fwd(c, ws=work, n=n) == 1 and b"workspace" in L.pdw_last_error()
    assert fwd(c, states=1, ws=1, n=kept - 1) == 1 and b"workspace" in L.pdw_last_error()
    assert bwd(c, ws=None, n=back) == 1 and b"workspace" in L.pdw_last_error()
    assert fwd(c, y=None, ws=1, n=need) == 1 and bwd(c, gy=None, ws=1, n=back) == 1 and bwd(c, states=None, ws=1, n=back) == 1
    assert step(c, last=None) == 1 and step(c, y=None) == 1
    # few steps need nothing between, none keep nothing
    assert L.pdw_delta_workspace_bytes(ctypes.addressof(delta_call(T=4)), 0, 0) == 0
    assert L.pdw_delta_states_bytes(ctypes.addressof(delta_call(T=0))) == 0
    # nothing to do
    for nothing in (dict(O=0), dict(W=0), dict(Hv=0, Hk=0)):
        c = delta_call(**nothing)
        assert fwd(c) == 0 and bwd(c) == 0 and step(c) == 0, nothing
    # more chunks than workgroups are counted in
    c = delta_call(O=1 << 20, W=1 << 8, Hv=1, Hk=1, T=2 << 6)
    huge = L.pdw_delta_workspace_bytes(ctypes.addressof(c), 0, 0)
    assert huge > 1 << 40 and fwd(c, ws=1, n=huge) == 1 and b"2^28 chunks" in L.pdw_last_error()
