"""What channel_norm, gated_residual and gated_scan refuse, and the library's answers to arguments, without a GPU."""
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


def test_norm_refusals():
    x, w = torch.zeros(4, 8), torch.ones(8)
    f = pcb().channel_norm
    refused(RuntimeError, "no CPU path", f, x, w)
    refused(ValueError, "kind", f, x, w, kind="batch")
    refused(ValueError, "rms or layer", f, x, w, kind="none")
    refused(ValueError, "weight has to be", f, x, torch.ones(7))
    refused(ValueError, "weight has to be", f, x, torch.ones(4, 8))
    refused(ValueError, "bias has to be", f, x, w, torch.ones(1))
    refused(TypeError, "weight is", f, x, w.half())
    refused(TypeError, "float32/float16/bfloat16", f, x.double(), w.double())
    refused(TypeError, "float32/float16/bfloat16", f, x.int(), None)
    refused(TypeError, "Tensor", f, [1.0], w)
    refused(TypeError, "x has to be", f, None)
    refused(ValueError, "C <= 8192", f, torch.zeros(1, 8193))
    refused(ValueError, "C <= 8192", f, torch.zeros(3, 0))
    refused(ValueError, "C <= 8192", f, torch.tensor(1.0))
    refused(ValueError, "eps", f, x, w, eps=-1e-6)
    refused(ValueError, "eps", pcb().gated_residual, x, x, eps=-1e-6)
    refused(ValueError, "kind", pcb().ChannelNorm, 8, kind="none")


def test_residual_refusals():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    f = pcb().gated_residual
    refused(RuntimeError, "no CPU path", f, x, x)
    refused(ValueError, "one shape", f, x, x[:, :2])
    refused(TypeError, "y is", f, x, x.half())
    refused(TypeError, "y has to be", f, x, None)
    refused(ValueError, "gate has to be", f, x, x, gate=torch.zeros(3, 8))
    refused(ValueError, "gate has to be", f, x, x, gate=torch.zeros(2, 1))
    refused(ValueError, "gate has to be", f, x, x, gate=torch.zeros(8))
    refused(TypeError, "gate is", f, x, x, gate=x.bfloat16())
    refused(ValueError, "scale has to be", f, x, x, scale=torch.ones(1))
    refused(ValueError, "without a gate", f, x, x, activation="silu")
    refused(ValueError, "activation has", f, x, x, gate=x, activation="relu")
    refused(ValueError, "kind has", f, x, x, kind="group")
    refused(ValueError, "next_kind has", f, x, x, next_kind="group")
    refused(ValueError, "without a next_kind", f, x, x, next_weight=w)
    refused(ValueError, "next_bias has", f, x, x, next_kind="rms", next_bias=torch.ones(3))
    block = pcb().GatedResidual(8)
    refused(ValueError, "another eps", block, x, x, next_norm=pcb().ChannelNorm(8, eps=1e-5))
    refused(ValueError, "depth", pcb().ResidualConvStack, 8, 0)
    refused(ValueError, "rows for 3 blocks", pcb().ResidualConvStack(8, 2), torch.zeros(1, 4, 4, 8), torch.zeros(3, 1, 8))


def test_scan_refusals():
    x = torch.zeros(2, 5, 3, 8)
    f = pcb().gated_scan
    refused(RuntimeError, "no CPU path", f, x, x)
    refused(ValueError, "any dimension but the channels", f, x, x, dim=-1)
    refused(ValueError, "any dimension but the channels", f, x, x, dim=3)
    refused(IndexError, "dim 4", f, x, x, dim=4)
    refused(IndexError, "dim -5", f, x, x, dim=-5)
    refused(ValueError, "one shape", f, x, x[..., :4])
    refused(TypeError, "g is", f, x, x.half())
    refused(ValueError, "even number", f, x[..., :7])
    refused(ValueError, "expected", f, torch.zeros(8), torch.zeros(8))
    refused(TypeError, "float32/float16/bfloat16", f, x.double(), x.double())
    refused(TypeError, "state is float32", f, x, x, torch.zeros(2, 5, 8).half())
    refused(ValueError, "state has to be", f, x, x, torch.zeros(2, 3, 8))
    refused(TypeError, "lengths is int32", f, x, x, lengths=torch.zeros(2, 5, dtype=torch.int64))
    refused(ValueError, "lengths has to be", f, x, x, lengths=torch.zeros(2, dtype=torch.int32))
    refused(ValueError, "lengths has to be", f, x, x, lengths=torch.zeros(2, 5, dtype=torch.int32), dim=1)
    refused(RuntimeError, "no CPU path", f, x, x, lengths=torch.zeros(2, dtype=torch.int32), dim=1)
    s = pcb().gated_scan_step
    x = torch.zeros(4, 8)
    refused(RuntimeError, "no CPU path", s, x, x, torch.zeros(4, 8))
    refused(TypeError, "state has to be", s, x, x)
    refused(TypeError, "float32, got", s, x, x, x.half())
    refused(ValueError, "dense and", s, x, x, torch.zeros(8, 4).t())
    refused(ValueError, "dense and", s, x, x, torch.zeros(4, 4))
    refused(ValueError, "dense and", s, x, None, torch.zeros(4, 8))
    refused(ValueError, "one shape", s, x, x[:2], torch.zeros(4, 8))
    store = torch.zeros(64)
    refused(ValueError, "overlap", s, x, x, store[:32].view(4, 8), store[8:40].view(4, 8))
    refused(ValueError, "overlap", s, store[8:40].view(4, 8), x, store[:32].view(4, 8))
    refused(ValueError, "overlap", s, x, store.view(4, 16)[:, 8:], x, store[:32].view(4, 8))
    refused(RuntimeError, "no CPU path", s, x, x, x)                                  # element by element: no harm in it
    refused(RuntimeError, "no CPU path", s, store[:32].view(4, 8), x, store[32:].view(4, 8))


def test_library_refuses_before_any_launch():
    import ctypes

    L = lib()
    one = (ctypes.c_longlong * 3)(8, 8, 8)
    norm = lambda N=4, C=8, kind=1, dtype=0, x=1: L.pdw_norm_fwd(x, 1, 1, 1, None, N, C, kind, 1e-6, dtype, None)
    for bad in (dict(N=-1), dict(C=0), dict(C=8193), dict(kind=0), dict(kind=3), dict(dtype=3), dict(x=None)):
        assert norm(**bad) == 1, bad
        assert L.pdw_last_error()
    assert norm(N=0) == 0
    assert L.pdw_norm_bwd(1, 1, 1, 1, 1, 1, 1, None, 0, 4, 8, 1, 0, None) == 1 and b"workspace" in L.pdw_last_error()
    assert L.pdw_norm_bwd(None, 1, 1, 1, 1, 1, 1, 1, 1 << 20, 4, 8, 1, 0, None) == 1
    need = L.pdw_norm_bwd_workspace_bytes(1000, 128, 2)
    assert need >= 2 * 128 * 4 and L.pdw_norm_bwd_workspace_bytes(0, 128, 2) == 0 and L.pdw_norm_bwd_workspace_bytes(8, 9999, 2) == 0
    res = lambda N=8, P=4, act=0, kind=1, nxt=0, out2=None, gate=1: L.pdw_residual_fwd(
        1, 1, gate, 1, 1, 1, 1, 1, 1, out2, None, None, N, 8, P, 0, act, kind, nxt, 1e-6, 0, None)
    for bad in (dict(P=3), dict(P=0), dict(act=3), dict(act=-1), dict(kind=-1), dict(nxt=5), dict(nxt=1)):
        assert res(**bad) == 1, bad
    assert res(N=0) == 0
    bwd = lambda ws, nbytes, P=4, stats=1, out=1: L.pdw_residual_bwd(1, 1, out, 1, 1, 1, 1, 1, 1, stats, 1, 1, 1, 1, 1, 1, 1, 1, 1,
                                                                           ws, nbytes, 8, 8, P, 0, 0, 1, 1, 0, None)
    assert bwd(None, 0) == 1 and b"workspace" in L.pdw_last_error()
    need = L.pdw_residual_bwd_workspace_bytes(8, 8, 4, 1, 0)
    assert need == 2 * 4 * 8 * 4   # a segment for each image, four sums
    assert bwd(1, need - 1) == 1 and bwd(1, need, stats=None) == 1 and bwd(1, need, out=None) == 1
    fwd = lambda O=2, T=5, W=1, I=8, x=1, dtype=0, s=one: L.pdw_scan_fwd(x, 1, None, None, 1, 1, None, None, 0, O, T, W, I, s, s, 0, dtype, None)
    for bad in (dict(O=-1), dict(T=-1), dict(W=-1), dict(I=-1), dict(x=None), dict(dtype=9), dict(s=None), dict(O=1 << 20, W=1 << 20), dict(T=1 << 31)):
        assert fwd(**bad) == 1, bad
    assert fwd(O=0) == 0 and fwd(I=0) == 0
    need = L.pdw_scan_workspace_bytes(1, 10000, 1, 64, 0)
    assert need > 0 and L.pdw_scan_workspace_bytes(4096, 100, 1, 64, 0) == 0 and L.pdw_scan_workspace_bytes(0, 100, 1, 64, 0) == 0
    assert L.pdw_scan_fwd(1, 1, None, None, 1, 1, None, 1, need - 1, 1, 10000, 1, 64, one, one, 0, 0, None) == 1
    assert b"workspace" in L.pdw_last_error()
    assert L.pdw_scan_bwd(1, None, 1, 1, None, None, 1, 1, None, 1, 1 << 30, 1, 10, 1, 64, one, one, one, one, 0, 0, None) == 1
    assert L.pdw_scan_states_bytes(3, 7, 2, 8) >= 3 * 2 * 8 * 4 and L.pdw_scan_states_bytes(3, 0, 2, 8) == 0
    assert L.pdw_scan_step(None, 1, 1, 1, 1, 4, 8, 8, 8, 0, None) == 1 and L.pdw_scan_step(1, 1, 1, 1, 1, -1, 8, 8, 8, 0, None) == 1
    assert L.pdw_scan_step(1, 1, 1, 1, 1, 0, 8, 8, 8, 0, None) == 0


def test_modules_have_the_parameters_they_name():
    stack = pcb().ResidualConvStack(16, depth=2, kernel_size=3, kind="layer", bias=True)
    names = set(dict(stack.named_parameters()))
    for i in range(2):
        assert {f"residuals.{i}.scale", f"residuals.{i}.weight", f"residuals.{i}.bias", f"blocks.{i}.conv_up.weight"} <= names
    assert {f"norms.{i}.{p}" for i in range(3) for p in ("weight", "bias")} <= names
    assert pcb().GatedResidual(8, kind="none", init_scale=None).state_dict() == {}
    assert list(pcb().GatedScan(dim=1, reverse=True).parameters()) == []
    assert "dim=1" in repr(pcb().GatedScan(dim=1)) and "rms" in repr(pcb().ChannelNorm(8)) and "silu" in repr(
        pcb().GatedResidual(8, activation="silu"))


def test_more_channels_than_32_bits_count_are_refused():
    """2^31 channels (views of one element: nothing is allocated): refused by name, not cut to 32 bits."""
    one = torch.zeros(1)
    x = one.expand(2, 1 << 31)
    refused(ValueError, "2\\^31 - 1", pcb().gated_scan, x, x, dim=0)
    refused(ValueError, "2\\^31 - 1", pcb().gated_scan_step, one.expand(1, 1 << 32), one.expand(1, 1 << 32), one.expand(1, 1 << 32))
    refused(ValueError, "2\\^31 - 1", pcb().gated_scan_step, one.expand(1, (1 << 32) + 8), one.expand(1, (1 << 32) + 8), torch.zeros(1, 8))


def test_dimensions_past_32_bits_are_refused():
    x = torch.zeros(2, 5, 8)
    for dim in (1 << 32, (1 << 32) + 1, -(1 << 32)):
        refused(IndexError, f"dim {dim}", pcb().gated_scan, x, x, dim=dim)
    refused(OverflowError, "too large", pcb().gated_scan, x, x, dim=1 << 70)


def test_function_forms_refuse_the_same():
    """The Function forms are public, and a trace's replays call them with whatever tensors they are given: as many checks, before any launch."""
    x, w = torch.zeros(4, 8), torch.ones(8)
    norm, residual, scan = (getattr(pcb(), n + "Function").apply for n in ("ChannelNorm", "GatedResidual", "GatedScan"))
    refused(RuntimeError, "no CPU path", norm, x, w, None, 1, 1e-6)
    refused(ValueError, "weight has to be", norm, x, torch.ones(7), None, 1, 1e-6)
    refused(TypeError, "bias is", norm, x, w, w.half(), 1, 1e-6)
    refused(ValueError, "C <= 8192", norm, torch.zeros(1, 8193), None, None, 1, 1e-6)
    refused(ValueError, "code", norm, x, w, None, 3, 1e-6)
    args = lambda y=x, gate=None, scale=w, act=0, kind=1, next_kind=0, eps=1e-6: (x, y, gate, scale, w, w, None, None, act, kind, next_kind, eps)
    refused(RuntimeError, "no CPU path", residual, *args())
    refused(ValueError, "one shape", residual, *args(y=x[:2]))
    refused(TypeError, "y is", residual, *args(y=x.half()))
    refused(ValueError, "gate has to be", residual, *args(gate=torch.zeros(2, 8)))
    refused(ValueError, "scale has to be", residual, *args(scale=torch.ones(4)))
    refused(ValueError, "eps", residual, *args(eps=-1.0))
    x = torch.zeros(2, 5, 8)
    refused(RuntimeError, "no CPU path", scan, x, x, None, None, 1, False)
    refused(ValueError, "one shape", scan, x, x[:, :4], None, None, 1, False)
    refused(TypeError, "g has to be", scan, x, None, None, None, 1, False)
    refused(ValueError, "state has to be", scan, x, x, torch.zeros(2, 7), None, 1, False)
    refused(TypeError, "lengths is int32", scan, x, x, None, torch.zeros(2, dtype=torch.int64), 1, False)
    refused(ValueError, "any dimension but the channels", scan, x, x, None, None, 2, False)


def test_axes_behind_a_traced_scan_stay_apart_where_their_product_is_too_large():
    """The function form's extents: one axis of chains up to 2^31 - 1 of them, two beyond (an int would be cut)."""
    from pyramidconvblock_amd import ops

    meta = lambda *shape: torch.empty(shape, device="meta")
    assert ops._scan_extents(meta(2, 3, 4, 5, 8), 1) == (2, 3, 1, 160)
    assert ops._scan_extents(meta(1, 2, 1 << 20, 1 << 12), 1) == (1, 2, 1 << 20, 1 << 12)
    assert ops._scan_extents(meta(3, 1, (1 << 31) - 1), 1) == (3, 1, 1, (1 << 31) - 1)
    assert list(ops._scan_strides(2, 1 << 20, 1 << 12)) == [1 << 33, 1 << 32, 1 << 12]


def test_calls_of_more_threads_than_a_launch_holds_are_refused():
    """HIP cuts the grid of 2^32 threads and more without an error, so single launches of that many are refused, before any of them: pools,
    bilinear maps, gates and direct convolutions of 2^32 results, a thread each."""
    L = lib()
    side = 1 << 11   # 2^11 x 2^11 pixels, 2^10 images, one channel: 2^32
    for call in (lambda b: L.pdw_avgpool_fwd(16, 16, b, side, side, 1, side, side, 0, None),
                 lambda b: L.pdw_bilinear_fwd(16, 16, b, side, side, 1, side, side, 0, 0, None),
                 lambda b: L.pdw_gate_fwd(16, 16, b * side * side, 2, 0, 0, None),
                 lambda b: L.pdw_dwconv_fwd(16, 16, 16, b, side + 1, side + 1, 1, 2, 2, 1, 1, 0, 0, 1, 1, 0, None),
                 lambda b: L.pdw_dwconv_dgrad(16, 16, 16, b, side, side, 1, 2, 2, 1, 1, 0, 0, 1, 1, 0, None)):
        assert call(1 << 10) == 1 and b"too large for one launch" in L.pdw_last_error(), L.pdw_last_error()
