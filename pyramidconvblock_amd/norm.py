"""Norms over the channels of channels-last tensors, and the gated residual that closes a block, backed by libpdw.so
(``csrc/row_norm.h``): what goes before and after a mixing block such as ``ConvBlock``.

    norm     layer: (v - mean v) / sqrt(mean (v - mean v)^2 + eps) * weight + bias;   rms: v / sqrt(mean v^2 + eps) * weight + bias
    residual out = x + scale * act(gate) * norm(y);   next = norm'(out), where a block follows

Any leading dimensions, 1 to 8192 channels, float32, float16 and bfloat16; every tensor of a call is of one type.  Statistics and
sums are 32-bit, each result is rounded once, and results are the same from call to call.  The gradients have no derivatives
of their own (``create_graph=True`` raises).  A gate of its type's lowest value or -inf closes the branch under sigmoid and silu: 0, with
gradients of 0.  Everything can be captured in a HIP graph; before a backward pass is captured, drop
the outputs of eager passes over the same tensors: torch's gradient accumulators remember the stream they were made on, and where that is
the default stream, which a capture cannot make wait, the captured backward raises.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, ops


def _code(table, name, what):
    try:
        return table[name]
    except KeyError:
        raise ValueError(f"{what} has to be one of {', '.join(table)}, got {name!r}") from None


def _dense(t):
    return None if t is None else t.detach().contiguous()


class ChannelNormFunction(torch.autograd.Function):
    """apply(x, weight, bias, kind, eps), kind a value of ops.NORM_KINDS: channel_norm for calls that its native node does not take
    (a trace)."""

    @staticmethod
    def forward(ctx, x, weight, bias, kind, eps):
        _lib.ext().check_norm(x, weight, bias, kind, eps)
        x, weight, bias = _dense(x), _dense(weight), _dense(bias)
        y, stats = ops.norm_forward(x, weight, bias, kind, eps, stats=True)
        ctx.kind, ctx.has_bias = kind, bias is not None
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, weight, stats = ctx.saved_tensors
        return (*ops.norm_backward(gy.contiguous(), x, weight, stats, ctx.kind, ctx.has_bias), None, None)


def channel_norm(x, weight=None, bias=None, kind="rms", eps=1e-6):
    """The norm of every row of x [..., C] over its channels; weight and bias [C] (1 and 0 where they are None)."""
    code = _code(ops.NORM_KINDS, kind, "kind")
    if code == 0:
        raise ValueError("kind has to be rms or layer")
    y = _lib.ext().norm(x, weight, bias, code, eps)
    if y is None:   # under forward-mode differentiation, a functorch transform or a trace
        y = ChannelNormFunction.apply(x, weight, bias, code, eps)
    return y


class GatedResidualFunction(torch.autograd.Function):
    """apply(x, y, gate, scale, weight, bias, next_weight, next_bias, act, kind, next_kind, eps), the last four as codes and a number:
    gated_residual for calls that its native node does not take (a trace)."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, weight, bias, next_weight, next_bias, act, kind, next_kind, eps):
        _lib.ext().check_residual(x, y, gate, scale, weight, bias, next_weight, next_bias, act, kind, next_kind, eps)
        x, *rest = (_dense(t) for t in (x, y, gate, scale, weight, bias, next_weight, next_bias))
        out, nxt, stats, next_stats = ops.residual_forward(x, *rest, act, kind, next_kind, eps, stats=True)
        ctx.codes, ctx.has_next_bias = (act, kind, next_kind), next_bias is not None
        ctx.save_for_backward(x if next_kind else None, *rest[:-1], stats, next_stats)
        return out if nxt is None else (out, nxt)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gout, gnext=None):
        x, *rest, stats, next_stats = ctx.saved_tensors
        gout, gnext = gout.contiguous(), None if gnext is None else gnext.contiguous()
        grads = ops.residual_backward(gout, gnext, x, *rest, ctx.has_next_bias, stats, next_stats, *ctx.codes)
        return (*grads, None, None, None, None)


def gated_residual(x, y, weight=None, bias=None, gate=None, scale=None, kind="none", activation="none", next_weight=None,
                   next_bias=None, next_kind="none", eps=1e-6):
    """``x + scale * act(gate) * norm(y)``, and with a ``next_kind`` the pair of it and its norm.

    x, y [..., C].  gate: of their shape (it may be a slice of a wider tensor's channels), or [x.shape[0], C], one row for each image.
    weight, bias, scale, next_weight, next_bias [C]; None stands for 1, 0 and 1.  kind and next_kind: rms, layer or none; activation:
    none, sigmoid or silu.  The next norm is taken of the sum before it is rounded."""
    codes = (_code(ops.ACTIVATIONS, activation, "activation"), _code(ops.NORM_KINDS, kind, "kind"),
             _code(ops.NORM_KINDS, next_kind, "next_kind"))
    if codes[0] and gate is None:
        raise ValueError("an activation without a gate")
    if not codes[2] and (next_weight is not None or next_bias is not None):
        raise ValueError("next_weight or next_bias without a next_kind")
    args = (x, y, gate, scale, weight, bias, next_weight, next_bias, *codes, eps)
    out = _lib.ext().residual(*args)
    if out is None:   # as in channel_norm
        out = GatedResidualFunction.apply(*args)
    return out


class ChannelNorm(nn.Module):
    """channel_norm with a weight of its own (ones), and a bias (zeros) where asked for: before a block."""

    def __init__(self, dim: int, kind="rms", bias=False, eps=1e-6):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise ValueError(f"kind has to be rms or layer, got {kind!r}")
        self.kind, self.eps = kind, eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim)) if bias else None

    def forward(self, x):
        return channel_norm(x, self.weight, self.bias, self.kind, self.eps)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, kind={self.kind!r}, bias={self.bias is not None}, eps={self.eps}"


class GatedResidual(nn.Module):
    """gated_residual with weights of its own: after a block.  ``scale`` starts at ``init_scale`` (None: there is none), the norm of
    the branch at ones (``kind="none"``: there is none).  ``forward(x, y, gate=None, next_norm=None)`` gives the sum, or with a
    ``ChannelNorm`` as next_norm the pair of it and its norm."""

    def __init__(self, dim: int, kind="rms", bias=False, init_scale=1e-2, activation="none", eps=1e-6):
        super().__init__()
        _code(ops.NORM_KINDS, kind, "kind")
        _code(ops.ACTIVATIONS, activation, "activation")
        self.dim, self.kind, self.activation, self.eps = dim, kind, activation, eps
        self.scale = None if init_scale is None else nn.Parameter(torch.full((dim,), float(init_scale)))
        self.weight = nn.Parameter(torch.ones(dim)) if kind != "none" else None
        self.bias = nn.Parameter(torch.zeros(dim)) if bias and kind != "none" else None

    def forward(self, x, y, gate=None, next_norm=None):
        more = {}
        if next_norm is not None:
            if next_norm.eps != self.eps:
                raise ValueError(f"next_norm has another eps ({next_norm.eps}, here {self.eps})")
            more = dict(next_weight=next_norm.weight, next_bias=next_norm.bias, next_kind=next_norm.kind)
        return gated_residual(x, y, self.weight, self.bias, gate, self.scale, self.kind,
                              self.activation if gate is not None else "none", eps=self.eps, **more)

    def extra_repr(self):
        return (f"{self.dim}, kind={self.kind!r}, bias={self.bias is not None}, scale={self.scale is not None}, "
                f"activation={self.activation!r}, eps={self.eps}")


class ResidualConvStack(nn.Module):
    """``depth`` times x + scale * act(gate) * norm(ConvBlock(norm(x))), and a last norm: ConvBlocks as a model's stage.

    One pass over the stream closes a block and begins the next (gated_residual with its next norm).  ``forward(x, gate=None)`` takes
    x [B, H, W, dim] and optionally a gate row for each block and image [depth, B, dim], and returns (stream, its norm)."""

    def __init__(self, dim: int, depth: int, kernel_size=9, kind="rms", bias=False, init_scale=1e-2, activation="none", eps=1e-6):
        from .conv_block import ConvBlock

        super().__init__()
        if depth < 1:
            raise ValueError(f"depth has to be at least 1, got {depth}")
        self.norms = nn.ModuleList([ChannelNorm(dim, kind, bias, eps) for _ in range(depth + 1)])
        self.blocks = nn.ModuleList([ConvBlock(dim, kernel_size=kernel_size) for _ in range(depth)])
        self.residuals = nn.ModuleList([GatedResidual(dim, kind, bias, init_scale, activation, eps) for _ in range(depth)])

    def forward(self, x, gate=None):
        if gate is not None and gate.shape[0] != len(self.blocks):
            raise ValueError(f"gate has rows for {gate.shape[0]} blocks, there are {len(self.blocks)}")
        z = self.norms[0](x)
        for i, (block, residual) in enumerate(zip(self.blocks, self.residuals)):
            x, z = residual(x, block(z), None if gate is None else gate[i], self.norms[i + 1])
        return x, z
