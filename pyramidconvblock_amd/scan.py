"""The gated linear recurrence along an axis of a channels-last tensor, backed by libpdw.so (``csrc/scan.h``):

    h_t = a_t * h_(t-1) + (1 - a_t) * x_t,    a_t = sigmoid(g_t),    y_t = h_t,    every channel by itself

the recursive counterpart of the depthwise convolution: context from the whole axis at a cost that does not depend on its
length.  float32, float16 and bfloat16; states are 32-bit throughout, results are the same from call to call.  A chain is composed in
pieces: the results differ from a loop's by roundings, and past a state that has become infinite they may be NaN.  For gradients of
gradients and captures see ``norm.py``.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, ops


class GatedScanFunction(torch.autograd.Function):
    """apply(x, g, state, lengths, dim, reverse): gated_scan for calls that its native node does not take (a trace)."""

    @staticmethod
    def forward(ctx, x, g, state, lengths, dim, reverse):
        if g is None:
            raise TypeError("g has to be a tensor")
        _lib.ext().check_scan(x, g, state, lengths, dim, reverse)
        dim %= x.dim()
        x, g = x.detach().contiguous(), g.detach().contiguous()
        state, lengths = (None if t is None else t.detach().contiguous() for t in (state, lengths))
        y, last, states = ops.scan_forward(x, g, state, lengths, dim, reverse, states=True)
        ctx.dim, ctx.reverse, ctx.has_state = dim, reverse, state is not None
        ctx.save_for_backward(x, g, lengths, states)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, glast):
        x, g, lengths, states = ctx.saved_tensors
        gx, gg, gstate = ops.scan_backward(gy.contiguous(), glast.contiguous(), x, g, lengths, states, ctx.dim, ctx.reverse)
        return gx, gg, gstate if ctx.has_state else None, None, None, None


def gated_scan(x, g=None, state=None, lengths=None, dim=-2, reverse=False):
    """-> (y like x, the last state, float32, x's shape without ``dim``).

    x, g [..., T, ..., C], the recurrence runs along ``dim`` (any but the last), from its end with ``reverse``.  g None: x holds
    both in halves of its channels [..., 2 C], as one projection makes them.  state: the state before the first step, like the last one
    (None: 0).  lengths (int32, x.shape[:dim]): valid steps of each sequence, limited to 0..T; what lies behind them is not read, y and the
    gradients are 0 there, and the last state is the one after the last valid step.  Slices of a wider tensor's channels are
    read where they lie."""
    y = _lib.ext().scan(x, g, state, lengths, dim, reverse)
    if y is None:   # under forward-mode differentiation, a functorch transform or a trace
        if g is None:
            x, g = x.chunk(2, -1)
        y = GatedScanFunction.apply(x, g, state, lengths, dim, reverse)
    return y


def gated_scan_step(x, g=None, state=None, new_state=None):
    """One step for every chain: x, g [..., C] (or both in halves of x's channels), state float32 [..., C] -> (y, the new state), which is
    written into ``new_state``, or into ``state`` itself where that is None.  Without gradients."""
    y = _lib.ext().scan_step(x, g, state, new_state)
    return y, state if new_state is None else new_state


class GatedScan(nn.Module):
    """gated_scan along one dimension: ``forward(x, g=None, state=None, lengths=None)`` -> (y, last state).  It has no parameters."""

    def __init__(self, dim=-2, reverse=False):
        super().__init__()
        self.dim, self.reverse = dim, reverse

    def forward(self, x, g=None, state=None, lengths=None):
        return gated_scan(x, g, state, lengths, self.dim, self.reverse)

    def extra_repr(self):
        return f"dim={self.dim}, reverse={self.reverse}"
