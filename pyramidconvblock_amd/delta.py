"""The gated delta rule along an axis of channels-last heads, backed by libpdw.so (``csrc/delta_fwd.h``): for every value head, with a state S of
dk x dv,

    u_t = beta_t (v_t - a_t S_(t-1)^T k_t),   S_t = a_t S_(t-1) + k_t u_t^T,   y_t = scale S_t^T q_t,     a_t = sigmoid(g_t), beta_t = sigmoid(b_t)

the recurrence of ``scan.py`` with a matrix for a state: what a key had stood for is replaced by beta of the way, everything fades by a.  float32, float16
and bfloat16, 1 to 128 channels a head; states are 32-bit throughout, results are the same from call to call.  It runs in chunks: results differ
from a loop's by roundings; keys longer than 1 can make the rule itself grow (a step takes S along k by 1 - beta |k|^2), so rows of unit length are
its usual input (``head_rotary`` with ``kind="l2"``).  Infinities come out as NaN.  What is not finite reaches y from its own step on (in v: in its
channel) and no step before it; among the gradients it can reach the whole chunk of 64 steps.  For gradients of gradients and captures see ``norm.py``.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, ops
from .norm import _dense


class GatedDeltaFunction(torch.autograd.Function):
    """apply(q, k, v, g, b, state, lengths, dim, reverse, scale, logits): gated_delta for calls that its native node does not take (a trace)."""

    @staticmethod
    def forward(ctx, q, k, v, g, b, state, lengths, dim, reverse, scale, logits):
        _lib.ext().check_delta(q, k, v, g, b, state, lengths, dim, reverse, scale, logits)
        dim %= q.dim()
        q, k, v, g, b, state, lengths = (_dense(t) for t in (q, k, v, g, b, state, lengths))
        y, last, states = ops.delta_forward(q, k, v, g, b, state, lengths, dim, reverse, scale, logits, states=True)
        ctx.more, ctx.has_state = (dim, reverse, scale, logits), state is not None
        ctx.save_for_backward(q, k, v, g, b, lengths, states)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, glast):
        q, k, v, g, b, lengths, states = ctx.saved_tensors
        *grads, gstate = ops.delta_backward(gy.contiguous(), glast.contiguous(), q, k, v, g, b, lengths, states, *ctx.more)
        return (*grads, gstate if ctx.has_state else None, *[None] * 5)


def _scale(q, scale):
    if scale is not None:
        return scale
    return q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0


def gated_delta(q, k, v, g, b, state=None, lengths=None, dim=-3, reverse=False, scale=None, logits=True):
    """-> (y like v, the last state, float32, v's shape without ``dim``, its last dimension made [dk, dv]).

    q, k [..., T, ..., hk, dk], v [..., T, ..., hv, dv], g, b [..., T, ..., hv]: the rule runs along ``dim`` of q (any but the heads' and the
    channels'), from its end with ``reverse``.  hv is a multiple of hk: neighbouring value heads share a key head.  g and b are logits, or with
    ``logits=False`` the log decay (at most 0) and the write strength themselves; of q's type or float32 (beside 16-bit tensors their gradients hold
    some 17 bits of the terms that they are sums of).  scale: None is dk^-1/2.  state: before the first step, like the last one (None: 0).  lengths (int32, q.shape[:dim]): valid steps of each sequence, limited to 0..T; what lies behind them has
    no part in any result, y and the gradients are 0 there, and the last state is the one after the last valid step.  A g of -inf or its type's lowest value forgets all
    that was before its step.  Slices of a wider tensor's channels are read where they lie."""
    args = (q, k, v, g, b, state, lengths, dim, reverse, _scale(q, scale), logits)
    y = _lib.ext().delta(*args)
    if y is None:   # under forward-mode differentiation, a functorch transform or a trace
        y = GatedDeltaFunction.apply(*args)
    return y


def gated_delta_step(q, k, v, g, b, state=None, new_state=None, scale=None, logits=True):
    """One step for every stream: q, k [..., hk, dk], v [..., hv, dv], g, b [..., hv], state float32 [..., hv, dk, dv] (a tensor, always) -> (y, the
    new state), which is written into ``new_state``, or into ``state`` itself where that is None.  Without gradients."""
    y = _lib.ext().delta_step(q, k, v, g, b, state, new_state, _scale(q, scale), logits)
    return y, state if new_state is None else new_state


class GatedDelta(nn.Module):
    """gated_delta along one dimension: ``forward(q, k, v, g, b, state=None, lengths=None)`` -> (y, last state).  It has no parameters."""

    def __init__(self, dim=-3, reverse=False, scale=None, logits=True):
        super().__init__()
        self.dim, self.reverse, self.scale, self.logits = dim, reverse, scale, logits

    def forward(self, q, k, v, g, b, state=None, lengths=None):
        return gated_delta(q, k, v, g, b, state, lengths, self.dim, self.reverse, self.scale, self.logits)

    def extra_repr(self):
        return f"dim={self.dim}, reverse={self.reverse}, scale={self.scale}, logits={self.logits}"
