"""Norms of queries and keys for each head with the rotation by their positions in the same pass, backed by libpdw.so (``csrc/rotary.h``):

    n = x (none),   x / sqrt(mean x^2 + eps) * weight (rms)   or   x / sqrt(sum x^2 + eps) * weight (l2)

for every row of d channels; the first 2 P channels of n are pairs (a, b), and pair i becomes (a cos t - b sin t, b cos t + a sin t) with
t = position * frequency_i, the position along the axis that the pair belongs to: a text's one, an image's rows and columns, a video's frames, rows and
columns.  float32, float16 and bfloat16, 1 to 256 channels a head; sums are 32-bit, angles are counted in 64 bits (so a far position is as good as a
near one), each result is rounded once, and results are the same from call to call.  For gradients of gradients and captures see ``norm.py``.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, ops
from .norm import _code, _dense


class HeadRotaryFunction(torch.autograd.Function):
    """apply(q, k, weight, key_weight, positions, frequencies, axes, sections, base, kind, neighbours, eps), kind a value of ops.HEAD_KINDS:
    head_rotary for calls that its native node does not take (a trace)."""

    @staticmethod
    def forward(ctx, q, k, weight, key_weight, positions, frequencies, axes, sections, base, kind, neighbours, eps):
        more = (axes, sections, base, kind, neighbours, eps)
        _lib.ext().check_rotary(q, k, weight, key_weight, positions, frequencies, *more)
        q, k, weight, key_weight, positions, frequencies = (_dense(t) for t in (q, k, weight, key_weight, positions, frequencies))
        y, yk = ops.rotary_forward(q, k, (weight, key_weight), positions, frequencies, *more)
        ctx.more, ctx.sizes = more, [None if t is None else tuple(t.shape) for t in (q, k)]
        ctx.save_for_backward(*((q, k) if kind else (None, None)), weight, key_weight, positions, frequencies)
        return y if yk is None else (y, yk)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gyk=None):
        q, k, weight, key_weight, positions, frequencies = ctx.saved_tensors
        grads = [None if g is None else g.contiguous() for g in (gy, gyk)]
        return (*ops.rotary_backward(grads, (q, k), (weight, key_weight), ctx.sizes, positions, frequencies, *ctx.more), *[None] * 8)


def _sections(d, axes, sections):
    """Pairs of each axis; all of a head's in equal parts, the first ones one larger, where nothing is said."""
    if sections is None:
        return tuple(d // 2 // axes + (a < d // 2 % axes) for a in range(axes))
    return tuple(sections)


def head_rotary(q, k=None, weight=None, key_weight=None, positions=None, axes=1, sections=None, frequencies=None, base=1e4, kind="none",
                neighbours=False, eps=1e-6):
    """-> q's heads, or the pair of q's and k's, normed and rotated; dense, of their shapes.

    q, k [..., heads, d]: of one type and alike but for their heads; slices of a wider tensor's channels are read where they lie.  weight and key_weight
    [d] (None: 1), with a norm only.  positions: None, then the last ``axes`` dimensions before the heads are a grid and count from 0; or
    int32, int64 or float32 [..., axes], for q's dimensions before the heads or the last ones of them.  sections: how many pairs belong to each axis
    (None: all pairs in equal parts); channels behind them are not rotated.  frequencies: float32, radians a position for every pair
    (None: base^(-j / section) for pair j of each section).  A pair is channels (i, P + i), or (2 i, 2 i + 1) with ``neighbours``."""
    code = _code(ops.HEAD_KINDS, kind, "kind")
    if sections is None and not (isinstance(q, torch.Tensor) and q.dim() and isinstance(axes, int) and axes > 0):
        sections = ()   # (refused below)
    args = (q, k, weight, key_weight, positions, frequencies, axes, sections if sections == () else _sections(q.shape[-1], axes, sections), base,
            code, neighbours, eps)
    y = _lib.ext().rotary(*args)
    if y is None:   # under forward-mode differentiation, a functorch transform or a trace
        y = HeadRotaryFunction.apply(*args)
    return y


class HeadRotary(nn.Module):
    """head_rotary with weights of its own (ones) for queries and keys: ``forward(q, k=None, positions=None)``.  ``kind="none"`` and ``weights=False``
    have none."""

    def __init__(self, head_dim: int, axes=1, sections=None, base=1e4, kind="rms", weights=True, neighbours=False, eps=1e-6):
        super().__init__()
        _code(ops.HEAD_KINDS, kind, "kind")
        self.head_dim, self.axes, self.base, self.kind, self.neighbours, self.eps = head_dim, axes, base, kind, neighbours, eps
        self.sections = _sections(head_dim, axes, sections)
        own = weights and kind != "none"
        self.weight = nn.Parameter(torch.ones(head_dim)) if own else None
        self.key_weight = nn.Parameter(torch.ones(head_dim)) if own else None

    def forward(self, q, k=None, positions=None):
        return head_rotary(q, k, self.weight, self.key_weight if k is not None else None, positions, self.axes, self.sections, None, self.base,
                           self.kind, self.neighbours, self.eps)

    def extra_repr(self):
        return (f"{self.head_dim}, axes={self.axes}, sections={self.sections}, base={self.base}, kind={self.kind!r}, "
                f"weights={self.weight is not None}, neighbours={self.neighbours}, eps={self.eps}")
