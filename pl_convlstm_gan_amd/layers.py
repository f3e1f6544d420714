"""Layer operators beside the ConvLSTM cell: a gated linear recurrence over long sequences, group norm with an
activation on channels-last tensors, and dropout whose mask is computed from a counter instead of being stored.

None has a counterpart in the reference.  All are HIP kernels of libplconvlstm (include/plconvlstm.h, "Layer
operators"); float32, bfloat16 and float16 tensors, states, statistics and sums in float32.  They are differentiable
once, in reverse mode (a tensor with a forward-mode tangent raises), run on the current stream of their tensors' device,
and can be captured into a HIP graph (a training pass only while no output of an earlier pass over the same leaf tensors
on the default stream is alive, wherever between the leaves and the loss the operators are: that raises).  torch.jit.trace and torch.fx cannot record them: that raises too.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib, ops


def gated_linear_scan(x, f, h0=None, lengths=None, coupled=True):
    """h_t = s_t h_{t-1} + (1 - s_t) x_t (``coupled``) or h_t = s_t h_{t-1} + x_t, s = sigmoid(f), elementwise over
    [B, T, ...]; returns (h of every step in x's type, last state in float32 [B, ...]).

    ``h0``: float32 [B, ...], the state in front of the first step (default zeros).  ``lengths``: int32 [B] on x's
    device; behind a sample's length the outputs and gradients are 0, whatever the padding holds, and its state stands
    still.  An infinite x makes the states behind it infinite or NaN, and so does, coupled, an x - h beyond float32's range.
    Strided x and f are read in place as long as their trailing dimensions are contiguous."""
    return _lib.binding().scan(x, f, h0, lengths, coupled)


def gated_linear_step(x, f, state, coupled=True, inplace=False):
    """One step of gated_linear_scan for serving, without gradients: x, f [B, ...], ``state`` float32 [B, ...];
    returns (h in x's type, new state).  ``inplace``: the new state overwrites ``state`` (and is an in-place change of it
    to autograd: a backward pass that needs the old one refuses to run)."""
    return _lib.binding().step(x, f, state, coupled, inplace)


def counter_dropout(x, p, seed, offset=0, residual=None):
    """Dropout whose mask is a function of (``seed``, ``offset``, element): element e (in the logical order of x) stays
    when its 16-bit value of Philox4x32-10 is at least round(65536 p), and is scaled by the inverse of the exact
    probability of staying; a dropped element is 0.  ``residual`` is added to the result.

    Calls that must not share a mask take different offsets.  ``offset`` is an integer or an int64 tensor of one element on
    x's device that the kernel reads when it runs: a captured graph that advances it draws a new mask on every replay
    (the backward pass keeps the value its forward pass used; a pass that is recomputed reads it again)."""
    seed, offset, offset_t = ops._draw(seed, offset)
    return _lib.binding().dropout(x, p, seed, offset, offset_t, residual)


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", p=0.0, seed=0, offset=0):
    """Group norm over [N, C, H, W], activation (``"none"``, ``"relu"``, ``"silu"``) and, for ``p`` > 0, dropout in one
    pass.  ``weight`` and ``bias``: float32 [C] or None.  x is taken channels last in memory (another layout is copied into
    it first) and the result is channels last.  ``seed`` and ``offset`` as in counter_dropout; elements are counted in
    [N, H, W, C] order."""
    seed, offset, offset_t = ops._draw(seed, offset)
    return _lib.binding().norm(x, num_groups, weight, bias, eps, ops._act(act), p, seed, offset, offset_t)


def _first_offset(p, seed):
    """-> (seed, first offset): without a seed, a point of seed 0's 2^64 offsets drawn from torch's generator, so that modules
    have masks of their own, torch.manual_seed repeats them and the state_dict holds where they are."""
    if seed is None and p > 0:
        return 0, torch.randint(0, 1 << 62, (1,), dtype=torch.int64)
    return seed or 0, torch.zeros(1, dtype=torch.int64)


def _next_offset(module, offset):
    """The offset of a module's pass: the caller's, or the module's own, of which a pass that runs a second time inside the
    backward pass would read another value than the first time."""
    if offset is not None:
        return offset
    if ops._inside_backward():
        raise RuntimeError(f"{type(module).__name__} with dropout runs inside a backward pass (activation recomputation?), where its own "
                           "offset has moved on and the mask would be another one: give forward() the offset of the pass")
    return module.offset


class GroupNormAct(nn.Module):
    """group_norm_act with its parameters; ``p``: dropout of the training mode.  The dropout's offset is a buffer that
    every training pass advances by one on the device, so passes draw different masks, replays of a captured pass too.
    Without a ``seed`` its first value is drawn from torch's default generator, and modules draw masks of their own (copies of
    one module the same, as they share its offset; a module made with ``p`` = 0 draws nothing).  With one it counts from 0, and
    modules that share a seed share their masks.

    Where a pass is recomputed (torch.utils.checkpoint), give ``forward`` the ``offset`` of the pass, an integer or an int64 tensor
    that nothing changes before the backward pass is done; the buffer is then neither read nor advanced.  Without it a
    recomputation raises: the buffer has moved on by then."""

    def __init__(self, num_groups, num_channels, act="none", p=0.0, eps=1e-5, affine=True, seed=None):
        super().__init__()
        self.num_groups, self.num_channels, self.act, self.p, self.eps = num_groups, num_channels, act, p, eps
        self.seed, offset = _first_offset(p, seed)
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None
        self.register_buffer("offset", offset)

    def forward(self, x, offset=None):
        p = self.p if self.training else 0.0
        if p == 0:
            return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act)
        y = group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act, p, self.seed, _next_offset(self, offset))
        if offset is None:
            self.offset.add_(1)
        return y


class CounterDropout(nn.Module):
    """counter_dropout in training mode, the identity (plus ``residual``) otherwise; the seed and the offset as in GroupNormAct."""

    def __init__(self, p, seed=None):
        super().__init__()
        self.p = p
        self.seed, offset = _first_offset(p, seed)
        self.register_buffer("offset", offset)

    def forward(self, x, residual=None, offset=None):
        if not self.training or self.p == 0:
            return x if residual is None else x + residual
        y = counter_dropout(x, self.p, self.seed, _next_offset(self, offset), residual)
        if offset is None:
            self.offset.add_(1)
        return y
