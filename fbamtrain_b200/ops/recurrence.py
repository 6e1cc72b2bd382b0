"""Gated linear recurrence over sequences (``csrc/recurrence.cu``): an LSTM layer's gating without its products between
steps, so that a sequence is a scan instead of a chain.

Projections of a whole sequence come as one tensor ``(B, T, 3, D)`` (candidates, gates, output gates), as
``attention_qkv`` takes its projections, and its gradient is one tensor too.  The forward keeps the fp32 state in front of
every eighth step and nothing else; the backward rebuilds the states in between.
"""
from __future__ import annotations

import torch

from . import native as nv
from .derivatives import first_only, tracked

F32 = torch.float32


def _ordered_like(x: torch.Tensor, *inner: int) -> torch.Tensor:
    """An empty ``(B, T, *inner)`` tensor that is time-major in memory where ``x`` is."""
    b, t = x.shape[:2]
    if b > 1 and x.stride(0) < x.stride(1):
        return x.new_empty((t, b, *inner)).transpose(0, 1)
    return x.new_empty((b, t, *inner))


def _forward(zgo, state, resets, keep):
    """``(y, state, saved)``; ``saved`` with ``keep``: what the backward needs."""
    b, t, _, d = zgo.shape
    dev = zgo.device
    y = _ordered_like(zgo, d)
    out = zgo.new_empty((b, d), dtype=F32) if state is None else torch.empty_like(state)
    lib = nv.lib(zgo)
    saved = None
    if keep:
        chunk = lib.fbam_recurrence_chunk()
        saved = out.new_empty((b, (t + chunk - 1) // chunk, d))
    zb, zt, zk, _ = zgo.stride()
    yb, yt, _ = y.stride()
    rb, rt = (0, 0) if resets is None else resets.stride()
    nv.check(lib.fbam_recurrence_fwd(zgo.data_ptr(), zb, zt, zk, nv.addr(state), nv.addr(resets), rb, rt, y.data_ptr(), yb, yt,
                                     out.data_ptr(), nv.addr(saved), b, t, d, nv.status_word(dev).data_ptr(), nv.stream()),
             "fbam_recurrence_fwd")
    return y, out, saved


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, zgo, state, resets):
        ctx.set_materialize_grads(False)
        y, out, saved = _forward(zgo, state, resets, True)
        ctx.save_for_backward(zgo, resets, saved)
        ctx.linked = (state,)
        return y, out

    @staticmethod
    @first_only("gated_recurrence")
    def backward(ctx, dy, d_out):
        zgo, resets, saved = ctx.saved_tensors
        b, t, _, d = zgo.shape
        dev = zgo.device
        if dy is None:
            dy = zgo.new_zeros((b, t, d))
        elif dy.stride(2) != 1:
            dy = dy.contiguous()
        if d_out is not None:
            d_out = d_out.contiguous()
        d_zgo = _ordered_like(zgo, 3, d)
        d_state = saved.new_empty((b, d)) if ctx.needs_input_grad[1] else None
        zb, zt, zk, _ = zgo.stride()
        yb, yt, _ = dy.stride()
        db, dt, _, _ = d_zgo.stride()
        rb, rt = (0, 0) if resets is None else resets.stride()
        nv.check(nv.lib(zgo).fbam_recurrence_bwd(zgo.data_ptr(), zb, zt, zk, nv.addr(resets), rb, rt, saved.data_ptr(),
                                                 dy.data_ptr(), yb, yt, nv.addr(d_out), d_zgo.data_ptr(), db, dt,
                                                 nv.addr(d_state), b, t, d, nv.status_word(dev).data_ptr(), nv.stream()),
                 "fbam_recurrence_bwd")
        return d_zgo, d_state, None


def gated_recurrence(zgo, state, resets):
    for name, x in (("state", state), ("resets", resets)):
        if x is not None and x.device != zgo.device:
            raise ValueError(f"{name} is on {x.device}, the sequence on {zgo.device}")
    if zgo.stride(3) != 1:
        zgo = zgo.contiguous()
    if state is not None:
        state = state.contiguous()
    if tracked(zgo, state):
        return _GatedRecurrence.apply(zgo, state, resets)
    return _forward(zgo, state, resets, False)[:2]
