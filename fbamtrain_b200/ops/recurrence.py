"""Gated linear recurrence over sequences (``csrc/recurrence.cu``): an LSTM layer's gating without its products between
steps, so that a sequence is a scan instead of a chain.

Projections of a whole sequence come as one tensor ``(B, T, 3, D)`` (candidates, gates, output gates), as
``attention_qkv`` takes its projections, and its gradient is one tensor too.  The forward keeps the fp32 state in front of
every eighth step and nothing else; the backward rebuilds the states in between.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as nv


def _ordered_like(x: torch.Tensor, *inner: int) -> torch.Tensor:
    """An empty ``(B, T, *inner)`` tensor that is time-major in memory where ``x`` is."""
    b, t = x.shape[:2]
    if x.stride(0) < x.stride(1) and b > 1:
        return torch.empty(t, b, *inner, dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty(b, t, *inner, dtype=x.dtype, device=x.device)


def _strides(t: torch.Tensor, *dims: int):
    return tuple(C.c_longlong(t.stride(d)) for d in dims)


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, zgo, state, resets, keep):
        b, t, _, d = zgo.shape
        if zgo.stride(3) != 1:
            zgo = zgo.contiguous()
        if state is not None:
            state = state.contiguous()
        ctx.set_materialize_grads(False)
        y = _ordered_like(zgo, d)
        out = torch.empty(b, d, dtype=torch.float32, device=zgo.device)
        lib = nv.lib(zgo)
        saved = None
        if keep:
            chunk = lib.fbam_recurrence_chunk()
            saved = torch.empty(b, (t + chunk - 1) // chunk, d, dtype=torch.float32, device=zgo.device)
        rs = (C.c_longlong(0), C.c_longlong(0)) if resets is None else _strides(resets, 0, 1)
        nv.check(lib.fbam_recurrence_fwd(nv.ptr(zgo), *_strides(zgo, 0, 1, 2), nv.ptr(state), nv.ptr(resets), *rs, nv.ptr(y),
                                         *_strides(y, 0, 1), nv.ptr(out), nv.ptr(saved), b, t, d,
                                         nv.ptr(nv.status_word(zgo.device)), nv.stream_ptr()),
                 "fbam_recurrence_fwd")
        ctx.save_for_backward(zgo, resets, saved)
        return y, out

    @staticmethod
    def backward(ctx, dy, d_out):
        zgo, resets, saved = ctx.saved_tensors
        b, t, _, d = zgo.shape
        if dy is None:
            dy = torch.zeros(b, t, d, dtype=zgo.dtype, device=zgo.device)
        elif dy.stride(2) != 1:
            dy = dy.contiguous()
        if d_out is not None:
            d_out = d_out.contiguous()
        d_zgo = _ordered_like(zgo, 3, d)
        d_state = torch.empty(b, d, dtype=torch.float32, device=zgo.device) if ctx.needs_input_grad[1] else None
        rs = (C.c_longlong(0), C.c_longlong(0)) if resets is None else _strides(resets, 0, 1)
        nv.check(nv.lib(zgo).fbam_recurrence_bwd(nv.ptr(zgo), *_strides(zgo, 0, 1, 2), nv.ptr(resets), *rs, nv.ptr(saved),
                                                 nv.ptr(dy), *_strides(dy, 0, 1), nv.ptr(d_out), nv.ptr(d_zgo),
                                                 *_strides(d_zgo, 0, 1), nv.ptr(d_state), b, t, d,
                                                 nv.ptr(nv.status_word(zgo.device)), nv.stream_ptr()),
                 "fbam_recurrence_bwd")
        return d_zgo, d_state, None, None


def gated_recurrence(zgo, state, resets):
    for name, x in (("state", state), ("resets", resets)):
        if x is not None and x.device != zgo.device:
            raise ValueError(f"{name} is on {x.device}, the sequence on {zgo.device}")
    keep = torch.is_grad_enabled() and (zgo.requires_grad or (state is not None and state.requires_grad))
    return _GatedRecurrence.apply(zgo, state, resets, keep)
