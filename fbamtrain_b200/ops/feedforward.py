"""Gated feed-forward block on the tcgen05 GEMMs (``csrc/gated_mlp.cu``): ``y = (v · act(g)) W_outᵀ + b_out + residual``
with ``(v, g) = x W_inᵀ + b_in``; the first half of the projection is the value and the second the gate, as in ``geglu``.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as nv
from .native_ops import _colsum, _need_elem, gemm, gemm_nn, gemm_tn, weight_grad_splits

GATES = {"gelu": 0, "silu": 1}


def _dense(x: torch.Tensor) -> torch.Tensor:
    return x if x.is_contiguous() else x.contiguous()


def _wider(w_in, w_out, b_in, inner: int):
    """The weights with the inner width padded to a multiple of 8 by zero rows and columns, which add nothing: 16-byte rows
    for the tensor maps."""
    wide = (inner + 7) // 8 * 8
    if wide == inner:
        return w_in, w_out, b_in, inner
    dim = w_in.shape[1]
    w1 = w_in.new_zeros(2, wide, dim)
    w1[:, :inner] = w_in.view(2, inner, dim)
    w2 = w_out.new_zeros(w_out.shape[0], wide)
    w2[:, :inner] = w_out
    if b_in is not None:
        b1 = b_in.new_zeros(2, wide)
        b1[:, :inner] = b_in.view(2, inner)
        b_in = b1.view(-1)
    return w1.view(2 * wide, dim), w2, b_in, wide


def _bias_grad(d: torch.Tensor) -> torch.Tensor:
    """Column sums; the kernel takes columns in eights."""
    rows, cols = d.shape
    if cols % 8:
        wide = d.new_zeros(rows, (cols + 7) // 8 * 8)
        wide[:, :cols] = d
        return _colsum(wide, d.dtype)[:cols]
    return _colsum(d, d.dtype)


def _gated_act(vg, dh, out, rows, inner, act):
    nv.check(nv.lib(out).fbam_gated_act(nv.ptr(vg), nv.ptr(dh), nv.ptr(out), C.c_longlong(rows), inner, act, nv.stream_ptr()),
             "fbam_gated_act")
    return out


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, act, residual):
        inner, dim = w_out.shape[1], w_out.shape[0]
        x2 = _dense(x.reshape(-1, x.shape[-1]))
        res2 = None if residual is None else _dense(residual.reshape(-1, dim))
        w1, w2, b1, wide = _wider(_dense(w_in), _dense(w_out), b_in, inner)
        rows = x2.shape[0]
        vg = gemm(x2, w1, bias=b1, out_dtype=torch.float32)
        h = _gated_act(vg, None, torch.empty(rows, wide, dtype=x.dtype, device=x.device), rows, wide, act)
        y = gemm(h, w2, bias=b_out, residual=res2)
        ctx.save_for_backward(x2, w1, w2, vg, h)
        ctx.meta = (x.shape, inner, act, b_in is not None, b_out is not None)
        return y.view(*x.shape[:-1], dim)

    @staticmethod
    def backward(ctx, dy):
        x2, w1, w2, vg, h = ctx.saved_tensors
        shape, inner, act, has_b_in, has_b_out = ctx.meta
        need = ctx.needs_input_grad
        rows, dim = x2.shape[0], w2.shape[0]
        wide = w2.shape[1]
        dy2 = _dense(dy.reshape(-1, dim))
        dx = dw_in = dw_out = db_in = db_out = None
        if need[0] or need[1] or need[3]:
            dh = gemm_nn(dy2, w2, out_dtype=torch.float32)
            dvg = _gated_act(vg, dh, torch.empty(rows, 2 * wide, dtype=dy.dtype, device=dy.device), rows, wide, act)
            if need[0]:
                dx = gemm_nn(dvg, w1).view(shape)
            if need[1]:
                dw_in = gemm_tn(dvg, x2, splits=weight_grad_splits(2 * wide, x2.shape[1], rows))
                if wide != inner:
                    dw_in = dw_in.view(2, wide, -1)[:, :inner].reshape(2 * inner, -1)
            if has_b_in and need[3]:
                db_in = _bias_grad(dvg)
                if wide != inner:
                    db_in = db_in.view(2, wide)[:, :inner].reshape(-1)
        if need[2]:
            dw_out = gemm_tn(dy2, h, splits=weight_grad_splits(dim, wide, rows))
            if wide != inner:
                dw_out = dw_out[:, :inner].contiguous()
        if has_b_out and need[4]:
            db_out = _bias_grad(dy2)
        return dx, dw_in, dw_out, db_in, db_out, None, dy if need[6] else None


def gated_mlp(x, w_in, w_out, b_in, b_out, act, residual):
    _need_elem(x, w_in, w_out, b_in, b_out, residual)
    return _GatedMlp.apply(x, w_in, w_out, b_in, b_out, GATES[act], residual)
