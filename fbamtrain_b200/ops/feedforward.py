"""Gated feed-forward block on the tcgen05 GEMMs (``csrc/gated_mlp.cu``): ``y = (v · act(g)) W_outᵀ + b_out + residual``
with ``(v, g) = x W_inᵀ + b_in``; the first half of the projection is the value and the second the gate, as in ``geglu``.
"""
from __future__ import annotations

import torch

from ..utils import flops
from . import native as nv
from . import tuning
from .native_ops import _colsum, _need_elem, _tma_pitch, gemm, weight_grad_splits

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


def _product(a, b, m, n, a_mn=False, b_mn=False, bias=None, residual=None, splits=0):
    """:func:`gemm` with the launchers' own choices, which cost a short call less time to pass on."""
    if tuning.active():
        return gemm(a, b, a_mn=a_mn, b_mn=b_mn, bias=bias, residual=residual, splits=splits)
    a, b = _tma_pitch(a), _tma_pitch(b)
    k = a.shape[0] if a_mn else a.shape[1]
    out = a.new_empty((m, n))
    slabs = None
    splits = min(splits, (k + 63) // 64)
    if splits > 1 and m * n % 8 == 0:
        slabs = a.new_empty((splits, m, n), dtype=torch.float32)
    else:
        splits = 0
    nv.check(nv.lib(a).fbam_product(a.data_ptr(), a.stride(0), a_mn, b.data_ptr(), b.stride(0), b_mn, m, n, k, out.data_ptr(), n,
                                    nv.addr(bias), nv.addr(residual), n, nv.addr(slabs), splits,
                                    nv.status_word(a.device).data_ptr(), nv.stream()), "fbam_product")
    flops.add(2.0 * m * n * k)
    return out


def _project(x2, w1, b1, act, keep):
    """``(h, vg)``: the gated hidden values and, with ``keep``, both factors before the activation, ``(2, rows, inner)`` fp32."""
    rows, inner = x2.shape[0], w1.shape[0] // 2
    x2, w1 = _tma_pitch(x2), _tma_pitch(w1)
    h = x2.new_empty((rows, inner))
    vg = x2.new_empty((2, rows, inner), dtype=torch.float32) if keep else None
    v, g = (vg[0].data_ptr(), vg[1].data_ptr()) if keep else (0, 0)
    nv.check(nv.lib(x2).fbam_gated_fwd(x2.data_ptr(), x2.stride(0), w1.data_ptr(), w1.stride(0), nv.addr(b1), h.data_ptr(), v, g,
                                       rows, inner, x2.shape[1], act, nv.status_word(x2.device).data_ptr(), nv.stream()),
             "fbam_gated_fwd")
    flops.add(4.0 * rows * inner * x2.shape[1])
    return h, vg


def _project_grad(dy2, w2, vg, act, sums):
    """The gradient of the projection ``(rows, 2 · inner)``, values first, and with ``sums`` its column sums."""
    _, rows, inner = vg.shape
    dy2, w2 = _tma_pitch(dy2), _tma_pitch(w2)
    d_vg = dy2.new_empty((rows, 2 * inner))
    work = vg.new_empty(((rows + 31) // 32, 2 * inner)) if sums else None
    db = dy2.new_empty(2 * inner) if sums else None
    nv.check(nv.lib(dy2).fbam_gated_bwd(dy2.data_ptr(), dy2.stride(0), w2.data_ptr(), w2.stride(0), vg[0].data_ptr(),
                                        vg[1].data_ptr(), d_vg.data_ptr(), nv.addr(work), nv.addr(db), rows, inner, dy2.shape[1],
                                        act, nv.status_word(dy2.device).data_ptr(), nv.stream()), "fbam_gated_bwd")
    flops.add(2.0 * rows * inner * dy2.shape[1])
    return d_vg, db


# Rows up to which the weights are streamed past the rows instead of tiled.
FEW_ROWS = 32


def _few_rows(x2, w1, w2, b1, b_out, act, res2):
    """The block on up to ``FEW_ROWS`` rows, or None where a row does not start on a 16-byte boundary."""
    rows, depth = x2.shape
    dim, inner = w2.shape
    if depth % 8 or (x2.data_ptr() | w1.data_ptr() | w2.data_ptr()) % 16:
        return None
    h, y = x2.new_empty((rows, inner)), x2.new_empty((rows, dim))
    nv.check(nv.lib(x2).fbam_gated_few_rows(x2.data_ptr(), depth, w1.data_ptr(), depth, nv.addr(b1), w2.data_ptr(), inner,
                                            nv.addr(b_out), nv.addr(res2), dim, h.data_ptr(), y.data_ptr(), rows, depth, inner, dim,
                                            act, nv.stream()), "fbam_gated_few_rows")
    flops.add(2.0 * rows * inner * (2 * depth + dim))
    return y


def _forward(x, w_in, w_out, b_in, b_out, act, residual, keep):
    """``(y, x2, w1, w2, vg, h)``; the later ones for the backward."""
    inner, dim = w_out.shape[1], w_out.shape[0]
    x2 = _dense(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    res2 = None if residual is None else _dense(residual if residual.dim() == 2 else residual.reshape(-1, dim))
    w1, w2, b1, _ = _wider(_dense(w_in), _dense(w_out), None if b_in is None else _dense(b_in), inner)
    if b_out is not None:
        b_out = _dense(b_out)
    y = h = vg = None
    if not keep and x2.shape[0] <= FEW_ROWS:
        y = _few_rows(x2, w1, w2, b1, b_out, act, res2)
    if y is None:
        h, vg = _project(x2, w1, b1, act, keep)
        y = _product(h, w2, x2.shape[0], dim, bias=b_out, residual=res2)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], dim), x2, w1, w2, vg, h


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, act, residual):
        y, x2, w1, w2, vg, h = _forward(x, w_in, w_out, b_in, b_out, act, residual, True)
        ctx.save_for_backward(x2, w1, w2, vg, h)
        ctx.meta = (x.shape, w_out.shape[1], act)
        return y

    @staticmethod
    def backward(ctx, dy):
        x2, w1, w2, vg, h = ctx.saved_tensors
        shape, inner, act = ctx.meta
        need = ctx.needs_input_grad
        rows, wide = h.shape
        dim = w2.shape[0]
        dy2 = _dense(dy if dy.dim() == 2 else dy.reshape(-1, dim))
        dx = dw_in = dw_out = db_in = db_out = None
        if need[0] or need[1] or need[3]:
            d_vg, db_in = _project_grad(dy2, w2, vg, act, need[3])
            if need[0]:
                dx = _product(d_vg, w1, rows, w1.shape[1], b_mn=True)
                if len(shape) != 2:
                    dx = dx.view(shape)
            if need[1]:
                dw_in = _product(d_vg, x2, 2 * wide, x2.shape[1], True, True, splits=weight_grad_splits(2 * wide, x2.shape[1], rows))
                if wide != inner:
                    dw_in = dw_in.view(2, wide, -1)[:, :inner].reshape(2 * inner, -1)
            if need[3] and wide != inner:
                db_in = db_in.view(2, wide)[:, :inner].reshape(-1)
        if need[2]:
            dw_out = _product(dy2, h, dim, wide, True, True, splits=weight_grad_splits(dim, wide, rows))
            if wide != inner:
                dw_out = dw_out[:, :inner].contiguous()
        if need[4]:
            db_out = _bias_grad(dy2)
        return dx, dw_in, dw_out, db_in, db_out, None, dy if need[6] else None


def gated_mlp(x, w_in, w_out, b_in, b_out, act, residual):
    _need_elem(x, w_in, w_out, b_in, b_out, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_in, w_out, b_in, b_out, residual)):
        return _GatedMlp.apply(x, w_in, w_out, b_in, b_out, GATES[act], residual)
    return _forward(x, w_in, w_out, b_in, b_out, GATES[act], residual, False)[0]
