"""Gated feed-forward block on the tensor cores (``csrc/gated_mlp.cu``): ``y = (v · act(g)) W_outᵀ + b_out + residual`` with
``(v, g) = x W_inᵀ + b_in``; the first half of the projection is the value and the second the gate, as in ``geglu``.

Widths that are no multiple of 8 are refitted: rows of ``x``, the weights and ``dy`` get zeros up to the next one (tensor maps
want 16-byte rows), which add nothing to any product; gradients are formed in padded widths and cut, since a product that stores
rows of other lengths stores them value by value (1000 x 2730 from 1001 rows: 56 us, padded and cut 29 + 6).
"""
from __future__ import annotations

import torch

from ..utils import debug, flops
from . import native as nv
from . import native_ops, tuning
from .derivatives import first_only, tracked
from .native_ops import _need_elem, _sum_partials, gemm, gemm_nn, gemm_tn, weight_grad_splits

GATES = {"gelu": 0, "silu": 1}
F32 = torch.float32

# Rows up to which the weights are streamed past the rows instead of tiled.  us, streamed | tiled: 8 x 1024 x 4096 17 | 36, 32 x
# 1024 x 4096 24 | 34, 8 x 2048 x 8192 34 | 71, 32 x 2048 x 8192 54 | 60.
FEW_ROWS = 32


# What the launchers make of native_ops.TWO_CTA: pairs of CTAs by size, never, always.
PAIRS = {"auto": -1, False: 0, True: 1}


def _watched() -> bool:
    """Whether a switch is on that looks at launches or at fresh memory."""
    return debug.PROFILE_LABELS or debug.SYNC_EVERY_OP or debug.POISON_ALLOC or debug.DEBUG_KERNEL_LAUNCH


def _apart(watched: bool) -> bool:
    """Whether the plain products are made one by one through ``gemm``: with a table of tuned tiles, and where a switch that it
    honours is not as usual."""
    return watched or native_ops.TWO_CTA != "auto" or not native_ops.USE_MN_MAJOR or tuning.active()


def _launch(watched: bool, entry: str, like: torch.Tensor, args: tuple) -> None:
    if watched:
        with debug.label(lambda: f"{entry[5:]} of {tuple(like.shape)}"):
            code = getattr(nv.lib(like), entry)(*args)
        nv.check(code, entry)
        debug.after_launch(entry[5:], like)
    else:
        nv.check(getattr(nv.lib(like), entry)(*args), entry)


def _fresh(like: torch.Tensor, shape: tuple, dtype=None) -> torch.Tensor:
    """``new_empty`` that honours the poison switch."""
    return debug.fresh(shape, dtype or like.dtype, like.device)


def _up8(n: int) -> int:
    return (n + 7) // 8 * 8


def _dense(x: torch.Tensor) -> torch.Tensor:
    return x if x.is_contiguous() else x.contiguous()


def _flat(x: torch.Tensor) -> torch.Tensor:
    """The rows of ``x``, dense, the first one on a 16-byte boundary.  The pitch is the width: a single row counts as dense
    whatever its stride says."""
    x = _dense(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    return x.clone() if x.data_ptr() % 16 else x


def _refit(src: torch.Tensor, blocks: int, rows: int, cols: int) -> torch.Tensor:
    """``src`` as ``blocks`` blocks of rows, each cut or padded with zeros to ``(rows, cols)``."""
    out = src.new_empty((blocks * rows, cols))
    nv.check(nv.lib(src).fbam_refit(src.data_ptr(), src.shape[1], out.data_ptr(), blocks, src.shape[0] // blocks, src.shape[1],
                                    rows, cols, nv.stream()), "fbam_refit")
    return out


def _forward(x, w_in, w_out, b_in, b_out, act, residual, keep):
    """``(y, x2, w1, w2, vg, h)``; the later ones for the backward, in their padded widths."""
    dim, inner = w_out.shape
    depth, wide = _up8(x.shape[-1]), _up8(inner)
    x2, w1, w2 = _flat(x), _flat(w_in), _flat(w_out)
    rows = x2.shape[0]
    if depth != x2.shape[1]:
        x2 = _refit(x2, 1, rows, depth)
    if depth != w1.shape[1] or wide != inner:
        w1 = _refit(w1, 2, wide, depth)
    if wide != inner:
        w2 = _refit(w2, 1, dim, wide)
        if b_in is not None:
            b_in = _refit(_dense(b_in).view(2, inner), 2, 1, wide)
    b_in = None if b_in is None else _dense(b_in)
    b_out = None if b_out is None else _dense(b_out)
    res2 = None if residual is None else _flat(residual)
    watched = _watched()
    h = _fresh(x2, (rows, wide)) if watched else x2.new_empty((rows, wide))
    product = False                        # the second product was made, and counted, by `gemm`
    if not keep and rows <= FEW_ROWS:
        y, vg = _fresh(x2, (rows, dim)) if watched else x2.new_empty((rows, dim)), None
        _launch(watched, "fbam_gated_few_rows", x2,
                (x2.data_ptr(), depth, w1.data_ptr(), depth, nv.addr(b_in), w2.data_ptr(), wide, nv.addr(b_out), nv.addr(res2), dim,
                 h.data_ptr(), y.data_ptr(), rows, depth, wide, dim, act, nv.stream()))
    else:
        apart = _apart(watched)
        vg = (_fresh(x2, (2, rows, wide), F32) if watched else x2.new_empty((2, rows, wide), dtype=F32)) if keep else None
        v = vg.data_ptr() if keep else 0
        product = apart
        y = None if apart else x2.new_empty((rows, dim))
        _launch(watched, "fbam_gated_block_fwd", x2,
                (x2.data_ptr(), depth, w1.data_ptr(), depth, nv.addr(b_in), w2.data_ptr(), wide, nv.addr(b_out), nv.addr(res2),
                 h.data_ptr(), v, v + 4 * rows * wide if keep else 0, nv.addr(y), rows, wide, depth, dim, act, PAIRS[native_ops.TWO_CTA],
                 nv.status_word(x2.device).data_ptr(), nv.stream()))
        if apart:
            y = gemm(h, w2, bias=b_out, residual=res2)
    flops.add(2.0 * rows * inner * (2 * x.shape[-1] + (0 if product else dim)))
    return y if x.dim() == 2 else y.view(*x.shape[:-1], dim), x2, w1, w2, vg, h


def _slabs(like, splits, m, n):
    """fp32 workspace of a weight gradient in ``splits`` parts, or None where it is not split."""
    return like.new_empty((splits, m, n), dtype=F32) if splits > 1 else None


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, act, residual):
        need_x, need_in, _, need_bin = ctx.needs_input_grad[:4]
        y, x2, w1, w2, vg, h = _forward(x, w_in, w_out, b_in, b_out, act, residual, need_x or need_in or need_bin)
        ctx.save_for_backward(x2, w1, w2, vg, h)
        ctx.linked = [t for t, rows in ((x, x2), (w_in, w1), (w_out, w2), (b_in, None)) if t is not rows and t.requires_grad]
        ctx.meta = (x.shape, w_out.shape[1], act)
        return y

    @staticmethod
    @first_only("gated_mlp")
    def backward(ctx, dy):
        x2, w1, w2, vg, h = ctx.saved_tensors
        shape, inner, act = ctx.meta
        need_x, need_in, need_out, need_bin, need_bout, _, need_res = ctx.needs_input_grad
        rows, wide = h.shape
        dim, width, depth = w2.shape[0], shape[-1], x2.shape[1]
        dy2 = _flat(dy)
        if dim % 8:
            dy2 = _refit(dy2, 1, rows, _up8(dim))
        dx = dw_in = dw_out = db_in = db_out = d_vg = sums = work = slabs_in = slabs_out = None
        splits_in = splits_out = 0
        watched = _watched()
        apart = _apart(watched)
        if need_x or need_in or need_bin:
            d_vg = _fresh(h, (rows, 2 * wide)) if watched else h.new_empty((rows, 2 * wide))
            if need_bin:
                db_in, sums = h.new_empty(2 * wide), vg.new_empty(((rows + 31) // 32, 2 * wide))
            if need_x:
                dx = None if apart else h.new_empty((rows, depth))
            if need_in and not apart:
                dw_in = h.new_empty((2 * wide, depth))
                splits_in = weight_grad_splits(2 * wide, depth, rows)
                slabs_in = _slabs(h, splits_in, 2 * wide, depth)
        if need_out and not apart:
            dw_out = h.new_empty((dim, wide))
            splits_out = weight_grad_splits(dim, wide, rows)
            slabs_out = _slabs(h, splits_out, dim, wide)
        if need_bout:
            db_out = h.new_empty(_up8(dim))
            parts = _sum_partials("fbam_colsum_partials", rows, _up8(dim), 0)
            work = h.new_empty(parts * _up8(dim), dtype=F32) if parts else None
        v = nv.addr(vg)
        _launch(watched, "fbam_gated_block_bwd", h,
                (dy2.data_ptr(), dy2.shape[1], x2.data_ptr(), depth, w1.data_ptr(), depth, w2.data_ptr(), wide, v, v and v + 4 * rows * wide,
                 h.data_ptr(), nv.addr(d_vg), nv.addr(sums), nv.addr(db_in), nv.addr(dx), nv.addr(dw_in), nv.addr(dw_out), nv.addr(db_out),
                 nv.addr(work), nv.addr(slabs_in), splits_in if slabs_in is not None else 0, nv.addr(slabs_out),
                 splits_out if slabs_out is not None else 0, rows, wide, depth, dim, act, PAIRS[native_ops.TWO_CTA],
                 nv.status_word(h.device).data_ptr(), nv.stream()))
        flops.add(2.0 * rows * inner * (dim * ((d_vg is not None) + (dw_out is not None)) + 2 * width * ((dx is not None) + (dw_in is not None))))
        if apart:
            splits = weight_grad_splits if native_ops.USE_MN_MAJOR else (lambda *sizes: 0)
            dx = gemm_nn(d_vg, w1) if need_x else None
            dw_in = gemm_tn(d_vg, x2, splits=splits(2 * wide, depth, rows)) if need_in else None
            dw_out = gemm_tn(dy2[:, :dim], h, splits=splits(dim, wide, rows)) if need_out else None
        if depth != width and dx is not None:
            dx = _refit(dx, 1, rows, width)
        if (wide != inner or depth != width) and dw_in is not None:
            dw_in = _refit(dw_in, 2, inner, width)
        if wide != inner:
            dw_out = None if dw_out is None else _refit(dw_out, 1, dim, inner)
            db_in = None if db_in is None else _refit(db_in.view(2, wide), 2, 1, inner).view(-1)
        if db_out is not None and dim % 8:
            db_out = db_out[:dim]
        if dx is not None and len(shape) != 2:
            dx = dx.view(shape)
        return dx, dw_in, dw_out, db_in, db_out, None, dy if need_res else None


def gated_mlp(x, w_in, w_out, b_in, b_out, act, residual):
    _need_elem(x, w_in, w_out, b_in, b_out, residual)
    if tracked(x, w_in, w_out, b_in, b_out, residual):
        return _GatedMlp.apply(x, w_in, w_out, b_in, b_out, GATES[act], residual)
    return _forward(x, w_in, w_out, b_in, b_out, GATES[act], residual, False)[0]
