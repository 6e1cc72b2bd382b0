"""Attention over a sliding window and the first few tokens (``csrc/window_attention.cu``, ``csrc/window_attention_bwd.cu``).

Query heads may share key heads.  Heads come as views: of three tensors, or of one fused projection ``(B, T, heads + 2 kv_heads,
D)``, whose gradient is one tensor then (gradients of three selections would each be a zero-filled tensor of the full size).  The
forward keeps its output, what rounding took off it and one fp32 value per query row for the backward.
"""
from __future__ import annotations

import functools

import torch

from ..utils import flops
from . import native as nv
from .derivatives import first_only, tracked

F32 = torch.float32
_FAR = 2 ** 30 - 1                                        # windows beyond see everything


def _usable(x: torch.Tensor) -> bool:
    """Whether the copy engine can fetch ``x`` ``(..., heads, channels)`` where it lies: channels side by side, a start and strides of 16
    bytes, nothing expanded."""
    *outer, inner = x.stride()
    if inner != 1 or x.data_ptr() % 16:
        return False
    for s, n in zip(outer, x.shape):
        if s % 8 or (s == 0 and n > 1):
            return False
    return True


def _fetchable(x: torch.Tensor) -> torch.Tensor:
    return x if _usable(x) else x.clone(memory_format=torch.contiguous_format)


def _reach(window, sinks):
    """A window (0: none) and first tokens that fit the kernels' integers."""
    return 0 if window is None or window > _FAR else window, min(sinks, _FAR)


def _pairs(b, t, window):
    """Pairs of a query and a key in ``b`` sequences of ``t`` tokens, the first tokens apart."""
    w = t if window is None else min(window, t)
    return b * (w * (w + 1) // 2 + (t - w) * w)


def _of(x):
    """Where heads lie, as the entry points take them: the first one's address and the strides."""
    return x.data_ptr(), x.stride()[:3]


def _parts(qkv, kv):
    """The query, key and value heads of a fused projection in this form (views of them would cost the host as much as the launch)."""
    at, strides = _of(qkv)
    step = strides[2] * 2                                # 16-bit values
    heads = qkv.shape[2] - 2 * kv
    return (at, strides), (at + heads * step, strides), (at + (heads + kv) * step, strides)


def _forward(like, shape, q, k, v, window, sinks, lengths, scale, keep):
    """``(out, kept)``; the latter with ``keep``, for the backward: an fp32 value for each row of each tile, and behind them, 16-bit,
    what rounding took off ``out``."""
    b, t, h, kv, d = shape
    out = like.new_empty((b, t, h, d))
    kept, lse, low = None, 0, 0
    if keep:
        rows = _lse_rows(shape)
        kept = like.new_empty((rows + b * t * h * d // 2,), dtype=F32)
        lse = kept.data_ptr()
        low = lse + 4 * rows
    (qp, qs), (kp, ks), (vp, vs) = q, k, v
    nv.check(nv.lib(like).fbam_window_fwd(qp, *qs, kp, vp, *ks, *vs, out.data_ptr(), low, lse, nv.addr(lengths), b, t, kv, h // kv, d,
                                          *_reach(window, sinks), scale, nv.status_word(like.device).data_ptr(), nv.stream()), "fbam_window_fwd")
    flops.add(4.0 * h * d * _pairs(b, t, window))
    return out, kept


def _lse_rows(shape):
    b, t, h, kv, _ = shape
    tokens = 128 // (h // kv)                            # of a tile of 128 rows
    return b * kv * ((t + tokens - 1) // tokens) * 128


def _backward(shape, q, k, v, out, kept, lengths, d_out, dq, dk, dv, window, sinks, scale):
    """Writes the gradients of the heads where ``dq``, ``dk`` and ``dv`` say."""
    b, t, h, kv, d = shape
    d_out = _fetchable(d_out)
    lib = nv.lib(out)
    how = (b, t, kv, h // kv, d, *_reach(window, sinks))
    floats = lib.fbam_window_bwd_workspace(*how)
    work = kept.new_empty(floats)
    lse = kept.data_ptr()
    (qp, qs), (kp, ks), (vp, vs), (dqp, dqs), (dkp, dks), (dvp, dvs) = q, k, v, dq, dk, dv
    nv.check(lib.fbam_window_bwd(qp, *qs, kp, vp, *ks, *vs, out.data_ptr(), lse + 4 * _lse_rows(shape), d_out.data_ptr(), *d_out.stride()[:3], lse,
                                 nv.addr(lengths), work.data_ptr(), floats, dqp, *dqs, dkp, *dks, dvp, *dvs, *how, scale,
                                 nv.status_word(out.device).data_ptr(), nv.stream()), "fbam_window_bwd")
    flops.add(10.0 * h * d * _pairs(b, t, window))


def _shape(q, k):
    b, t, h, d = q.shape
    return b, t, h, k.shape[2], d


def _shape_qkv(qkv, kv):
    b, t, all_heads, d = qkv.shape
    return b, t, all_heads - 2 * kv, kv, d


class _Window(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, lengths, scale):
        out, kept = _forward(q, _shape(q, k), _of(q), _of(k), _of(v), window, sinks, lengths, scale, True)
        ctx.save_for_backward(q, k, v, out, kept, lengths)
        ctx.linked = ()
        ctx.how = (window, sinks, scale)
        return out

    @staticmethod
    @first_only("window_attention")
    def backward(ctx, d_out):
        q, k, v, out, kept, lengths = ctx.saved_tensors
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        _backward(_shape(q, k), _of(q), _of(k), _of(v), out, kept, lengths, d_out, _of(dq), _of(dk), _of(dv), *ctx.how)
        return dq, dk, dv, None, None, None, None


class _WindowQkv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, kv, window, sinks, lengths, scale):
        out, kept = _forward(qkv, _shape_qkv(qkv, kv), *_parts(qkv, kv), window, sinks, lengths, scale, True)
        ctx.save_for_backward(qkv, out, kept, lengths)
        ctx.linked = ()
        ctx.how = (window, sinks, scale)
        ctx.kv = kv
        return out

    @staticmethod
    @first_only("window_attention_qkv")
    def backward(ctx, d_out):
        qkv, out, kept, lengths = ctx.saved_tensors
        kv = ctx.kv
        grad = qkv.new_empty(qkv.shape)
        _backward(_shape_qkv(qkv, kv), *_parts(qkv, kv), out, kept, lengths, d_out, *_parts(grad, kv), *ctx.how)
        return grad, None, None, None, None, None


def _lengths(lengths, like):
    if lengths is None:
        return None
    if lengths.device != like.device:
        raise ValueError(f"lengths are on {lengths.device}, the heads on {like.device}")
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, 2 ** 31 - 1)          # cut to 32 bits 2^32 + 3 would be 3
    return lengths.to(torch.int32).contiguous()


def window_attention(q, k, v, window, sinks, lengths, scale):
    lengths = _lengths(lengths, q)
    for name, x in (("keys", k), ("values", v)):
        if x.device != q.device:
            raise ValueError(f"{name} are on {x.device}, the queries on {q.device}")
    q, k, v = _fetchable(q), _fetchable(k), _fetchable(v)
    if tracked(q, k, v):
        return _Window.apply(q, k, v, window, sinks, lengths, scale)
    return _forward(q, _shape(q, k), _of(q), _of(k), _of(v), window, sinks, lengths, scale, False)[0]


def window_attention_qkv(qkv, kv, window, sinks, lengths, scale):
    lengths = _lengths(lengths, qkv)
    qkv = _fetchable(qkv)
    if tracked(qkv):
        return _WindowQkv.apply(qkv, kv, window, sinks, lengths, scale)
    return _forward(qkv, _shape_qkv(qkv, kv), *_parts(qkv, kv), window, sinks, lengths, scale, False)[0]


@functools.lru_cache(maxsize=1024)
def _splits(units: int, blocks: int, slots: int, sums: float) -> int:
    """How many thread blocks share the keys of one tile (or pair of tiles) of queries, where ``units`` of them have up to ``blocks``
    key blocks each and the machine holds ``slots`` thread blocks.  In key blocks: the longer of one share and of all shares over all
    slots, three a share for its start and end; half a share that the last ones are on their own; and where there are shares, eight for
    joining them (another launch, and on the host two more tensors) and ``sums`` for each, which writes and reads them.  64 sequences of
    16384 tokens, 4 key heads of 128 (256 units for 296 slots), shares of each: 1 303 us, 3 281, 5 268, 8 272, 24 315; 20 of up to 16000,
    8 key heads: 1 228, 4 168, 8 167, 24 186; 100 of up to 2000, 4 key heads of 64: 1 50, 2 53, 4 63."""
    best, splits = None, 1
    for s in range(1, min(64, blocks) + 1):
        share = blocks / s + 3
        cost = max(share, units * s * share / slots) + share / 2 + (8 + s * sums if s > 1 else 0)
        if best is None or cost < best:
            best, splits = cost, s
    return splits


def cache_attention(q, k_pages, v_pages, tables, lengths, offsets, window, sinks):
    n, h, d = q.shape
    b, most = tables.shape
    pages, page, kv, _ = k_pages.shape
    q = _fetchable(q)
    q_row, q_head, _ = q.stride()
    out = q.new_empty((n, h, d))
    lib = nv.lib(q)
    per = 2 * (128 // (h // kv))
    single = offsets is None and h // kv <= 16              # one token a sequence: two thread blocks a multiprocessor
    units = kv * (b if offsets is None else n // per + min(n, b))
    keys = most * page if window is None else min(most * page, window + per + sinks + 256)
    slots = 296 if single else 148
    splits = _splits(units, max(1, (keys + 127) // 128), slots, n * h / (64 * slots))
    part_o = part_ml = None
    if splits > 1:
        part_o = q.new_empty((splits, n, h, d), dtype=F32)
        part_ml = part_o.new_empty((splits, n, h, 2))
    nv.check(lib.fbam_cache_attention(
        q.data_ptr(), q_row, q_head, k_pages.data_ptr(), *k_pages.stride()[:3], v_pages.data_ptr(), *v_pages.stride()[:3],
        tables.data_ptr(), tables.stride(0), lengths.data_ptr(), nv.addr(offsets), out.data_ptr(), nv.addr(part_o), nv.addr(part_ml),
        splits, n, b, most, page, pages, kv, h // kv, d, *_reach(window, sinks), d ** -0.5, nv.status_word(q.device).data_ptr(), nv.stream()),
        "fbam_cache_attention")
    return out
