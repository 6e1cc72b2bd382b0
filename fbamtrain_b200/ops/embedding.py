"""Token embedding with scaling, and its gradient by sorted tokens (``csrc/embedding.cu``).

The gradient of a table row is a sum over the positions that name it.  Adding rows up with atomics would make its last bits
depend on the order in which blocks run; here the positions are sorted by token first and every sum has one order.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as nv
from .derivatives import first_only, tracked

F32 = torch.float32


def _forward(ids, flat, table, scale, out_dtype, elem):
    vocab, dim = table.shape
    out = table.new_empty((*ids.shape, dim), dtype=out_dtype)
    n = flat.numel()
    if n:
        nv.check(nv.lib(elem).fbam_embed_fwd(flat.data_ptr(), flat.dtype == torch.int64, table.data_ptr(), table.stride(0),
                                             table.dtype == F32, out.data_ptr(), out_dtype == F32, n, vocab, dim, scale,
                                             nv.stream()), "fbam_embed_fwd")
    return out


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, flat, table, scale, out_dtype, elem):
        ctx.save_for_backward(flat)
        ctx.linked = ()
        ctx.meta = (*table.shape, table.dtype, elem, scale)
        return _forward(ids, flat, table, scale, out_dtype, elem)

    @staticmethod
    @first_only("embed_tokens")
    def backward(ctx, d_out):
        (flat,) = ctx.saved_tensors
        vocab, dim, dtype, elem, scale = ctx.meta
        n = flat.numel()
        if n == 0:
            return None, None, d_out.new_zeros((vocab, dim), dtype=dtype), None, None, None
        d_out = d_out.contiguous()
        d_table = d_out.new_empty((vocab, dim), dtype=dtype)
        lib = nv.lib(elem)
        words, floats = C.c_longlong(), C.c_longlong()
        lib.fbam_embed_bwd_workspace(n, dim, C.byref(words), C.byref(floats))
        work = flat.new_empty(words.value, dtype=torch.int64)
        partial = d_out.new_empty(floats.value, dtype=F32)
        nv.check(lib.fbam_embed_bwd(flat.data_ptr(), flat.dtype == torch.int64, d_out.data_ptr(), d_out.dtype == F32,
                                    d_table.data_ptr(), dtype == F32, n, vocab, dim, scale, work.data_ptr(),
                                    partial.data_ptr(), nv.stream()), "fbam_embed_bwd")
        return None, None, d_table, None, None, None


def embed_tokens(ids, table, scale, out_dtype):
    if ids.device != table.device:
        raise ValueError(f"ids are on {ids.device}, the table on {table.device}")
    flat = ids if ids.dim() == 1 else ids.reshape(-1)
    if not flat.is_contiguous():
        flat = flat.contiguous()
    if table.stride(1) != 1:
        table = table.contiguous()
    elem = table.dtype if table.dtype != F32 else out_dtype
    run = _EmbedTokens.apply if tracked(table) else _forward
    return run(ids, flat, table, float(scale), out_dtype, elem)
