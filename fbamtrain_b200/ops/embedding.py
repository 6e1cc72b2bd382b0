"""Token embedding with scaling, and its gradient by sorted tokens (``csrc/embedding.cu``).

The gradient of a table row is a sum over the positions that name it.  Adding rows up with atomics would make its last bits
depend on the order in which blocks run; here the positions are sorted by token first and every sum has one order.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as nv


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, out_dtype):
        vocab, dim = table.shape
        flat = ids.reshape(-1)
        if not flat.is_contiguous():
            flat = flat.contiguous()
        if table.stride(1) != 1:
            table = table.contiguous()
        n = flat.numel()
        out = torch.empty(*ids.shape, dim, dtype=out_dtype, device=table.device)
        elem = table.dtype if table.dtype != torch.float32 else out_dtype
        if n:
            nv.check(nv.lib(elem).fbam_embed_fwd(nv.ptr(flat), int(flat.dtype == torch.int64), nv.ptr(table),
                                                 C.c_longlong(table.stride(0)), int(table.dtype == torch.float32), nv.ptr(out),
                                                 int(out_dtype == torch.float32), C.c_longlong(n), vocab, dim, C.c_float(scale),
                                                 nv.stream_ptr()), "fbam_embed_fwd")
        ctx.save_for_backward(flat)
        ctx.meta = (vocab, dim, table.dtype, elem, scale)
        return out

    @staticmethod
    def backward(ctx, d_out):
        (flat,) = ctx.saved_tensors
        vocab, dim, dtype, elem, scale = ctx.meta
        n = flat.numel()
        if n == 0:
            return None, torch.zeros(vocab, dim, dtype=dtype, device=d_out.device), None, None
        d_out = d_out.contiguous()
        d_table = torch.empty(vocab, dim, dtype=dtype, device=d_out.device)
        lib = nv.lib(elem)
        words, floats = C.c_longlong(), C.c_longlong()
        lib.fbam_embed_bwd_workspace(C.c_longlong(n), dim, C.byref(words), C.byref(floats))
        work = torch.empty(words.value, dtype=torch.int32, device=d_out.device)
        partial = torch.empty(floats.value, dtype=torch.float32, device=d_out.device)
        nv.check(lib.fbam_embed_bwd(nv.ptr(flat), int(flat.dtype == torch.int64), nv.ptr(d_out),
                                    int(d_out.dtype == torch.float32), nv.ptr(d_table), int(dtype == torch.float32),
                                    C.c_longlong(n), vocab, dim, C.c_float(scale), nv.ptr(work), nv.ptr(partial),
                                    nv.stream_ptr()), "fbam_embed_bwd")
        return None, d_table, None, None


def embed_tokens(ids, table, scale, out_dtype):
    if not ids.is_cuda or ids.device != table.device:
        raise ValueError(f"ids are on {ids.device}, the table on {table.device}")
    return _EmbedTokens.apply(ids, table, float(scale), out_dtype)
