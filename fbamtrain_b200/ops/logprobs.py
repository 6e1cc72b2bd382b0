"""Log probabilities of given tokens, entropy and the most likely alternatives, one pass over the logits
(``csrc/logprobs.cu``)."""
from __future__ import annotations

import ctypes as C

import torch

from . import native as nv


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, inv_t):
        rows, vocab = logits.shape
        dev = logits.device
        ctx.set_materialize_grads(False)
        logprob = None if targets is None else torch.empty(rows, dtype=torch.float32, device=dev)
        entropy = torch.empty(rows, dtype=torch.float32, device=dev)
        stats = torch.empty(rows, 2, dtype=torch.float32, device=dev)
        top_lp = top_ids = None
        if top:
            top_lp = torch.empty(rows, top, dtype=torch.float32, device=dev)
            top_ids = torch.empty(rows, top, dtype=torch.int64, device=dev)
            ctx.mark_non_differentiable(top_lp, top_ids)
        if rows:
            nv.check(nv.lib(logits).fbam_logprobs_fwd(
                nv.ptr(logits), int(logits.dtype == torch.float32), C.c_longlong(logits.stride(0)), nv.ptr(targets),
                nv.ptr(logprob), nv.ptr(entropy), nv.ptr(stats), nv.ptr(top_lp), nv.ptr(top_ids), C.c_longlong(rows), vocab,
                top, C.c_float(inv_t), nv.stream_ptr()), "fbam_logprobs_fwd")
        ctx.save_for_backward(logits, targets, stats, entropy)
        ctx.inv_t = inv_t
        return logprob, entropy, top_lp, top_ids

    @staticmethod
    def backward(ctx, d_logprob, d_entropy, _lp, _ids):
        logits, targets, stats, entropy = ctx.saved_tensors
        rows, vocab = logits.shape
        d_logprob = None if d_logprob is None else d_logprob.contiguous()
        d_entropy = None if d_entropy is None else d_entropy.contiguous()
        # rows of 16 bytes each, whatever the vocabulary
        per = 16 // logits.element_size()
        d = torch.empty(rows, (vocab + per - 1) // per * per, dtype=logits.dtype, device=logits.device)[:, :vocab]
        if rows:
            nv.check(nv.lib(logits).fbam_logprobs_bwd(
                nv.ptr(logits), int(logits.dtype == torch.float32), C.c_longlong(logits.stride(0)), nv.ptr(targets),
                nv.ptr(stats), nv.ptr(entropy), nv.ptr(d_logprob), nv.ptr(d_entropy), nv.ptr(d), C.c_longlong(d.stride(0)),
                C.c_longlong(rows), vocab, C.c_float(ctx.inv_t), nv.stream_ptr()), "fbam_logprobs_bwd")
        return d, None, None, None


def token_logprobs(logits, targets, top, temperature):
    if targets is not None and targets.device != logits.device:
        raise ValueError(f"targets are on {targets.device}, the logits on {logits.device}")
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    flat = logits.reshape(-1, vocab)
    if flat.stride(1) != 1:
        flat = flat.contiguous()
    if targets is not None:
        targets = targets.reshape(-1).long().contiguous()
    logprob, entropy, top_lp, top_ids = _TokenLogprobs.apply(flat, targets, top, 1.0 / temperature)
    return (None if logprob is None else logprob.view(shape), entropy.view(shape),
            None if top_lp is None else top_lp.view(*shape, top), None if top_ids is None else top_ids.view(*shape, top))
