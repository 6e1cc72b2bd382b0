"""Log probabilities of given tokens, entropy and the most likely alternatives, one pass over the logits
(``csrc/logprobs.cu``)."""
from __future__ import annotations

import torch

from . import native as nv
from .derivatives import first_only, tracked

F32 = torch.float32


def _forward(logits, targets, top, inv_t, keep):
    """``(logprob, entropy, top logprobs, top ids, stats)``; ``stats`` with ``keep``: what the backward needs."""
    rows, vocab = logits.shape
    entropy = logits.new_empty(rows, dtype=F32)
    logprob = None if targets is None else torch.empty_like(entropy)
    stats = entropy.new_empty((rows, 2)) if keep else None
    top_lp = top_ids = None
    if top:
        top_lp = entropy.new_empty((rows, top))
        top_ids = entropy.new_empty((rows, top), dtype=torch.int64)
    if rows:
        nv.check(nv.lib(logits).fbam_logprobs_fwd(logits.data_ptr(), logits.dtype == F32, logits.stride(0), nv.addr(targets),
                                                  nv.addr(logprob), entropy.data_ptr(), nv.addr(stats), nv.addr(top_lp),
                                                  nv.addr(top_ids), rows, vocab, top, inv_t, nv.stream()),
                 "fbam_logprobs_fwd")
    return logprob, entropy, top_lp, top_ids, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, inv_t):
        ctx.set_materialize_grads(False)
        logprob, entropy, top_lp, top_ids, stats = _forward(logits, targets, top, inv_t, True)
        if top:
            ctx.mark_non_differentiable(top_lp, top_ids)
        ctx.save_for_backward(logits, targets, stats, entropy)
        ctx.linked = ()
        ctx.inv_t = inv_t
        return logprob, entropy, top_lp, top_ids

    @staticmethod
    @first_only("token_logprobs")
    def backward(ctx, d_logprob, d_entropy, _lp, _ids):
        logits, targets, stats, entropy = ctx.saved_tensors
        rows, vocab = logits.shape
        d_logprob = None if d_logprob is None else d_logprob.contiguous()
        d_entropy = None if d_entropy is None else d_entropy.contiguous()
        # rows that lie in their 16-byte pieces as the logits' do: dense where those are, else whole pieces
        per = 16 // logits.element_size()
        width = vocab if logits.stride(0) == vocab else (vocab + per - 1) // per * per
        d = logits.new_empty((rows, width))
        if rows:
            nv.check(nv.lib(logits).fbam_logprobs_bwd(logits.data_ptr(), logits.dtype == F32, logits.stride(0), nv.addr(targets),
                                                      stats.data_ptr(), entropy.data_ptr(), nv.addr(d_logprob),
                                                      nv.addr(d_entropy), d.data_ptr(), width, rows, vocab, ctx.inv_t,
                                                      nv.stream()), "fbam_logprobs_bwd")
        return d if width == vocab else d[:, :vocab], None, None, None


def token_logprobs(logits, targets, top, temperature):
    if targets is not None and targets.device != logits.device:
        raise ValueError(f"targets are on {targets.device}, the logits on {logits.device}")
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    flat = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if flat.stride(1) != 1:
        flat = flat.contiguous()
    if targets is not None and not (targets.dim() == 1 and targets.dtype == torch.int64 and targets.is_contiguous()):
        targets = targets.reshape(-1).long().contiguous()
    if tracked(flat):
        out = _TokenLogprobs.apply(flat, targets, top, 1.0 / temperature)
    else:
        out = _forward(flat, targets, top, 1.0 / temperature, False)[:4]
    if logits.dim() == 2:
        return out
    logprob, entropy, top_lp, top_ids = out
    return (None if logprob is None else logprob.view(shape), entropy.view(shape),
            None if top_lp is None else top_lp.view(*shape, top), None if top_ids is None else top_ids.view(*shape, top))
