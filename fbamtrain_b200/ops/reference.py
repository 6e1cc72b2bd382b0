"""Plain-PyTorch definitions of every op.  They are the numerics oracle for the CUDA kernels
(tests run them in fp32) and the execution path on CPU, where autograd differentiates them.

Layouts: activations NHWC / token-major, conv weights OHWI, linear weights ``(out, in)``, LSTM
weights ``(4H, in)`` with gate order i, f, g, o, time-major LSTM sequences ``(T, B, ·)``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F


def cell_embed(cells: torch.Tensor, cp_embed: torch.Tensor, pos_embed: torch.Tensor, colour_embed: torch.Tensor,
               out_dtype: torch.dtype) -> torch.Tensor:
    """``cells`` int32 ``(N, P, 3)`` → ``(N, P, E)``.

    ``out[n, p] = cp_embed[cp] (zero when cp is outside the table) + pos_embed[p mod P]
    + Σ_c (channel_c / 255) · colour_embed[c]`` with c over fg r,g,b then bg r,g,b, accumulated in
    fp32 (reference: ``kernel_gen/kernel_gen/kernels/build_cell_embeds.py:74-134``)."""
    n, p, _ = cells.shape
    cp = cells[..., 0].long()
    valid = (cp >= 0) & (cp < cp_embed.shape[0])
    e = cp_embed.float()[cp.clamp(0, cp_embed.shape[0] - 1)] * valid.unsqueeze(-1)
    e = e + pos_embed.float()[torch.arange(p, device=cells.device) % pos_embed.shape[0]].unsqueeze(0)
    fg, bg = cells[..., 1].long(), cells[..., 2].long()
    chans = torch.stack([(fg >> 16) & 255, (fg >> 8) & 255, fg & 255,
                         (bg >> 16) & 255, (bg >> 8) & 255, bg & 255], dim=-1).float() / 255.0
    e = e + chans @ colour_embed.float()
    return e.to(out_dtype)


def conv2d_nhwc(x: torch.Tensor, w_ohwi: torch.Tensor, stride: int, padding: int, dilation: int) -> torch.Tensor:
    y = F.conv2d(x.permute(0, 3, 1, 2), w_ohwi.permute(0, 3, 1, 2), None, stride, padding, dilation)
    return y.permute(0, 2, 3, 1).contiguous()


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    return y.to(x.dtype)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    return F.layer_norm(x.float(), (x.shape[-1],), weight.float(), None if bias is None else bias.float(), eps).to(x.dtype)


def gelu(x: torch.Tensor) -> torch.Tensor:
    """Exact (erf) GELU (reference: ``kernel_gen/kernel_gen/kernels/act.py:43-63``)."""
    return F.gelu(x.float(), approximate="none").to(x.dtype)


def gelu_grad(x: torch.Tensor) -> torch.Tensor:
    xf = x.float()
    return 0.5 * (1.0 + torch.erf(xf / math.sqrt(2.0))) + xf * torch.exp(-0.5 * xf * xf) / math.sqrt(2.0 * math.pi)


def geglu(x: torch.Tensor) -> torch.Tensor:
    """Channel-split gated GELU: first half is the value, second half the gate."""
    v, g = x.chunk(2, dim=-1)
    return (v.float() * F.gelu(g.float())).to(x.dtype)


def avg_pool2x2_nhwc(x: torch.Tensor) -> torch.Tensor:
    n, h, w, c = x.shape
    return x.float().reshape(n, h // 2, 2, w // 2, 2, c).mean(dim=(2, 4)).to(x.dtype)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], act: str = "none") -> torch.Tensor:
    y = x.float() @ weight.float().t()
    if bias is not None:
        y = y + bias.float()
    if act == "gelu":
        y = F.gelu(y)
    elif act == "relu":
        y = F.relu(y)
    return y.to(x.dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool) -> torch.Tensor:
    """``q, k, v``: ``(B, T, H, D)`` (possibly strided views of a fused qkv buffer); returns ``(B, T, H, D)``."""
    d = q.shape[-1]
    s = torch.einsum("bthd,bshd->bhts", q.float(), k.float()) / math.sqrt(d)
    if causal:
        t = q.shape[1]
        mask = torch.ones(t, k.shape[1], dtype=torch.bool, device=q.device).tril()
        s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("bhts,bshd->bthd", p, v.float()).to(q.dtype)


def lstm_cell(gates: torch.Tensor, c_prev: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``gates`` fp32 ``(B, 4H)`` pre-activations in order i, f, g, o → ``(h, c)`` fp32."""
    i, f, g, o = gates.float().chunk(4, dim=-1)
    c = torch.sigmoid(f) * c_prev.float() + torch.sigmoid(i) * torch.tanh(g)
    h = torch.sigmoid(o) * torch.tanh(c)
    return h, c


def lstm_sequence(x: torch.Tensor, w_ih: torch.Tensor, w_hh: torch.Tensor, b_ih: torch.Tensor, b_hh: torch.Tensor,
                  h0: torch.Tensor, c0: torch.Tensor, compute_dtype: torch.dtype):
    """Time-major LSTM.  ``x`` ``(T, B, I)``; weights fp32 ``(4H, I)``/``(4H, H)`` cast to
    ``compute_dtype`` for the matrix products; gates and cell state in fp32; ``h`` is rounded to
    ``compute_dtype`` between steps, as the reference does (reference:
    ``tensorlib/include/streaming_lstm.h:60-75``, ``kernel_gen/kernel_gen/kernels/lstm_cell.py:126-144``).
    ``h0``/``c0`` are ``(H,)`` and broadcast over the batch.  Returns ``(y (T,B,H), h_T, c_T)``."""
    t_len, b, _ = x.shape
    hdim = w_hh.shape[1]
    wi, wh = w_ih.to(compute_dtype), w_hh.to(compute_dtype)
    bias = (b_ih.float() + b_hh.float())
    h = h0.to(compute_dtype).unsqueeze(0).expand(b, hdim)
    c = c0.float().unsqueeze(0).expand(b, hdim)
    xg = (x.to(compute_dtype).reshape(t_len * b, -1) @ wi.t()).float().reshape(t_len, b, 4 * hdim)
    ys = []
    for t in range(t_len):
        gates = xg[t] + (h @ wh.t()).float() + bias
        hf, c = lstm_cell(gates, c)
        h = hf.to(compute_dtype)
        ys.append(h)
    return torch.stack(ys, 0), h, c


def cross_entropy_sum(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    return F.cross_entropy(logits.float(), targets.long(), reduction="sum")


def lm_head_ce(x: torch.Tensor, w_head: torch.Tensor, targets: torch.Tensor, vocab: int, scale: float) -> torch.Tensor:
    """``x`` ``(rows, H)``, ``w_head`` ``(V_pad, H)``; columns ≥ ``vocab`` are padding and ignored.
    Returns ``scale · Σ_rows CE`` (reference: ``src/main.cpp:1377-1463, 2428``)."""
    logits = (x.float() @ w_head.float().t())[:, :vocab]
    return cross_entropy_sum(logits, targets) * scale


def embed_tokens(ids: torch.Tensor, table: torch.Tensor, scale: float, out_dtype: torch.dtype) -> torch.Tensor:
    """``out[i] = scale · table[ids[i]]``; a row of zeros for ids outside the table."""
    valid = (ids >= 0) & (ids < table.shape[0])
    rows = table.float()[ids.clamp(0, table.shape[0] - 1).long()]
    return torch.where(valid.unsqueeze(-1), rows * scale, 0.0).to(out_dtype)


def gated_recurrence(zgo: torch.Tensor, state: Optional[torch.Tensor], resets: Optional[torch.Tensor]):
    """``zgo`` ``(B, T, 3, D)``: candidates, gates, output gates.  ``h_t = f h_{t-1} + (1 - f) z`` with ``f = σ(g)``, where a
    reset drops ``h_{t-1}``; ``y = σ(o) h``.  Returns ``y (B, T, D)`` and the last ``h`` in fp32."""
    b, t_len, _, d = zgo.shape
    z, g, o = zgo.float().unbind(2)
    f, f1, s = torch.sigmoid(g), torch.sigmoid(-g), torch.sigmoid(o)
    h = torch.zeros(b, d, dtype=torch.float32, device=zgo.device) if state is None else state
    ys = []
    for t in range(t_len):
        if resets is not None:
            h = torch.where(resets[:, t].bool().unsqueeze(1), 0.0, h)
        h = f[:, t] * h + f1[:, t] * z[:, t]
        ys.append(s[:, t] * h)
    y = torch.stack(ys, 1) if ys else zgo.new_empty(b, 0, d).float()
    return y.to(zgo.dtype), h


def gated_mlp(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, b_in: Optional[torch.Tensor],
              b_out: Optional[torch.Tensor], act: str, residual: Optional[torch.Tensor]) -> torch.Tensor:
    """``(v · act(g)) W_outᵀ + b_out + residual`` with ``(v, g) = x W_inᵀ + b_in``: value half first."""
    vg = x.float() @ w_in.float().t()
    if b_in is not None:
        vg = vg + b_in.float()
    v, g = vg.chunk(2, dim=-1)
    y = (v * (F.silu(g) if act == "silu" else F.gelu(g))) @ w_out.float().t()
    if b_out is not None:
        y = y + b_out.float()
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor], top: int, temperature: float):
    """``(log p[target], entropy, top log p, top ids)`` of ``softmax(logits / temperature)``; ties go to the lowest id, a NaN
    counts as -inf among the alternatives.  A target outside the vocabulary has 0 and no gradient; a row of -inf only has
    entropy 0, log probabilities of -inf and no gradient."""
    vocab = logits.shape[-1]
    x = logits.float() / temperature
    nothing = (x == float("-inf")).all(-1)
    logp = torch.log_softmax(x.masked_fill(nothing.unsqueeze(-1), 0.0), dim=-1)
    entropy = -(logp.exp() * logp.masked_fill(logp == float("-inf"), 0.0)).sum(-1).masked_fill(nothing, 0.0)
    logp = logp.masked_fill(nothing.unsqueeze(-1), float("-inf"))
    logprob = None
    if targets is not None:
        valid = (targets >= 0) & (targets < vocab)
        logprob = logp.gather(-1, targets.clamp(0, vocab - 1).long().unsqueeze(-1)).squeeze(-1).masked_fill(~valid, 0.0)
    if top == 0:
        return logprob, entropy, None, None
    with torch.no_grad():
        order = logits.float()
        order = torch.where(order.isnan(), float("-inf"), order)
        ids = order.sort(dim=-1, descending=True, stable=True)[1][..., :top]
        return logprob, entropy, logp.gather(-1, ids), ids


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs, heads: int, interleaved: bool) -> torch.Tensor:
    """``x`` ``(B, T, H, D)``: the pairs of the first ``2 len(freqs.turns)`` channels of the first ``heads`` heads turned by
    ``positions`` (broadcast to ``(B, T)``) times the frequencies; whole turns fall away as multiples of 2^64 do."""
    n = 2 * len(freqs.turns)
    turns = torch.tensor([t - (t >> 63 << 64) for t in freqs.turns], dtype=torch.int64, device=x.device)
    part = positions.expand(x.shape[:2]).long().unsqueeze(-1) * turns
    angle = (part.double() * (2 * math.pi / 2 ** 64)).unsqueeze(2)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    cos, sin = (freqs.magnitude * angle.cos()).to(wide), (freqs.magnitude * angle.sin()).to(wide)
    r = x[:, :, :heads, :n].to(wide)
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :n // 2], r[..., n // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    turned = torch.cat([r.to(x.dtype), x[:, :, :heads, n:]], -1)
    return torch.cat([turned, x[:, :, heads:]], 2)


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, at: torch.Tensor, end, window: Optional[int], sinks: int) -> torch.Tensor:
    """One sequence: ``q`` ``(n, H, D)`` at positions ``at``, ``k`` and ``v`` ``(m, Hkv, D)`` from position 0 on, of which the
    first ``end`` are there; queries that see nothing give zeros."""
    n, h, d = q.shape
    kv, like = k.shape[1], q
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    j = torch.arange(k.shape[0], device=q.device)
    seen = (j <= at.unsqueeze(1)) & (j < end) & (at.unsqueeze(1) < end)
    if window is not None:
        seen = seen & ((at.unsqueeze(1) - j < window) | (j < sinks))
    # what lies behind the end, and keys and values that no query sees, can hold anything
    q = torch.where((at < end).view(-1, 1, 1), q.to(wide), 0.0)
    some = seen.any(0).view(-1, 1, 1)
    k, v = torch.where(some, k.to(wide), 0.0), torch.where(some, v.to(wide), 0.0)
    s = torch.einsum("ngrd,mgd->grnm", q.reshape(n, kv, h // kv, d), k) * d ** -0.5
    nothing = ~seen.any(1)
    s = s.masked_fill(~seen & ~nothing.unsqueeze(1), float("-inf"))
    p = torch.softmax(s, dim=-1).masked_fill(nothing.unsqueeze(1), 0.0)
    o = torch.einsum("grnm,mgd->ngrd", p, v).reshape(n, h, d)
    return o.masked_fill(nothing.view(-1, 1, 1), 0.0).to(like.dtype)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int], sinks: int,
                     lengths: Optional[torch.Tensor]) -> torch.Tensor:
    """``q`` ``(B, T, H, D)``, ``k`` and ``v`` ``(B, T, Hkv, D)``: query ``i`` sees key ``j`` where ``j <= i`` and ``i - j <
    window`` or ``j < sinks``, both within the sequence's length; other queries give zeros."""
    b, t = q.shape[:2]
    at = torch.arange(t, device=q.device)
    rows = [_attend(q[i], k[i], v[i], at, t if lengths is None else lengths[i], window, sinks) for i in range(b)]
    return torch.stack(rows) if rows else q + 0 * (k.sum() + v.sum())        # empty, and a function of all three


def _new_tokens(n: int, tables: torch.Tensor, lengths: torch.Tensor, offsets: Optional[torch.Tensor]):
    """Of each sequence: its number, the rows of its new tokens and its length."""
    starts = list(range(tables.shape[0] + 1)) if offsets is None else offsets.tolist()
    return [(b, starts[b], min(starts[b + 1], n), max(length, 0)) for b, length in enumerate(lengths.tolist())]


def cache_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                 offsets: Optional[torch.Tensor], freqs, interleaved: bool, q_heads: int, kv_heads: int) -> torch.Tensor:
    """Turns the queries and keys of new tokens by their positions, writes keys and values into the pages and returns the
    queries; rows of no sequence, or in front of one's start, give zeros, and tokens without a page are not written."""
    pages, page = k_pages.shape[:2]
    q = qkv.new_zeros((qkv.shape[0], q_heads, qkv.shape[2]))
    for b, lo, hi, length in _new_tokens(qkv.shape[0], tables, lengths, offsets):
        for n in range(lo, hi):
            at = length - (hi - n)
            if at < 0:
                continue
            row = qkv[n:n + 1].unsqueeze(0)
            if freqs is not None:
                row = rotary(row, torch.tensor([[at]], device=qkv.device), freqs, q_heads + kv_heads, interleaved)
            q[n] = row[0, 0, :q_heads]
            where = int(tables[b, at // page]) if at // page < tables.shape[1] else -1
            if 0 <= where < pages:
                k_pages[where, at % page] = row[0, 0, q_heads:q_heads + kv_heads]
                v_pages[where, at % page] = row[0, 0, q_heads + kv_heads:]
    return q


def cache_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                    offsets: Optional[torch.Tensor], window: Optional[int], sinks: int) -> torch.Tensor:
    """New tokens ``(N, H, D)``, the last ones of their sequences, over the keys and values that the sequences have in the pages
    (zeros where an entry of the table is no page); rows of no sequence, or in front of one's start, give zeros."""
    pages, page = k_pages.shape[:2]
    out = torch.zeros_like(q)
    for b, lo, hi, length in _new_tokens(q.shape[0], tables, lengths, offsets):
        first = length - (hi - lo)
        skip = max(0, -first)
        if lo + skip >= hi:
            continue
        ids = tables[b].long()
        there = ((ids >= 0) & (ids < pages)).view(-1, 1, 1, 1)
        k, v = (torch.where(there, x[ids.clamp(0, pages - 1)], 0.0).flatten(0, 1) for x in (k_pages, v_pages))
        at = torch.arange(first + skip, length, device=q.device)
        # queries behind the end of the table see what is in front of it
        out[lo + skip:hi] = _attend(q[lo + skip:hi], k[:length], v[:length], at, length, window, sinks)
    return out
