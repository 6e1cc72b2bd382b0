"""Backend selection for the functional ops (see the package docstring)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import reference as ref

import os

_BACKEND = "auto"  # "auto": native kernels for CUDA tensors, PyTorch on CPU; "torch": PyTorch everywhere

# Per-family preference from the environment, as the reference's FBAMTRAIN_PREFER_{GEMM,CONV2D,MHA}_BACKEND
# (reference: ``src/passes/matmul_pass.cpp:35-62``, ``conv2d_pass.cpp:140-172``, ``mha_attention_pass.cpp:290-313``).
# Values: "native" (the sm_100a kernels of this package; the default) or "torch" (the vendor-library path).
_FAMILIES = ("gemm", "conv2d", "mha")
_prefer = {}
_last = {}


def _read_preferences() -> None:
    _prefer.clear()
    for fam in _FAMILIES:
        raw = os.environ.get(f"FBAMTRAIN_PREFER_{fam.upper()}_BACKEND", "native").strip().lower()
        if raw not in ("native", "torch"):
            raise ValueError(f"FBAMTRAIN_PREFER_{fam.upper()}_BACKEND must be 'native' or 'torch', got '{raw}'")
        _prefer[fam] = raw


_read_preferences()


def last_backend(family: str) -> str:
    """Which implementation the most recent call of an op family used: "native", "torch" or "" (not called yet).
    Tests assert on it the way the reference's tests assert that the expected backend was chosen."""
    return _last.get(family, "")


def set_backend(name: str) -> None:
    global _BACKEND
    if name not in ("auto", "torch"):
        raise ValueError("backend must be 'auto' or 'torch'")
    _BACKEND = name


def get_backend() -> str:
    return _BACKEND


_warned_dtypes = set()


def _native(t: torch.Tensor, dtype: Optional[torch.dtype] = None, family: Optional[str] = None) -> bool:
    """The hand-written kernels compute in bf16 or fp16 (fp32 accumulate; one library per element type).  CUDA
    tensors of another activation dtype (fp32 debugging runs) take the PyTorch definitions, i.e. the vendor
    libraries."""
    use = _native_inner(t, dtype, family)
    if family is not None:
        _last[family] = "native" if use else "torch"
    return use


def _native_inner(t: torch.Tensor, dtype: Optional[torch.dtype], family: Optional[str]) -> bool:
    if not (t.is_cuda and _BACKEND == "auto"):
        return False
    if family is not None and _prefer.get(family, "native") == "torch":
        return False
    dtype = dtype or t.dtype
    if dtype in (torch.bfloat16, torch.float16):
        return True
    if dtype not in _warned_dtypes:
        _warned_dtypes.add(dtype)
        from ..utils.logging import LOG
        LOG("WARN", f"ops: {dtype} activations on a GPU run on the PyTorch / vendor-library path; the sm_100a kernels "
                    "of this package compute in bf16 or fp16")
    return False


def cell_embed(cells, cp_embed, pos_embed, colour_embed, out_dtype):
    if _native(cells, out_dtype):
        from .native_ops import cell_embed as f
        return f(cells, cp_embed, pos_embed, colour_embed, out_dtype)
    return ref.cell_embed(cells, cp_embed, pos_embed, colour_embed, out_dtype)


def conv2d_nhwc(x, w_ohwi, stride: int, padding: int, dilation: int):
    # the implicit-GEMM kernels tile the input channels in blocks of 64; other channel counts take the library
    if x.shape[3] % 64 == 0 and _native(x, family="conv2d"):
        from .native_ops import conv2d_nhwc as f
        return f(x, w_ohwi, stride, padding, dilation)
    return ref.conv2d_nhwc(x, w_ohwi, stride, padding, dilation)


def rms_norm(x, weight, eps: float):
    if _native(x):
        from .native_ops import rms_norm as f
        return f(x, weight, eps)
    return ref.rms_norm(x, weight, eps)


def rms_norm_residual(x, weight, eps: float):
    """``(rms_norm(x), x)``, for a block that goes on with both: their gradients are added in one kernel."""
    if _native(x):
        from .native_ops import rms_norm_residual as f
        return f(x, weight, eps)
    return ref.rms_norm(x, weight, eps), x


def layer_norm(x, weight, bias, eps: float):
    if _native(x):
        from .native_ops import layer_norm as f
        return f(x, weight, bias, eps)
    return ref.layer_norm(x, weight, bias, eps)


def gelu(x):
    if _native(x):
        from .native_ops import gelu as f
        return f(x)
    return ref.gelu(x)


def geglu(x):
    if _native(x):
        from .native_ops import geglu as f
        return f(x)
    return ref.geglu(x)


def avg_pool2x2_nhwc(x):
    if _native(x):
        from .native_ops import avg_pool2x2_nhwc as f
        return f(x)
    return ref.avg_pool2x2_nhwc(x)


def gelu_avg_pool2x2_nhwc(x):
    """``avg_pool2x2_nhwc(gelu(x))``; one pass on the native path."""
    if _native(x) and x.shape[3] % 8 == 0:
        from .native_ops import gelu_avg_pool2x2_nhwc as f
        return f(x)
    return avg_pool2x2_nhwc(gelu(x))


def global_avg_pool_nhwc(x):
    """``(N, H, W, C)`` → ``(N, C)`` mean over the spatial positions (fp32 accumulate)."""
    if _native(x):
        from .native_ops import global_avg_pool_nhwc as f
        return f(x)
    return x.float().mean(dim=(1, 2)).to(x.dtype)


def conv_gelu_stack_pool(x, weights, stride: int, paddings, dilations):
    """``[conv3x3 (no bias) → GELU] x n → mean over positions``: ``(N, H, W, C)`` → ``(N, C_last)``."""
    if _native(x, family="conv2d") and all(w.shape[3] % 64 == 0 for w in weights):
        from .native_ops import conv_gelu_stack_pool as f
        return f(x, weights, stride, paddings, dilations)
    for w, pad, dil in zip(weights, paddings, dilations):
        x = gelu(conv2d_nhwc(x, w, stride, pad, dil))
    return global_avg_pool_nhwc(x)


def embconv_enabled() -> bool:
    """``FBAMTRAIN_EMBCONV=0`` keeps the cell embedding and the first convolution as separate kernels."""
    return os.environ.get("FBAMTRAIN_EMBCONV", "1") != "0"


def cell_conv_gelu_stack_pool(cells, cp_embed, pos_embed, colour_embed, rows: int, cols: int, out_dtype, weights,
                              stride: int, paddings, dilations):
    """``cells (N, rows·cols, 3)`` → cell embedding → ``[conv3x3 (no bias) → GELU] x n`` → mean over positions
    ``(N, C_last)``.  On the native path the embedding and the first convolution are fused into table look-ups
    (``ops/embconv.py``) when the shapes allow; otherwise this is the composition of the separate ops."""
    if (_native(cells, out_dtype, family="conv2d") and embconv_enabled() and
            all(w.shape[3] % 64 == 0 for w in weights)):
        from . import embconv
        if embconv.supported(cells, cp_embed, weights[0]):
            from .native_ops import cell_conv_gelu_stack_pool as f
            return f(cells, cp_embed, pos_embed, colour_embed, rows, cols, weights, stride, paddings, dilations)
    x = cell_embed(cells, cp_embed, pos_embed, colour_embed, out_dtype).view(cells.shape[0], rows, cols, -1)
    return conv_gelu_stack_pool(x, weights, stride, paddings, dilations)


def linear(x, weight, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None):
    """``act(x·Wᵀ + b) [+ residual]``; on the native path the residual rides in the GEMM epilogue."""
    if _native(x, family="gemm"):
        from .native_ops import linear as f
        return f(x, weight, bias, act, residual)
    y = ref.linear(x, weight, bias, act)
    return y if residual is None else y + residual.reshape(y.shape)


def attention(q, k, v, causal: bool):
    if _native(q, family="mha"):
        from .native_ops import attention as f
        return f(q, k, v, causal)
    if q.is_cuda:  # PyTorch baseline on GPU: library flash attention
        import torch.nn.functional as F
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=causal)
        return o.transpose(1, 2).contiguous()
    return ref.attention(q, k, v, causal)


def attention_qkv(qkv, causal: bool):
    """Attention on a fused projection output ``(B, T, 3, H, D)`` (q, k, v along dimension 2) → ``(B, T, H, D)``."""
    if _native(qkv, family="mha"):
        from .mha import flash_attention_qkv
        return flash_attention_qkv(qkv, causal)
    return attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], causal)


def lstm_sequence(x, w_ih, w_hh, b_ih, b_hh, h0, c0, compute_dtype):
    if _native(x, compute_dtype) and x.dtype == compute_dtype:
        from .native_ops import lstm_sequence as f
        return f(x, w_ih, w_hh, b_ih, b_hh, h0, c0, compute_dtype)
    if x.is_cuda and h0.dim() == 1:
        # PyTorch baseline on GPU: the library (cuDNN) LSTM instead of a Python loop over time steps
        b = x.shape[1]
        params = [w_ih.to(compute_dtype), w_hh.to(compute_dtype), b_ih.to(compute_dtype), b_hh.to(compute_dtype)]
        hx = (h0.to(compute_dtype).expand(1, b, -1).contiguous(), c0.to(compute_dtype).expand(1, b, -1).contiguous())
        y, h_n, c_n = torch._VF.lstm(x.to(compute_dtype), hx, params, True, 1, 0.0, True, False, False)
        return y, h_n[0], c_n[0].float()
    return ref.lstm_sequence(x, w_ih, w_hh, b_ih, b_hh, h0, c0, compute_dtype)


def lm_head_ce(x, w_head, targets, vocab: int, scale: float):
    if _native(x):
        from .native_ops import lm_head_ce as f
        return f(x, w_head, targets, vocab, scale)
    return ref.lm_head_ce(x, w_head, targets, vocab, scale)


def embed_tokens(ids, table, scale: float = 1.0, out_dtype: Optional[torch.dtype] = None):
    """``scale · table[ids]``: ``ids`` ``(...)`` int32 or int64, ``table`` ``(V, D)`` → ``(..., D)`` in ``out_dtype`` (the
    table's by default).  Ids outside ``[0, V)`` give a row of zeros.  The table's gradient is dense, in its own type, and
    summed in fp32 in an order that the ids alone fix."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"token ids are int32 or int64, got {ids.dtype}")
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"the table is (rows, width), got {tuple(table.shape)}")
    out_dtype = out_dtype or table.dtype
    if not (table.dtype == out_dtype or table.dtype == torch.float32):
        raise TypeError(f"a {table.dtype} table gives rows of its own type, not {out_dtype}")
    if table.is_cuda and _BACKEND == "auto" and out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        from .embedding import embed_tokens as f
        return f(ids, table, scale, out_dtype)
    return ref.embed_tokens(ids, table, scale, out_dtype)


def gated_recurrence(zgo, state=None, resets=None):
    """``zgo`` ``(B, T, 3, D)``: candidates ``z``, gates ``g`` and output gates ``o`` of whole sequences (or of one step).
    ``h_t = σ(g) h_{t-1} + (1 - σ(g)) z``, ``y = σ(o) h``.  ``state`` ``(B, D)`` fp32 is the ``h`` before the first step
    (zeros by default); where ``resets`` ``(B, T)`` bool is set, a step starts a new sequence and drops ``h_{t-1}``.
    Returns ``(y (B, T, D), state (B, D) fp32)``; sequences may be time-major views, which ``y`` then is too.

    An infinite candidate or state makes the state infinite until a reset, however small a share of it a finite gate keeps;
    infinities of both signs, and NaN, make it NaN until then.  The same holds backwards for gradients."""
    if zgo.dim() != 4 or zgo.shape[2] != 3 or zgo.shape[3] == 0:
        raise ValueError(f"the projections are (batch, steps, 3, width), got {tuple(zgo.shape)}")
    b, t, _, d = zgo.shape
    if state is not None and (state.shape != (b, d) or state.dtype != torch.float32):
        raise ValueError(f"the state is fp32 {(b, d)}, got {state.dtype} {tuple(state.shape)}")
    if resets is not None and (resets.shape != (b, t) or resets.dtype != torch.bool):
        raise ValueError(f"the resets are bool {(b, t)}, got {resets.dtype} {tuple(resets.shape)}")
    if b and t and _native(zgo):
        from .recurrence import gated_recurrence as f
        return f(zgo, state, resets)
    return ref.gated_recurrence(zgo, state, resets)


def gated_mlp(x, w_in, w_out, b_in=None, b_out=None, act: str = "gelu", residual=None):
    """``(v · act(g)) W_outᵀ + b_out + residual`` with ``(v, g) = x W_inᵀ + b_in``.  ``x`` ``(..., D)``, ``w_in``
    ``(2 F, D)`` with the value rows first and the gate rows behind them (the order of :func:`geglu`), ``w_out``
    ``(D', F)``, ``residual`` ``(..., D')``; ``act``: ``"gelu"`` (exact) or ``"silu"``."""
    if act not in ("gelu", "silu"):
        raise ValueError(f"the gate's activation is 'gelu' or 'silu', got '{act}'")
    if w_in.dim() != 2 or w_out.dim() != 2 or w_in.shape[0] != 2 * w_out.shape[1] or w_in.shape[1] != x.shape[-1] or 0 in w_in.shape:
        raise ValueError(f"weights {tuple(w_in.shape)} and {tuple(w_out.shape)} do not make a gated block on rows of {x.shape[-1]}")
    for name, bias, n in (("b_in", b_in, w_in.shape[0]), ("b_out", b_out, w_out.shape[0])):
        if bias is not None and bias.shape != (n,):
            raise ValueError(f"{name} is ({n},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], w_out.shape[0]):
        raise ValueError(f"the residual is {(*x.shape[:-1], w_out.shape[0])}, got {tuple(residual.shape)}")
    if x.numel() and w_out.shape[0] and _native(x, family="gemm"):
        from .feedforward import gated_mlp as f
        return f(x, w_in, w_out, b_in, b_out, act, residual)
    return ref.gated_mlp(x, w_in, w_out, b_in, b_out, act, residual)


MAX_ALTERNATIVES = 32


class TokenLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def token_logprobs(logits, targets=None, top: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Of ``softmax(logits / temperature)`` over the last dimension: ``logprob (...)`` of ``targets (...)`` (None without),
    ``entropy (...)`` in nats and the ``top`` most likely tokens, ``top_logprobs`` and ``top_ids`` ``(..., top)`` (None for
    0), ties to the lowest id; all fp32 but the int64 ids.  ``logprob`` and ``entropy`` are differentiable in the logits.

    A target outside the vocabulary (-1, -100) has log probability 0 and no gradient.  Logits of -inf have probability 0; a
    row of nothing else has entropy 0, log probabilities of -inf and no gradient.  A NaN makes ``logprob`` and ``entropy`` of
    its row NaN and counts as -inf among the alternatives."""
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits are (..., vocabulary), got {tuple(logits.shape)}")
    if targets is not None and (targets.shape != logits.shape[:-1] or targets.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"targets are int32 or int64 {tuple(logits.shape[:-1])}, got {targets.dtype} {tuple(targets.shape)}")
    if not 0 <= top <= min(MAX_ALTERNATIVES, logits.shape[-1]):
        raise ValueError(f"between 0 and {min(MAX_ALTERNATIVES, logits.shape[-1])} alternatives of {logits.shape[-1]} tokens, got {top}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"the temperature is above 0 and finite, got {temperature}")
    if logits.is_cuda and _BACKEND == "auto" and logits.dtype in (torch.float32, torch.bfloat16, torch.float16):
        from .logprobs import token_logprobs as f
        return TokenLogprobs(*f(logits, targets, top, temperature))
    return TokenLogprobs(*ref.token_logprobs(logits, targets, top, temperature))
