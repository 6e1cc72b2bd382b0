"""An action model that reads its own earlier actions: token embedding → gated linear recurrent blocks → log probabilities.

Beside :class:`~fbamtrain_b200.models.action_model.ActionModel`, which sees frames only and carries its memory through an LSTM,
this one adds the vector of the previous action to each frame's and replaces the LSTM by gated linear recurrences, whose
sequences are scans.  A block is ``x += W_o · recurrence(W_zgo · norm(x)); x += gated_mlp(norm(x))``.  ``forward`` scores whole
sequences (several recordings in a row where ``resets`` marks their first steps), ``step`` answers one frame at a time from a
carried state of one fp32 vector per block.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import nn

from .. import ops
from .blocks import GatedMlp, Linear, RmsNorm, TokenEmbedding
from .init_utils import SeedSequence, fill_uniform_fan_


class RecurrentBlock(nn.Module):
    def __init__(self, dim: int, inner: int, bias: bool, eps: float, dtype: torch.dtype, seeds: SeedSequence, act: str = "gelu"):
        super().__init__()
        self.ln1 = RmsNorm(dim, eps, dtype)
        self.zgo = Linear(dim, 3 * dim, True, dtype, seeds)
        # gates start around 3: a memory of some twenty steps
        with torch.no_grad():
            self.zgo.bias[dim:2 * dim] += 3.0
        self.proj = Linear(dim, dim, bias, dtype, seeds)
        self.ln2 = RmsNorm(dim, eps, dtype)
        self.mlp = GatedMlp(dim, inner, bias, dtype, seeds, act)

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                resets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``x`` ``(B, T, D)`` → the same, and the recurrence's state ``(B, D)`` after the last step."""
        b, t, d = x.shape
        zgo = self.zgo(self.ln1(x).reshape(b * t, d)).view(b, t, 3, d)
        y, state = ops.gated_recurrence(zgo, state, resets)
        x2 = self.proj(y.reshape(b * t, d), x.reshape(b * t, d))
        return self.mlp(self.ln2(x2), x2).view(b, t, d), state


class RecurrentDecoder(nn.Module):
    """``frames (B, T, E)``: one vector per frame, as the frame head gives them; ``previous (B, T)``: the action taken before
    each frame, any id outside the vocabulary where there was none."""

    def __init__(self, frame_dim: int, dim: int, layers: int, inner: int, vocab: int, dtype: torch.dtype, seeds: SeedSequence,
                 bias: bool = True, eps: float = 1e-5, act: str = "gelu"):
        super().__init__()
        self.vocab = vocab
        self.frame_proj = Linear(frame_dim, dim, bias, dtype, seeds)
        self.actions = TokenEmbedding(vocab, dim, dtype, seeds, scale=dim ** 0.5)
        self.block = nn.ModuleList([RecurrentBlock(dim, inner, bias, eps, dtype, seeds, act) for _ in range(layers)])
        self.ln_f = RmsNorm(dim, eps, dtype)
        # the head's width is a multiple of 8, as in ActionModel
        self.head_weight = nn.Parameter(torch.empty((vocab + 7) // 8 * 8, dim, dtype=dtype))
        fill_uniform_fan_(self.head_weight.data, dim, seeds)

    def features(self, frames: torch.Tensor, previous: torch.Tensor, state: Optional[List[torch.Tensor]] = None,
                 resets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, List[torch.Tensor]]:
        b, t, e = frames.shape
        x = self.frame_proj(frames.reshape(b * t, e), self.actions(previous).reshape(b * t, -1)).view(b, t, -1)
        states = []
        for i, block in enumerate(self.block):
            x, s = block(x, None if state is None else state[i], resets)
            states.append(s)
        return self.ln_f(x), states

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return ops.linear(hidden.reshape(-1, hidden.shape[-1]), self.head_weight, None)[:, : self.vocab]

    def forward(self, frames: torch.Tensor, previous: torch.Tensor, targets: torch.Tensor, resets: Optional[torch.Tensor] = None,
                top: int = 0, temperature: float = 1.0) -> ops.TokenLogprobs:
        """Log probability of ``targets (B, T)`` (0 where they lie outside the vocabulary) and entropy, ``(B, T)`` each."""
        x, _ = self.features(frames, previous, None, resets)
        r = ops.token_logprobs(self.logits(x), targets.reshape(-1), top, temperature)
        return ops.TokenLogprobs(*(None if v is None else v.view(*targets.shape, *v.shape[1:]) for v in r))

    def step(self, frame: torch.Tensor, previous: torch.Tensor, state: Optional[List[torch.Tensor]] = None, top: int = 1,
             temperature: float = 1.0) -> Tuple[ops.TokenLogprobs, List[torch.Tensor]]:
        """One frame ``(B, E)`` and the action before it ``(B,)``: the ``top`` most likely actions with their log
        probabilities, and the state for the next step (None for the first)."""
        x, state = self.features(frame.unsqueeze(1), previous.unsqueeze(1), state)
        return ops.token_logprobs(self.logits(x), None, top, temperature), state
