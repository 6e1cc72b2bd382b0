"""An action model that reads its own earlier actions through attention over a window: token embedding → windowed attention blocks
with rotary positions → log probabilities.

Beside :class:`~fbamtrain_b200.models.recurrent_decoder.RecurrentDecoder` this one keeps the last ``window`` frames and the first
``sinks`` of a recording as they were instead of a state.  ``forward`` scores whole sequences; ``extend`` and ``step`` answer new frames
from a :class:`PagedCache`: a window bounds its pages, however long the recordings get (up to the tokens that its tables are made for).
Query heads may share key heads.
"""
from __future__ import annotations

import operator
from typing import List, Optional, Sequence

import torch
from torch import nn

from .. import ops
from ..ops.dispatch import CACHE_WIDTHS, check_alternatives, runs_native
from .blocks import GatedMlp, Linear, RmsNorm, TokenEmbedding
from .init_utils import SeedSequence, fill_uniform_fan_


class PagedCache:
    """Keys and values of several sequences in pages that they take from one pool, and give back when a window has passed them.

    ``k`` and ``v``: ``(layers, pages, slots, kv_heads, head_dim)``; ``tables`` ``(sequences, most)`` int32, -1 where a sequence has no
    page; ``lengths`` ``(sequences,)`` int32: tokens of each, those of the call under way among them."""

    def __init__(self, layers: int, pages: int, slots: int, kv_heads: int, head_dim: int, sequences: int, most_tokens: int, dtype: torch.dtype,
                 device, window: Optional[int] = None, sinks: int = 0):
        if slots < 1 or slots % 8:
            raise ValueError(f"pages have a multiple of 8 slots, got {slots}")
        self.slots, self.window, self.sinks = slots, window, sinks
        self.most = -(-most_tokens // slots)
        with torch.inference_mode(False):                # tensors made in that mode could not be written outside of it
            self.k = torch.empty(layers, pages, slots, kv_heads, head_dim, dtype=dtype, device=device)
            self.v = torch.empty_like(self.k)
            self.tables = torch.full((sequences, self.most), -1, dtype=torch.int32, device=device)
            self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._lengths = [0] * sequences
        self._rows: List[dict] = [{} for _ in range(sequences)]      # page of each place in a sequence's row of the table
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reset(self, sequence: int) -> None:
        """Ends a sequence: its pages are free for others."""
        self._free.extend(self._rows[sequence].values())
        self._rows[sequence] = {}
        self._lengths[sequence] = 0
        self.tables[sequence] = -1
        self.lengths[sequence] = 0

    def make_room(self, new: Sequence[int]) -> None:
        """Counts ``new`` tokens of each sequence in, gives back pages that none of them sees and takes those that they need."""
        if len(new) != len(self._lengths):
            raise ValueError(f"the cache has {len(self._lengths)} sequences, got counts of {len(new)}")
        plan, need = [], 0
        for b, n in enumerate(new):
            length, row = self._lengths[b] + n, self._rows[b]
            if n < 0 or -(-length // self.slots) > self.most:
                raise ValueError(f"sequence {b} has {self._lengths[b]} tokens: {n} more do not fit {self.most} pages of {self.slots}")
            near = 0 if self.window is None or n == 0 else max(0, self._lengths[b] - self.window + 1)      # the first token that a new one sees
            gone = [i for i in row if (i + 1) * self.slots <= near and i * self.slots >= self.sinks]
            take = [i for i in range(self._lengths[b] // self.slots, -(-length // self.slots)) if i not in row]
            plan.append((gone, take, length))
            need += len(take) - len(gone)
        if need > len(self._free):
            raise RuntimeError(f"the cache is full: {need} more pages are needed, {len(self._free)} are free")
        where, what = [], []
        for b, (gone, take, length) in enumerate(plan):
            for i in gone:
                self._free.append(self._rows[b].pop(i))
                where.append(b * self.most + i)
                what.append(-1)
        for b, (gone, take, length) in enumerate(plan):
            for i in take:
                self._rows[b][i] = self._free.pop()
                where.append(b * self.most + i)
                what.append(self._rows[b][i])
            self._lengths[b] = length
        device = self.tables.device
        if where:
            self.tables.view(-1)[torch.tensor(where, device=device)] = torch.tensor(what, dtype=torch.int32, device=device)
        self.lengths.copy_(torch.tensor(self._lengths, dtype=torch.int32))


class WindowBlock(nn.Module):
    """``x += W_o · attention(rotary(W_qkv · norm(x))); x += gated_mlp(norm(x))``."""

    def __init__(self, dim: int, heads: int, kv_heads: int, inner: int, window: Optional[int], sinks: int, bias: bool, eps: float,
                 dtype: torch.dtype, seeds: SeedSequence, act: str = "gelu"):
        super().__init__()
        if dim % heads or heads % kv_heads:
            raise ValueError(f"{dim} channels do not make {heads} heads that share {kv_heads} key heads")
        self.heads, self.kv_heads, self.window, self.sinks = heads, kv_heads, window, sinks
        self.ln1 = RmsNorm(dim, eps, dtype)
        self.qkv = Linear(dim, (heads + 2 * kv_heads) * (dim // heads), bias, dtype, seeds)
        self.proj = Linear(dim, dim, bias, dtype, seeds)
        self.ln2 = RmsNorm(dim, eps, dtype)
        self.mlp = GatedMlp(dim, inner, bias, dtype, seeds, act)

    def _ends(self, o: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """Rows of attention ``(N, heads, head_dim)`` and of the block's input ``(N, dim)`` → the block's output."""
        x = self.proj(o.reshape(x.shape), x)
        return self.mlp(self.ln2(x), x)

    def forward(self, x: torch.Tensor, positions: torch.Tensor, freqs, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        b, t, d = x.shape
        qkv = self.qkv(self.ln1(x).reshape(b * t, d)).view(b, t, self.heads + 2 * self.kv_heads, d // self.heads)
        qkv = ops.rotary(qkv, positions, freqs, heads=self.heads + self.kv_heads)
        o = ops.window_attention_qkv(qkv, self.kv_heads, self.window, self.sinks, lengths)
        return self._ends(o, x.reshape(b * t, d)).view(b, t, d)

    def extend(self, x: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedCache, offsets: Optional[torch.Tensor], freqs) -> torch.Tensor:
        """New tokens ``(N, dim)`` of the cache's sequences, whose keys and values go into this block's pages."""
        n, d = x.shape
        qkv = self.qkv(self.ln1(x)).view(n, self.heads + 2 * self.kv_heads, d // self.heads)
        q = ops.cache_append(qkv, k, v, cache.tables, cache.lengths, offsets, freqs)
        return self._ends(ops.cache_attention(q, k, v, cache.tables, cache.lengths, offsets, self.window, self.sinks), x)


class AttentionDecoder(nn.Module):
    """``frames (B, T, E)``: one vector per frame, as the frame head gives them; ``previous (B, T)``: the action taken before
    each frame, any id outside the vocabulary where there was none.  ``factor`` and ``context`` scale the positions for recordings
    longer than those that the model was trained on (:func:`~fbamtrain_b200.ops.rotary_frequencies`).

    ``forward`` takes heads of any width.  The cache, on a GPU in 16 bits, takes heads of 64 or 128 channels: ``make_cache`` refuses others."""

    def __init__(self, frame_dim: int, dim: int, layers: int, heads: int, inner: int, vocab: int, dtype: torch.dtype, seeds: SeedSequence,
                 kv_heads: Optional[int] = None, window: Optional[int] = None, sinks: int = 0, bias: bool = True, eps: float = 1e-5,
                 act: str = "gelu", base: float = 10000.0, factor: float = 1.0, context: Optional[int] = None):
        super().__init__()
        self.vocab, self.heads, self.kv_heads, self.window, self.sinks = vocab, heads, kv_heads or heads, window, sinks
        self.frame_proj = Linear(frame_dim, dim, bias, dtype, seeds)
        self.actions = TokenEmbedding(vocab, dim, dtype, seeds, scale=dim ** 0.5)
        self.block = nn.ModuleList([WindowBlock(dim, heads, self.kv_heads, inner, window, sinks, bias, eps, dtype, seeds, act) for _ in range(layers)])
        self.freqs = ops.rotary_frequencies(dim // heads, base, factor, context)
        self.ln_f = RmsNorm(dim, eps, dtype)
        # the head's width is a multiple of 8, as in ActionModel
        self.head_weight = nn.Parameter(torch.empty((vocab + 7) // 8 * 8, dim, dtype=dtype))
        fill_uniform_fan_(self.head_weight.data, dim, seeds)

    def _inputs(self, frames: torch.Tensor, previous: torch.Tensor) -> torch.Tensor:
        return self.frame_proj(frames, self.actions(previous))

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return ops.linear(hidden.reshape(-1, hidden.shape[-1]), self.head_weight, None)[:, : self.vocab]

    def features(self, frames: torch.Tensor, previous: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        b, t, e = frames.shape
        x = self._inputs(frames.reshape(b * t, e), previous.reshape(b * t)).view(b, t, -1)
        positions = torch.arange(t, device=frames.device)
        for block in self.block:
            x = block(x, positions, self.freqs, lengths)
        return self.ln_f(x)

    def forward(self, frames: torch.Tensor, previous: torch.Tensor, targets: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                top: int = 0, temperature: float = 1.0) -> ops.TokenLogprobs:
        """Log probability of ``targets (B, T)`` (0 where they lie outside the vocabulary) and entropy, ``(B, T)`` each.  ``lengths``
        ``(B,)``: frames of each recording of a padded batch; what lies behind them has no meaning."""
        r = ops.token_logprobs(self.logits(self.features(frames, previous, lengths)), targets.reshape(-1), top, temperature)
        return ops.TokenLogprobs(*(None if v is None else v.view(*targets.shape, *v.shape[1:]) for v in r))

    def _cache_width(self) -> int:
        width = self.head_weight.shape[1] // self.heads
        if width not in CACHE_WIDTHS and runs_native(self.head_weight, "mha"):
            raise ValueError(f"the kernels keep heads of {' or '.join(map(str, CACHE_WIDTHS))} channels in a cache, this model's have {width}")
        return width

    def make_cache(self, sequences: int, most_tokens: int, slots: int = 16, pages: Optional[int] = None) -> PagedCache:
        """A cache for ``sequences`` recordings of up to ``most_tokens`` frames.  Without ``pages`` the pool holds all that they can need
        with single steps: with a window, of each the pages of the first tokens and of the window."""
        weight, width = self.head_weight, self._cache_width()
        if pages is None:
            each = -(-most_tokens // slots)
            if self.window is not None:
                each = min(each, -(-self.sinks // slots) + -(-self.window // slots) + 1)
            pages = sequences * each
        return PagedCache(len(self.block), pages, slots, self.kv_heads, width, sequences, most_tokens, weight.dtype,
                          weight.device, self.window, self.sinks)

    def _check_cache(self, cache: PagedCache) -> None:
        """A cache that does not go with this model would be found out with some layers written, or not at all."""
        weight = self.head_weight
        fits = (len(self.block), self.kv_heads, self._cache_width())
        if (cache.k.shape[0], *cache.k.shape[3:]) != fits or cache.k.dtype != weight.dtype or cache.k.device != weight.device:
            raise ValueError(f"the model has {fits[0]} layers of {fits[1]} key heads of {fits[2]}, {weight.dtype} on {weight.device}; the cache "
                             f"{cache.k.shape[0]} of {cache.k.shape[3]} of {cache.k.shape[4]}, {cache.k.dtype} on {cache.k.device}")
        if cache.window is not None and (self.window is None or cache.window < self.window or cache.sinks < self.sinks):
            raise ValueError(f"the cache gives back what a window of {cache.window} and {cache.sinks} first tokens do not see, the model sees "
                             f"{self.window} and {self.sinks}")

    @torch.no_grad()
    def extend(self, frames: torch.Tensor, previous: torch.Tensor, cache: PagedCache, new: Sequence[int], top: int = 1,
               temperature: float = 1.0) -> ops.TokenLogprobs:
        """New frames ``(N, E)``, ``new[b]`` of them of sequence ``b`` one after the other, with the actions before them ``(N,)``: the
        ``top`` most likely actions at each, with their log probabilities."""
        new = [operator.index(n) for n in new]
        if sum(new) != frames.shape[0]:
            raise ValueError(f"{sum(new)} new frames are counted, {frames.shape[0]} given")
        if previous.shape != (frames.shape[0],):
            raise ValueError(f"the actions before {frames.shape[0]} frames are ({frames.shape[0]},), got {tuple(previous.shape)}")
        self._check_cache(cache)
        check_alternatives(self.vocab, top, temperature)
        if frames.dtype != cache.k.dtype:
            raise TypeError(f"the cache is {cache.k.dtype}, the frames {frames.dtype}")
        if frames.shape[0] == 0:
            cache.make_room(new)
            return ops.token_logprobs(frames.new_empty((0, self.vocab)), None, top, temperature)
        x = self._inputs(frames, previous)
        cache.make_room(new)                             # from here on the cache counts them
        offsets = None
        if any(n != 1 for n in new):
            starts = [0]
            for n in new:
                starts.append(starts[-1] + n)
            offsets = torch.tensor(starts, dtype=torch.int32, device=frames.device)
        for i, block in enumerate(self.block):
            x = block.extend(x, cache.k[i], cache.v[i], cache, offsets, self.freqs)
        return ops.token_logprobs(self.logits(self.ln_f(x)), None, top, temperature)

    def step(self, frame: torch.Tensor, previous: torch.Tensor, cache: PagedCache, top: int = 1, temperature: float = 1.0) -> ops.TokenLogprobs:
        """One frame of every sequence, ``(B, E)``, and the action before it ``(B,)``."""
        return self.extend(frame, previous, cache, [1] * frame.shape[0], top, temperature)
