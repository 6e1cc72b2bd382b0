"""Rotary positions and the append of new tokens to a paged cache (``csrc/rotary.cu``)."""
from __future__ import annotations

import ctypes as C
import functools
import math
from decimal import Context, Decimal, localcontext
from typing import NamedTuple, Optional, Tuple

import torch

from . import native as nv
from .derivatives import first_only, tracked


class _Frequencies(NamedTuple):
    turns: Tuple[int, ...]
    magnitude: float


class RotaryFrequencies(_Frequencies):
    """How far each pair of channels turns a position: fractions of a turn, times 2^64, and the factor on what is turned."""

    @functools.cached_property
    def table(self) -> C.Array:
        """``turns`` as the kernels take them."""
        return (C.c_ulonglong * max(1, len(self.turns)))(*self.turns)

    def __reduce__(self):
        return type(self), tuple(self)                  # without the table, which has no pickled form

    @property
    def dims(self) -> int:
        return 2 * len(self.turns)


_TWO_PI = Decimal("6.28318530717958647692528676655900576839433879875")     # as it is written: a product would be rounded


def rotary_frequencies(dims: int, base: float, factor: float, context: Optional[int], few: float, many: float) -> RotaryFrequencies:
    # in 40 digits: with the 53 bits of a double the last ones of a fraction of 64, which far positions bring up, would be anything
    with localcontext(Context(prec=40)):
        slower, least, most = Decimal(float(factor)), Decimal(float(few)), Decimal(float(many))
        turns, turn, next_pair = [], 2 ** 64 / _TWO_PI, (Decimal(float(base)).ln() * -2 / max(dims, 1)).exp()
        for _ in range(dims // 2):
            scaled = turn
            if factor != 1.0:
                kept = Decimal(0)
                if context is not None:
                    around = context * turn / 2 ** 64
                    kept = min(Decimal(1), max(Decimal(0), (around - least) / (most - least)))
                scaled = turn * kept + turn * (1 - kept) / slower
            turns.append(int(scaled.to_integral_value()) % 2 ** 64)
            turn *= next_pair
    magnitude = 1.0 + 0.1 * math.log(factor) if factor > 1.0 and context is not None else 1.0
    return RotaryFrequencies(tuple(turns), magnitude)


def _turned(x, positions, freqs, heads, interleaved, inverse):
    b, t, h, d = x.shape
    if x.stride(3) != 1:
        x = x.contiguous()
    y = x.new_empty((b, t, h, d))
    sb, st, sh, _ = x.stride()
    *rows, pt = positions.stride()
    pb = rows[0] if rows and positions.shape[0] > 1 else 0          # one row of positions is everyone's
    nv.check(nv.lib(x).fbam_rotary(x.data_ptr(), sb, st, sh, y.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64, pb, pt,
                                   freqs.table, len(freqs.turns), freqs.magnitude, interleaved, inverse, b, t, h, d, heads, nv.stream()),
             "fbam_rotary")
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, freqs, heads, interleaved):
        ctx.save_for_backward(positions)
        ctx.linked = ()
        ctx.how = (freqs, heads, interleaved)
        return _turned(x, positions, freqs, heads, interleaved, False)

    @staticmethod
    @first_only("rotary")
    def backward(ctx, dy):
        positions, = ctx.saved_tensors
        return _turned(dy, positions, *ctx.how, True), None, None, None, None


def rotary(x, positions, freqs, heads, interleaved):
    if positions.device != x.device:
        raise ValueError(f"positions are on {positions.device}, the heads on {x.device}")
    if tracked(x):
        return _Rotary.apply(x, positions, freqs, heads, interleaved)
    return _turned(x, positions, freqs, heads, interleaved, False)


def cache_append(qkv, k_pages, v_pages, tables, lengths, offsets, freqs, interleaved, q_heads, kv_heads):
    n, _, d = qkv.shape
    row, head, inner = qkv.stride()
    if inner != 1 or (row | head) % 8 or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
        row, head, _ = qkv.stride()
    q = qkv.new_empty((n, q_heads, d))
    turns, pairs, magnitude = (None, 0, 1.0) if freqs is None else (freqs.table, len(freqs.turns), freqs.magnitude)
    nv.check(nv.lib(qkv).fbam_cache_append(
        qkv.data_ptr(), row, head, q.data_ptr(), k_pages.data_ptr(), *k_pages.stride()[:3], v_pages.data_ptr(),
        *v_pages.stride()[:3], tables.data_ptr(), tables.stride(0), lengths.data_ptr(), nv.addr(offsets), turns, pairs, magnitude,
        interleaved, n, tables.shape[0], tables.shape[1], k_pages.shape[1], k_pages.shape[0], q_heads, kv_heads, d, nv.stream()),
        "fbam_cache_append")
    # written through pointers: a backward that saved the pages has to see it, as it sees the definition's stores
    torch.autograd.graph.increment_version((k_pages, v_pages))
    return q
