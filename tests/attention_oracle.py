"""Rotary positions, windowed attention and the paged cache in 64 bits, written from their definitions, with bounds on what kernels
that round their operands to 16 bits may be off by: what the tests compare with.

A rounding to the type is off by at most ``UNIT`` relative to the value, and, in half, by 2^-25 where the value is subnormal."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
F64 = torch.float64


def within(got, want, bound):
    got, want = got.detach().to(F64), want.to(F64)
    assert got.shape == want.shape
    assert bool(got.isfinite().all()), "not finite"
    over = (got - want).abs() - bound
    assert over.numel() == 0 or float(over.max()) <= 0.0, (float(over.max()), float((got - want).abs().max()))


# ------------------------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------------------------
def speeds(dims, base=10000.0, factor=1.0, context=None, few=1.0, many=32.0):
    """Radians a position of each pair, and the magnitude."""
    out, size = [], 1.0
    for i in range(dims // 2):
        s = math.exp(-2.0 * i / dims * math.log(base))
        share = 0.0
        if context is not None:
            share = min(max((s * context / (2 * math.pi) - few) / (many - few), 0.0), 1.0)
        out.append(share * s + (1.0 - share) * s / factor)
    if context is not None:
        size = 1.0 + 0.1 * math.log(factor)
    return torch.tensor(out, dtype=F64), size


def turned(x, positions, speed, size, heads, interleaved, back=False):
    """``x`` ``(..., H, D)``, ``positions`` ``(...)``: the value and the sum of its terms' absolute values."""
    out, mass = x.to(F64).clone(), x.to(F64).abs()
    n = 2 * len(speed)
    angle = positions.to(F64).unsqueeze(-1) * speed.to(x.device)
    cos, sin = (size * angle.cos()).unsqueeze(-2), (size * angle.sin()).unsqueeze(-2) * (-1.0 if back else 1.0)
    one = slice(0, n, 2) if interleaved else slice(0, n // 2)
    two = slice(1, n, 2) if interleaved else slice(n // 2, n)
    a, b = (x.to(F64)[..., :heads, s] for s in (one, two))
    out[..., :heads, one], out[..., :heads, two] = a * cos - b * sin, b * cos + a * sin
    reach = size * (a.abs() + b.abs())
    mass[..., :heads, one], mass[..., :heads, two] = reach, reach
    return out, mass


def turned_bound(want, mass, positions, dtype):
    """One rounding; in fp32 the angle (2^-24 of a turn in the conversion, and what 64 bits lose at far positions), its sine and
    cosine and three roundings of the terms."""
    far = positions.to(F64).abs().unsqueeze(-1).unsqueeze(-1) * 2.0 ** -50
    return UNIT[dtype] * want.abs() + FLOOR[dtype] + (2.0 ** -20 + far) * mass


# ------------------------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------------------------
def sees(i, j, window, sinks, end):
    """``(n, m)``: whether the query at position ``i[n]`` sees the key at ``j[m]``; both lie in front of ``end``."""
    i, j = i.view(-1, 1), j.view(1, -1)
    out = (j <= i) & (j < end) & (i >= 0)
    if window is not None:
        out &= (i - j < window) | (j < sinks)
    return out


def attend(q, k, v, seen, dtype):
    """One head: ``q`` ``(n, D)``, ``k``, ``v`` ``(m, D)`` → output, probabilities, the bound of the output and the relative bound of a
    row's probabilities."""
    scale = q.shape[1] ** -0.5
    q, k, v = (x.to(F64) for x in (q, k, v))
    s = (q @ k.t()) * scale
    s = s.masked_fill(~seen, -math.inf)
    some = seen.any(1, keepdim=True)
    p = torch.softmax(s.masked_fill(~some, 0.0), 1) * some
    o = p @ v
    unit, floor = UNIT[dtype], FLOOR[dtype]
    # a score in fp32: D products and sums of them, the scale, the maximum taken off (times log2 e); then the exponential
    reach = ((q.abs() @ k.abs().t()) * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
    rel = 2.0 * ((q.shape[1] + 8) * 2.0 ** -24 * reach + 2.0 ** -20)
    mass = p @ v.abs()
    count = seen.sum(1, keepdim=True)
    wrong = unit * o.abs() + (unit + rel + count * 2.0 ** -23) * mass + floor * (1.0 + seen.to(F64) @ v.abs())
    return o, p, wrong, rel


def attend_grad(q, k, v, seen, dtype, d_o):
    """Gradients of ``attend`` and their bounds: ``(dq, dk, dv), (bounds)``."""
    scale = q.shape[1] ** -0.5
    o, p, o_wrong, rel = attend(q, k, v, seen, dtype)
    q, k, v, d_o = (x.to(F64) for x in (q, k, v, d_o))
    unit, floor = UNIT[dtype], FLOOR[dtype]
    dp, delta = d_o @ v.t(), (d_o * o).sum(1, keepdim=True)
    ds = p * (dp - delta) * scale
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    delta_wrong = (d_o.abs() * (o_wrong + d * 2.0 ** -24 * o.abs())).sum(1, keepdim=True)      # from the rounded output
    dp_wrong = (d + 8) * 2.0 ** -24 * (d_o.abs() @ v.abs().t())
    ds_wrong = p * scale * ((rel + 2.0 ** -22) * (dp - delta).abs() + dp_wrong + delta_wrong) + unit * ds.abs() + floor * seen
    p_wrong = p * (rel + unit) + floor * seen
    sums = 2.0 ** -23
    grads = (ds @ k, ds.t() @ q, p.t() @ d_o)
    wrong = (ds_wrong @ k.abs() + m * sums * (ds.abs() @ k.abs()), ds_wrong.t() @ q.abs() + n * sums * (ds.abs().t() @ q.abs()),
             p_wrong.t() @ d_o.abs() + n * sums * (p.t() @ d_o.abs()))
    return grads, wrong


def window(q, k, v, win, sinks, lengths, d_o=None):
    """``q`` ``(B, T, H, D)``, ``k``, ``v`` ``(B, T, Hkv, D)``: ``{name: (value, bound)}`` of the output and, with ``d_o``, the
    gradients.  Nothing behind a sequence's length is read."""
    dtype = q.dtype
    b, t, h, _ = q.shape
    group = h // k.shape[2]
    names = ["y"] + ([] if d_o is None else ["dq", "dk", "dv"])
    out = {n: [torch.zeros(x.shape, dtype=F64, device=q.device) for _ in range(2)] for n, x in zip(names, (q, q, k, v))}
    for i in range(b):
        size = t if lengths is None else min(max(int(lengths[i]), 0), t)
        at = torch.arange(size, device=q.device)
        if size == 0:
            continue
        seen = sees(at, at, win, sinks, size)
        for n in range(h):
            args = (q[i, :size, n], k[i, :size, n // group], v[i, :size, n // group], seen, dtype)
            o, _, wrong, _ = attend(*args)
            out["y"][0][i, :size, n], out["y"][1][i, :size, n] = o, wrong
            if d_o is not None:
                grads, wrongs = attend_grad(*args, d_o[i, :size, n])
                for name, g, w, head in zip(names[1:], grads, wrongs, (n, n // group, n // group)):
                    out[name][0][i, :size, head] += g
                    out[name][1][i, :size, head] += w
    for name in names[1:]:
        out[name][1] += UNIT[dtype] * out[name][0].abs() + FLOOR[dtype]
    return out


def cached(q, k_pages, v_pages, tables, lengths, offsets, win, sinks):
    """``(value, bound)`` of new tokens over a paged cache."""
    n, h, d = q.shape
    slots, kv = k_pages.shape[1:3]
    y = [torch.zeros(q.shape, dtype=F64, device=q.device) for _ in range(2)]
    starts = list(range(n + 1)) if offsets is None else offsets.tolist()
    for b, length in enumerate(lengths.tolist()):
        lo, hi = starts[b], starts[b + 1]
        first = length - (hi - lo)
        rows = [r for r in range(lo, hi) if first + r - lo >= 0]
        if not rows or length <= 0:
            continue
        at = torch.tensor([first + r - lo for r in rows], device=q.device)
        keys = torch.arange(min(length, tables.shape[1] * slots), device=q.device)
        seen = sees(at, keys, win, sinks, length)
        need = seen.any(0)
        k = torch.zeros(len(keys), kv, d, dtype=F64, device=q.device)
        v = k.clone()
        for j in need.nonzero().flatten().tolist():
            page = int(tables[b, j // slots])
            if 0 <= page < k_pages.shape[0]:
                k[j], v[j] = k_pages[page, j % slots].to(F64), v_pages[page, j % slots].to(F64)
        for c in range(h):
            o, _, wrong, _ = attend(q[rows, c], k[:, c * kv // h], v[:, c * kv // h], seen, q.dtype)
            y[0][rows, c], y[1][rows, c] = o, wrong
    return y
