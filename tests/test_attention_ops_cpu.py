"""Rotary positions, windowed attention and the paged cache on the CPU: the plain definitions against 64 bits, gradients against
differences, and what is refused."""
import math

import pytest
import torch

import attention_oracle as oracle
from fbamtrain_b200 import ops

F32, F64 = torch.float32, torch.float64


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("settings", [{}, {"base": 500000.0}, {"factor": 4.0}, {"factor": 8.0, "context": 512},
                                      {"factor": 8.0, "context": 512, "few": 2.0, "many": 5.0}])
def test_rotary_definition(interleaved, settings):
    torch.manual_seed(0)
    x = torch.randn(2, 5, 3, 12).requires_grad_()
    positions = torch.tensor([[0, 1, 5, -3, 100], [7, 7, 1000000, 2 ** 31 - 1, 2 ** 40]])
    freqs = ops.rotary_frequencies(8, **settings)
    speed, size = oracle.speeds(8, **settings)
    assert freqs.dims == 8 and freqs.magnitude == pytest.approx(size)
    y = ops.rotary(x, positions, freqs, heads=2, interleaved=interleaved)
    want, mass = oracle.turned(x.detach(), positions, speed, size, 2, interleaved)
    oracle.within(y, want, oracle.turned_bound(want, mass, positions, F32))
    dy = torch.randn_like(x)
    dx, = torch.autograd.grad((y,), (x,), (dy,))
    want, mass = oracle.turned(dy, positions, speed, size, 2, interleaved, back=True)
    oracle.within(dx, want, oracle.turned_bound(want, mass, positions, F32))


def test_rotary_oracle_gradient_is_the_derivative():
    torch.manual_seed(1)
    x, dy, v = (torch.randn(1, 4, 2, 6, dtype=F64) for _ in range(3))
    positions = torch.tensor([[0, 3, 17, 400]])
    speed, size = oracle.speeds(4, factor=3.0, context=100)
    for interleaved in (False, True):
        def f(at):
            return float((oracle.turned(at, positions, speed, size, 1, interleaved)[0] * dy).sum())
        g = oracle.turned(dy, positions, speed, size, 1, interleaved, back=True)[0]
        assert float((g * v).sum()) == pytest.approx((f(x + 1e-6 * v) - f(x - 1e-6 * v)) / 2e-6, rel=1e-6, abs=1e-7)


def test_scores_depend_on_distance_only():
    torch.manual_seed(2)
    q, k = torch.randn(1, 1, 1, 16, dtype=F64), torch.randn(1, 1, 1, 16, dtype=F64)
    freqs = ops.rotary_frequencies(16)
    dots = [(ops.rotary(q, torch.tensor([[p + 9]]), freqs) * ops.rotary(k, torch.tensor([[p]]), freqs)).sum() for p in (0, 1, 50, 10 ** 6)]
    for d in dots[1:]:
        assert float(d) == pytest.approx(float(dots[0]), rel=1e-9, abs=1e-9)


WINDOWS = [(None, 0), (1, 0), (3, 0), (3, 2), (4, 30), (100, 1)]


@pytest.mark.parametrize("win,sinks", WINDOWS)
@pytest.mark.parametrize("lengths", [None, [11, 0, 4]])
def test_window_definition(win, sinks, lengths):
    torch.manual_seed(3)
    lengths = None if lengths is None else torch.tensor(lengths)
    qkv = torch.randn(3, 11, 4 + 2 * 2, 6)
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            qkv[b, n:] = math.nan
    qkv.requires_grad_()
    dy = torch.randn(3, 11, 4, 6)
    want = oracle.window(*qkv.detach().split((4, 2, 2), 2), win, sinks, lengths, dy)
    y = ops.window_attention_qkv(qkv, 2, win, sinks, lengths)
    oracle.within(y, *want["y"])
    grad, = torch.autograd.grad((y,), (qkv,), (dy,))
    for part, name in zip(grad.split((4, 2, 2), 2), ("dq", "dk", "dv")):
        oracle.within(part, *want[name])
    parts = [x.detach().clone() for x in qkv.split((4, 2, 2), 2)]
    oracle.within(ops.window_attention(*parts, win, sinks, lengths), *want["y"])


def test_window_oracle_gradients_are_the_derivatives():
    torch.manual_seed(4)
    q, k, v, dy = torch.randn(1, 9, 4, 3, dtype=F64), torch.randn(1, 9, 2, 3, dtype=F64), torch.randn(1, 9, 2, 3, dtype=F64), torch.randn(1, 9, 4, 3, dtype=F64)
    oracle.UNIT[F64] = oracle.FLOOR[F64] = 0.0
    for win, sinks in WINDOWS:
        got = oracle.window(q, k, v, win, sinks, None, dy)

        def f(*at):
            return float((oracle.window(*at, win, sinks, None)["y"][0] * dy).sum())

        for n, name in enumerate(("dq", "dk", "dv")):
            at = [q, k, v]
            step = torch.randn_like(at[n])
            up, down = list(at), list(at)
            up[n], down[n] = at[n] + 1e-6 * step, at[n] - 1e-6 * step
            assert float((got[name][0] * step).sum()) == pytest.approx((f(*up) - f(*down)) / 2e-6, rel=1e-6, abs=1e-7)


def _cache(pages, slots, kv, d, tables):
    k, v = torch.randn(pages, slots, kv, d), torch.randn(pages, slots, kv, d)
    return k, v, torch.tensor(tables, dtype=torch.int32)


@pytest.mark.parametrize("win,sinks", WINDOWS)
def test_cache_definition(win, sinks):
    torch.manual_seed(5)
    k, v, tables = _cache(9, 4, 2, 6, [[3, 1, 7, 8], [0, 4, -1, -1], [5, 6, 2, -1], [-1, -1, -1, -1]])
    lengths = torch.tensor([14, 2, 9, 0], dtype=torch.int32)
    offsets = torch.tensor([0, 3, 4, 4, 6], dtype=torch.int32)          # the third sequence has no new token, the last no length
    q = torch.randn(8, 4, 6)                                            # two rows behind the last offset
    want = oracle.cached(q, k, v, tables, lengths, offsets, win, sinks)
    oracle.within(ops.cache_attention(q, k, v, tables, lengths, offsets, win, sinks), *want)
    single = torch.randn(4, 4, 6)
    want = oracle.cached(single, k, v, tables, lengths, None, win, sinks)
    oracle.within(ops.cache_attention(single, k, v, tables, lengths, None, win, sinks), *want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_then_attend_is_attention_over_the_whole(interleaved):
    torch.manual_seed(6)
    t, h, kv, d = 13, 4, 2, 8
    qkv = torch.randn(1, t, h + 2 * kv, d)
    freqs = ops.rotary_frequencies(8)
    whole = ops.rotary(qkv, torch.arange(t), freqs, heads=h + kv, interleaved=interleaved)
    want = ops.window_attention_qkv(whole, kv, 5, 2)[0]
    k, v, tables = _cache(5, 4, kv, d, [[2, 0, 4, 1]])
    k.fill_(math.nan), v.fill_(math.nan)
    got, at = [], 0
    for n in (6, 1, 1, 4, 1):
        lengths, offsets = torch.tensor([at + n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
        q = ops.cache_append(qkv[0, at:at + n], k, v, tables, lengths, offsets, freqs, interleaved)
        got.append(ops.cache_attention(q, k, v, tables, lengths, offsets, 5, 2))
        at += n
    torch.testing.assert_close(torch.cat(got), want, atol=1e-5, rtol=1e-5)
    assert bool(k[3].isnan().all())                                     # a page of nobody


def test_append_leaves_what_is_not_its_own():
    torch.manual_seed(7)
    k, v, tables = _cache(4, 4, 1, 6, [[1, -1], [2, 3], [0, 9]])
    before = k.clone(), v.clone()
    lengths, offsets = torch.tensor([5, 1, 6], dtype=torch.int32), torch.tensor([0, 1, 3, 4], dtype=torch.int32)
    qkv = torch.randn(5, 2 + 2, 6)
    q = ops.cache_append(qkv, k, v, tables, lengths, offsets)
    # no page; in front of the start; token 0 of the second; a page that is none; a row of nobody
    assert torch.equal(q[0], qkv[0, :2]) and not q[1].any() and torch.equal(q[2], qkv[2, :2]) and not q[4].any()
    assert torch.equal(k[2, 0], qkv[2, 2:3]) and torch.equal(v[2, 0], qkv[2, 3:])
    k[2, 0], v[2, 0] = before[0][2, 0], before[1][2, 0]
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def test_refusals():
    x, freqs = torch.randn(2, 3, 4, 8), ops.rotary_frequencies(8)
    for bad in ({"dims": 7}, {"dims": 258}, {"dims": -2}, {"dims": 8, "base": 0.0}, {"dims": 8, "factor": 0.5},
                {"dims": 8, "factor": math.inf}, {"dims": 8, "context": 0}, {"dims": 8, "context": 9, "few": 3.0, "many": 2.0}):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)
    with pytest.raises(ValueError, match="heads are"):
        ops.rotary(x[0], torch.arange(3), freqs)
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.rotary(x, torch.arange(3).float(), freqs)
    with pytest.raises(ValueError, match="positions"):
        ops.rotary(x, torch.arange(4), freqs)
    with pytest.raises(ValueError, match="heads turn"):
        ops.rotary(x, torch.arange(3), freqs, heads=5)
    with pytest.raises(ValueError, match="do not fit"):
        ops.rotary(x, torch.arange(3), ops.rotary_frequencies(16))

    q, k = torch.randn(2, 3, 4, 8), torch.randn(2, 3, 2, 8)
    for a, b, c in ((q[0], k, k), (q, k, k[:, :2]), (q, k[:1], k[:1]), (q, k[..., :4], k[..., :4])):
        with pytest.raises(ValueError, match="go together"):
            ops.window_attention(a, b, c)
    with pytest.raises(TypeError, match="one type"):
        ops.window_attention(q, k.double(), k)
    with pytest.raises(ValueError, match="share"):
        ops.window_attention(q[:, :, :3], k, k)
    with pytest.raises(ValueError, match="window"):
        ops.window_attention(q, k, k, 0)
    with pytest.raises(ValueError, match="first tokens"):
        ops.window_attention(q, k, k, 3, -1)
    with pytest.raises(ValueError, match="lengths"):
        ops.window_attention(q, k, k, 3, 0, torch.tensor([1]))
    with pytest.raises(ValueError, match="lengths"):
        ops.window_attention(q, k, k, 3, 0, torch.tensor([1.0, 2.0]))
    for kv in (0, 3, 4):
        with pytest.raises(ValueError, match="share"):
            ops.window_attention_qkv(torch.randn(1, 2, 7, 8), kv)
    with pytest.raises(ValueError, match="projection"):
        ops.window_attention_qkv(q[0], 1)

    kp, vp, tables = _cache(3, 4, 2, 8, [[0, 1], [2, -1]])
    lengths, new = torch.tensor([3, 2], dtype=torch.int32), torch.randn(2, 4, 8)
    fine = (kp, vp, tables, lengths)
    ops.cache_attention(new, *fine)
    with pytest.raises(ValueError, match="one new token"):
        ops.cache_attention(new[:1], *fine)
    with pytest.raises(ValueError, match="pages are"):
        ops.cache_attention(new, kp, vp[:2], tables, lengths)
    with pytest.raises(ValueError, match="pages are"):
        ops.cache_attention(new[..., :4], *fine)
    with pytest.raises(TypeError, match="the pages"):
        ops.cache_attention(new.double(), *fine)
    with pytest.raises(ValueError, match="page tables"):
        ops.cache_attention(new, kp, vp, tables.long(), lengths)
    with pytest.raises(ValueError, match="lengths"):
        ops.cache_attention(new, kp, vp, tables, lengths.long())
    with pytest.raises(ValueError, match="offsets"):
        ops.cache_attention(new, *fine, torch.tensor([0, 2], dtype=torch.int32))
    with pytest.raises(ValueError, match="share"):
        ops.cache_attention(new[:, :3], *fine)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.cache_attention(new.clone().requires_grad_(), *fine)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.cache_append(torch.randn(2, 8, 8).requires_grad_(), *fine)
    with pytest.raises(ValueError, match="share"):
        ops.cache_append(torch.randn(2, 4, 8), *fine)
    with pytest.raises(ValueError, match="do not fit"):
        ops.cache_append(torch.randn(2, 8, 8), *fine, freqs=ops.rotary_frequencies(16))
    with torch.no_grad():
        ops.cache_attention(new.clone().requires_grad_(), *fine)


def test_nothing_at_all():
    """No sequences, no tokens, no steps."""
    assert ops.window_attention(torch.empty(0, 3, 2, 8), torch.empty(0, 3, 1, 8), torch.empty(0, 3, 1, 8)).shape == (0, 3, 2, 8)
    assert ops.window_attention_qkv(torch.empty(2, 0, 4, 8), 1).shape == (2, 0, 2, 8)
    assert ops.rotary(torch.empty(2, 0, 4, 8), torch.arange(0), ops.rotary_frequencies(8)).shape == (2, 0, 4, 8)
    kp, vp, tables = _cache(3, 4, 2, 8, [[0, 1]])
    none = torch.empty(0, dtype=torch.int32)
    assert ops.cache_attention(torch.empty(0, 4, 8), kp, vp, tables[:0], none).shape == (0, 4, 8)
    q = ops.cache_attention(torch.randn(2, 4, 8), kp, vp, tables[:0], none, torch.zeros(1, dtype=torch.int32))
    assert q.shape == (2, 4, 8) and not q.any()
