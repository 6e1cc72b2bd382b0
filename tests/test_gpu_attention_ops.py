"""Rotary positions, windowed attention and the paged cache on the kernels against 64 bits, at the sizes, strides and masks where
they can go wrong."""
import math
import zlib

import pytest
import torch

import attention_oracle as oracle
from fbamtrain_b200 import ops
from fbamtrain_b200.ops import native as nv

pytestmark = pytest.mark.gpu
BF, HALF = torch.bfloat16, torch.float16
I32 = torch.int32


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _randn(gen, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _done():
    nv.check_status(torch.device("cuda", 0))


# ------------------------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------------------------
ROTARY = [  # batch, steps, heads, turned, width, turned channels
    (1, 1, 1, 1, 64, 64), (2, 7, 3, 2, 64, 64), (1, 33, 48, 32, 64, 32), (3, 100, 24, 20, 128, 96), (2, 257, 5, 5, 128, 128),
    (1, 3, 2, 1, 256, 256), (2, 9, 3, 2, 24, 16), (2, 9, 3, 2, 20, 6), (1, 5, 4, 4, 7, 2), (2, 5, 4, 0, 64, 64), (1, 40, 300, 300, 64, 64),
    (2, 3, 2, 2, 16, 0), (5, 1000, 1, 1, 64, 16)]


@pytest.mark.parametrize("b,t,h,turned,d,dims", ROTARY)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_rotary(b, t, h, turned, d, dims, interleaved, dtype):
    gen = _gen("rotary", b, t, h, d)
    settings = {"base": 500000.0, "factor": 4.0, "context": 1000} if t % 2 else {}
    freqs = ops.rotary_frequencies(dims, **settings)
    speed, size = oracle.speeds(dims, **settings)
    x = _randn(gen, b, t, h, d, dtype=dtype).requires_grad_()
    positions = torch.randint(-5, 2 ** 31 - 1 if t % 3 else 5000, (b, t), generator=gen, device="cuda")
    y = ops.rotary(x, positions, freqs, heads=turned, interleaved=interleaved)
    assert y.dtype == dtype
    want, mass = oracle.turned(x.detach(), positions, speed, size, turned, interleaved)
    oracle.within(y, want, oracle.turned_bound(want, mass, positions, dtype))
    assert torch.equal(y[:, :, turned:], x[:, :, turned:])                  # copied to the bit
    dy = _randn(gen, b, t, h, d, dtype=dtype)
    dx, = torch.autograd.grad((y,), (x,), (dy,))
    want, mass = oracle.turned(dy, positions, speed, size, turned, interleaved, back=True)
    oracle.within(dx, want, oracle.turned_bound(want, mass, positions, dtype))


def test_rotary_strides_and_positions():
    gen = _gen("rotary strides")
    freqs = ops.rotary_frequencies(64)
    speed, size = oracle.speeds(64)
    wide = _randn(gen, 3, 11, 9, 80)
    views = [wide[:, :, 2:5, :64], wide[:, ::2, :, 8:72], wide.transpose(0, 1)[:, :, :, 16:], wide[:, :, :, 1:65],
             wide.transpose(2, 3)[:, :, :64, :3].transpose(2, 3)]
    for x in views:
        for p in (torch.arange(x.shape[1], device="cuda"), torch.arange(x.shape[1], device="cuda", dtype=I32).view(1, -1),
                  torch.randint(0, 99, (x.shape[1], x.shape[0]), generator=gen, device="cuda").t()):
            at = p.expand(x.shape[:2])
            want, mass = oracle.turned(x, at, speed, size, 2, False)
            oracle.within(ops.rotary(x, p, freqs, heads=2), want, oracle.turned_bound(want, mass, at, BF))


# ------------------------------------------------------------------------------------------------------------------
# windowed attention
# ------------------------------------------------------------------------------------------------------------------
WINDOW = [  # batch, steps, heads, key heads, width, window, first tokens, padded
    (1, 1, 1, 1, 64, None, 0, False), (2, 2, 2, 1, 128, 1, 0, False), (1, 63, 2, 2, 64, 7, 2, False), (2, 127, 1, 1, 128, None, 0, False),
    (1, 128, 3, 1, 64, 128, 0, False), (2, 129, 2, 2, 128, 127, 1, True), (1, 255, 4, 4, 64, 64, 4, False), (1, 257, 2, 1, 64, 256, 0, False),
    (3, 300, 5, 1, 128, 129, 130, True), (2, 300, 4, 2, 64, None, 0, True), (1, 640, 8, 1, 128, 200, 128, False),
    (1, 641, 6, 2, 64, 1, 300, False), (2, 385, 7, 1, 64, 40, 3, True), (1, 1030, 2, 2, 128, 300, 5, False), (1, 1500, 1, 1, 64, 512, 0, False),
    (1, 500, 16, 1, 64, 100, 17, False), (1, 200, 128, 1, 64, 50, 1, False), (2, 130, 66, 2, 128, 20, 0, True), (1, 900, 2, 2, 64, 4000, 6, False),
    (1, 260, 2, 1, 96, 100, 4, True), (2, 140, 3, 3, 20, 30, 1, False), (4, 24, 2, 2, 64, 5, 1, True)]


@pytest.mark.parametrize("b,t,h,kv,d,win,sinks,padded", WINDOW)
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_window_forward(b, t, h, kv, d, win, sinks, padded, dtype):
    gen = _gen("window", b, t, h, d, win)
    qkv = _randn(gen, b, t, h + 2 * kv, d, dtype=dtype)
    lengths = None
    if padded:
        lengths = torch.tensor([max(0, t - 150 * i) for i in range(b)], device="cuda")
        lengths[-1] = t // 3
        if b > 2:
            lengths[1] = 0
        for i, n in enumerate(lengths.tolist()):
            qkv[i, n:] = math.nan
    want = oracle.window(*qkv.split((h, kv, kv), 2), win, sinks, lengths)
    y = ops.window_attention_qkv(qkv, kv, win, sinks, lengths)
    _done()
    oracle.within(y, *want["y"])


@pytest.mark.parametrize("b,t,h,kv,d,win,sinks,padded", WINDOW)
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_window_gradients(b, t, h, kv, d, win, sinks, padded, dtype):
    gen = _gen("window", b, t, h, d, win)
    qkv, dy = _randn(gen, b, t, h + 2 * kv, d, dtype=dtype), _randn(gen, b, t, h, d, dtype=dtype)
    lengths = None
    if padded:
        lengths = torch.tensor([max(0, t - 150 * i) for i in range(b)], device="cuda", dtype=I32)
        lengths[-1] = t // 3
        if b > 2:
            lengths[1] = 0
        for i, n in enumerate(lengths.tolist()):
            qkv[i, n:] = math.nan
            dy[i, n:] = math.nan
    want = oracle.window(*qkv.split((h, kv, kv), 2), win, sinks, lengths, dy)
    qkv.requires_grad_()
    y = ops.window_attention_qkv(qkv, kv, win, sinks, lengths)
    oracle.within(y, *want["y"])
    grad, = torch.autograd.grad((y,), (qkv,), (dy,))
    _done()
    for part, name in zip(grad.split((h, kv, kv), 2), ("dq", "dk", "dv")):
        oracle.within(part, *want[name])
    again, = torch.autograd.grad((ops.window_attention_qkv(qkv, kv, win, sinks, lengths),), (qkv,), (dy,))
    assert torch.equal(grad, again)


def test_window_three_tensors_and_strides():
    gen = _gen("window views")
    q, k, v, dy = (_randn(gen, 200, 2, n, 64).transpose(0, 1) for n in (4, 2, 2, 4))       # time-major
    k = _randn(gen, 2, 200, 64, 2).transpose(2, 3)                                         # channels apart
    wide = _randn(gen, 2, 200, 2, 67)[..., 3:]                                             # no 16-byte rows
    for value in (v, wide):
        named = [x.clone(memory_format=torch.preserve_format).requires_grad_() for x in (q, k, value)]
        want = oracle.window(q, k, value, 70, 3, None, dy)
        y = ops.window_attention(*named, 70, 3)
        oracle.within(y, *want["y"])
        for g, name in zip(torch.autograd.grad((y,), named, (dy,)), ("dq", "dk", "dv")):
            oracle.within(g, *want[name])
    _done()


# ------------------------------------------------------------------------------------------------------------------
# paged cache
# ------------------------------------------------------------------------------------------------------------------
def _batch(gen, lengths, new, slots, kv, d, dtype, spare=3, holes=True):
    """Pages in any order with NaN in every slot that no sequence has, tables with -1 behind the pages of a sequence."""
    per = [-(-n // slots) for n in lengths]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    k, v = (torch.full((pages, slots, kv, d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    tables = torch.full((len(lengths), max(1, *per) + 2), -1, dtype=I32)
    at = 0
    for b, n in enumerate(lengths):
        for i in range(per[b]):
            page, used = order[at], min(slots, n - i * slots)
            tables[b, i] = page
            k[page, :used], v[page, :used] = _randn(gen, used, kv, d, dtype=dtype), _randn(gen, used, kv, d, dtype=dtype)
            at += 1
    offsets = torch.tensor([0] + new, dtype=I32, device="cuda").cumsum(0).to(I32)
    return k, v, tables.cuda(), torch.tensor(lengths, dtype=I32, device="cuda"), offsets


CACHE = [  # lengths, new tokens, slots, heads, key heads, width, window, first tokens
    ([1], [1], 16, 1, 1, 64, None, 0), ([130, 1, 0, 77], [1, 1, 1, 1], 16, 4, 2, 64, None, 0), ([600, 300], [1, 1], 8, 8, 1, 128, None, 0),
    ([1000, 129, 128, 127], [1, 1, 1, 1], 24, 5, 5, 128, 100, 4), ([257], [257], 32, 2, 2, 64, None, 0), ([700, 300, 5], [300, 1, 5], 128, 6, 2, 128, None, 0),
    ([700, 300, 5, 64], [65, 0, 5, 1], 256, 3, 1, 64, 90, 130), ([2000], [40], 16, 16, 2, 64, 500, 16), ([900, 901], [129, 64], 40, 4, 1, 128, 1, 0),
    ([3, 500], [5, 200], 16, 2, 1, 64, 64, 1), ([1500], [1], 64, 2, 2, 128, 300, 2), ([520, 40, 300, 7, 260], [1, 1, 1, 1, 1], 8, 66, 1, 64, 200, 3)]


@pytest.mark.parametrize("lengths,new,slots,h,kv,d,win,sinks", CACHE)
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_cache_attention(lengths, new, slots, h, kv, d, win, sinks, dtype):
    gen = _gen("cache", lengths, slots, h)
    k, v, tables, lens, offsets = _batch(gen, lengths, new, slots, kv, d, dtype)
    if win is not None:                                  # pages that nothing sees any more are gone
        for b, (n, fresh) in enumerate(zip(lengths, new)):
            near = max(0, n - fresh - win + 1)
            for i in range(-(-sinks // slots), near // slots):
                k[tables[b, i]], v[tables[b, i]] = math.nan, math.nan
                tables[b, i] = -1 if i % 2 else tables[b, i]
    q = _randn(gen, sum(new) + 3, h, d, dtype=dtype)     # three rows of nobody
    want = oracle.cached(q, k, v, tables, lens, offsets, win, sinks)
    y = ops.cache_attention(q, k, v, tables, lens, offsets, win, sinks)
    _done()
    oracle.within(y, *want)
    assert not y[sum(new):].any()
    if set(new) == {1}:
        got = ops.cache_attention(q[:len(new)], k, v, tables, lens, None, win, sinks)
        oracle.within(got, *(x[:len(new)] for x in want))


def test_cache_pages_that_are_none():
    """Entries outside the pool where a query sees them count as zeros; a table may end in front of the sequence."""
    gen = _gen("holes")
    k, v, tables, lens, offsets = _batch(gen, [400, 300], [3, 2], 16, 2, 64, BF)
    tables[0, 2], tables[0, 5], tables[1, 0] = -7, 2 ** 31 - 1, k.shape[0]
    lens[1] = 1000
    k.nan_to_num_(0.5), v.nan_to_num_(0.5)               # the longer sequence has the slots that no one had
    q = _randn(gen, 5, 4, 64)
    want = oracle.cached(q, k, v, tables, lens, offsets, None, 0)
    oracle.within(ops.cache_attention(q, k, v, tables, lens, offsets), *want)
    want = oracle.cached(q, k, v, tables, lens, offsets, 600, 20)
    oracle.within(ops.cache_attention(q, k, v, tables, lens, offsets, 600, 20), *want)
    _done()


def test_cache_strides():
    """Keys and values in one tensor, slots and heads in another order, rows of the table longer than their part."""
    gen = _gen("cache strides")
    k, v, tables, lens, offsets = _batch(gen, [200, 90], [1, 4], 16, 2, 128, BF)
    q = _randn(gen, 5, 2 + 4, 128)[:, 1:5]
    want = oracle.cached(q, k, v, tables, lens, offsets, 50, 3)
    both = torch.stack([k, v], 1)
    other = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    wide = torch.cat([tables, tables], 1)[:, :tables.shape[1]]
    for kp, vp, t in ((both[:, 0], both[:, 1], tables), (*other, wide)):
        oracle.within(ops.cache_attention(q, kp, vp, t, lens, offsets, 50, 3), *want)
    _done()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("dims", [0, 32, 64])
def test_append(interleaved, dtype, dims):
    gen = _gen("append", dims)
    h, kv, d, slots = 4, 2, 64, 16
    k, v, tables, lens, offsets = _batch(gen, [40, 17, 9, 0, 300], [7, 17, 0, 2, 1], slots, kv, d, dtype)
    tables[4, 18] = 10 ** 6                              # the new token of the last sequence has no page
    tables[1, 0] = -1                                    # nor have sixteen of the second
    qkv = _randn(gen, 30, h + 2 * kv, d, dtype=dtype)
    freqs = ops.rotary_frequencies(dims) if dims else None
    speed, size = oracle.speeds(dims)
    before = k.clone(), v.clone()
    q = ops.cache_append(qkv, k, v, tables, lens, offsets, freqs, interleaved)
    _done()
    want_k, want_v = before[0].double(), before[1].double()
    bound_k = torch.zeros_like(want_k)
    for b in range(5):
        lo, hi = int(offsets[b]), int(offsets[b + 1])
        for n in range(lo, hi):
            at = int(lens[b]) - (hi - n)
            if at < 0:
                assert not q[n].any()
                continue
            p = torch.tensor([at], device="cuda")
            want, mass = oracle.turned(qkv[n:n + 1], p, speed, size, h + kv, interleaved)
            bound = oracle.turned_bound(want, mass, p, dtype)
            oracle.within(q[n:n + 1], want[:, :h], bound[:, :h])
            page = int(tables[b, at // slots])
            if 0 <= page < k.shape[0]:
                want_k[page, at % slots], bound_k[page, at % slots] = want[0, h:h + kv], bound[0, h:h + kv]
                want_v[page, at % slots] = qkv[n, h + kv:].double()
    assert not q[27:].any()
    assert torch.equal(v.double().nan_to_num(7.0), want_v.nan_to_num(7.0))
    oracle.within(k.double().nan_to_num(7.0), want_k.nan_to_num(7.0), bound_k)


def test_refusals_on_the_gpu():
    gen = _gen("refusals")
    k, v, tables, lens, offsets = _batch(gen, [20], [2], 16, 1, 64, BF)
    q, qkv = _randn(gen, 2, 2, 64), _randn(gen, 2, 4, 64)
    with pytest.raises(ValueError, match="multiple of 8 slots"):
        ops.cache_attention(q, k[:, :12], v[:, :12], tables, lens, offsets)
    with pytest.raises(ValueError, match="64 or 128"):
        ops.cache_attention(q[..., :32], k[..., :32], v[..., :32], tables, lens, offsets)
    with pytest.raises(ValueError, match="16-byte"):
        ops.cache_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3).expand(-1, -1, 1, -1).as_strided(k.shape, (1024, 63, 64, 1)), v, tables, lens, offsets)
    with pytest.raises(ValueError, match="channels in a cache"):
        ops.cache_append(qkv, k, v, tables, lens, offsets, ops.rotary_frequencies(8))
    with pytest.raises(ValueError, match="are on cpu"):
        ops.cache_attention(q, k, v, tables.cpu(), lens, offsets)
    with pytest.raises(ValueError, match="are on cpu"):
        ops.window_attention(q[None], k[:1, :2], v[:1, :2], 3, 0, torch.tensor([1]))
    with pytest.raises(ValueError, match="are on cpu"):
        ops.rotary(q[None], torch.arange(2), ops.rotary_frequencies(64))
