"""Rotary positions, windowed attention and the paged cache where calls meet each other: streams, captured graphs, views that are
expanded, tensors beyond 2^31 values, and what is refused."""
import zlib

import pytest
import torch

import attention_oracle as oracle
from fbamtrain_b200 import ops
from fbamtrain_b200.ops import native as nv

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
I32 = torch.int32


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _randn(gen, *shape, dtype=BF):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _cache(gen, lengths, slots, kv, d, most=None):
    per = [-(-n // slots) for n in lengths]
    order = torch.randperm(sum(per), generator=gen, device="cuda").to(I32)
    tables = torch.full((len(lengths), most or max(per)), -1, dtype=I32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        tables[b, :n] = order[at:at + n]
        at += n
    return (_randn(gen, sum(per), slots, kv, d), _randn(gen, sum(per), slots, kv, d), tables, torch.tensor(lengths, dtype=I32, device="cuda"))


def _everything(gen):
    """A call of each operator, as functions of nothing that return lists of tensors."""
    qkv, dy = _randn(gen, 2, 333, 8, 64).requires_grad_(), _randn(gen, 2, 333, 4, 64)
    positions, freqs = torch.arange(333, device="cuda"), ops.rotary_frequencies(64)
    cache = _cache(gen, [700, 260], 16, 2, 64)
    new, single, offsets = _randn(gen, 70, 8, 64), _randn(gen, 2, 4, 64), torch.tensor([0, 66, 70], dtype=I32, device="cuda")

    def train():
        turned = ops.rotary(qkv, positions, freqs, heads=6)
        y = ops.window_attention_qkv(turned, 2, 100, 5)
        return [y.detach(), *torch.autograd.grad((y,), (qkv,), (dy,))]

    def serve():
        q = ops.cache_append(new, *cache, offsets, freqs)
        return [q, ops.cache_attention(q, *cache, offsets, 150, 3), ops.cache_attention(single, *cache), cache[0], cache[1]]

    return train, serve


def test_another_stream():
    train, serve = _everything(_gen("streams"))
    first = [x.clone() for x in train() + serve()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = train() + serve()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """The same calls on two streams, each with its own workspace."""
    one, two = _everything(_gen("one"))[0], _everything(_gen("two"))[0]
    want = [x.clone() for x in one() + two()]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(a):
            first = one()
        with torch.cuda.stream(b):
            second = two()
    torch.cuda.synchronize()
    for x, y in zip(want, first + second):
        assert torch.equal(x, y)


def test_captured_and_replayed():
    """Each in a graph of its own, replayed in turn with other inputs in the same places."""
    gen = _gen("graphs")
    train, serve = _everything(gen)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for call in (train, serve):
            call()                                       # before a capture: what a first call sets up
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = call()
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    got = [[x.clone() for x in out] for _, out in graphs]
    want = [[x.clone() for x in call()] for call in (train, serve)]
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    nv.check_status(torch.device("cuda", 0))


def test_expanded_tensors():
    """One key head, one sequence and one gradient for all, as expanded views."""
    gen = _gen("expand")
    q, k, v = _randn(gen, 1, 150, 1, 64), _randn(gen, 1, 150, 1, 64), _randn(gen, 1, 150, 1, 64)
    wide = [x.expand(3, 150, 2, 64).requires_grad_() for x in (q, k, v)]
    dy = _randn(gen, 1, 1, 1, 64).expand(3, 150, 2, 64)
    y = ops.window_attention(*wide, 40, 2)
    want = oracle.window(*(x.detach().contiguous() for x in wide), 40, 2, None, dy)
    oracle.within(y, *want["y"])
    for g, name in zip(torch.autograd.grad((y,), wide, (dy,)), ("dq", "dk", "dv")):
        oracle.within(g, *want[name])
    grad, = torch.autograd.grad((ops.window_attention(*wide, 40, 2).float().sum(),), (wide[0],))
    assert bool(grad.isfinite().all())
    x = q.expand(2, 150, 3, 64).requires_grad_()
    turned = ops.rotary(x, torch.arange(150, device="cuda"), ops.rotary_frequencies(64))
    assert torch.equal(turned[0, :, 0], turned[1, :, 2])
    cache = _cache(gen, [90, 33], 16, 1, 64)
    one = _randn(gen, 1, 1, 64).expand(2, 4, 64)
    oracle.within(ops.cache_attention(one, *cache), *oracle.cached(one, *cache, None, None, 0))
    with pytest.raises(ValueError, match="16-byte"):
        ops.cache_attention(one, cache[0][:1].expand_as(cache[0]), cache[1], *cache[2:])


def test_one_gradient_at_a_time():
    gen = _gen("needs")
    named = [_randn(gen, 1, 140, n, 64) for n in (4, 2, 2)]
    dy = _randn(gen, 1, 140, 4, 64)
    want = oracle.window(*named, 30, 1, None, dy)
    for i, name in enumerate(("dq", "dk", "dv")):
        at = [x.clone().requires_grad_(j == i) for j, x in enumerate(named)]
        g, = torch.autograd.grad((ops.window_attention(*at, 30, 1),), (at[i],), (dy,))
        oracle.within(g, *want[name])


def test_second_derivatives_and_tangents_are_refused():
    from torch.autograd import forward_ad
    gen = _gen("second")
    qkv = _randn(gen, 1, 40, 4, 64).requires_grad_()
    calls = (lambda x: ops.window_attention_qkv(x, 1, 9), lambda x: ops.rotary(x, torch.arange(40, device="cuda"), ops.rotary_frequencies(64)))
    for call in calls:
        g, = torch.autograd.grad((call(qkv).float().pow(2).sum(),), (qkv,), create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad((g.float().sum(),), (qkv,))
        with forward_ad.dual_level(), pytest.raises(Exception):
            call(forward_ad.make_dual(qkv.detach(), torch.ones_like(qkv)))


@pytest.mark.parametrize("b,t,h,kv,win,sinks", [(1, 3000, 1, 1, None, 0), (1, 4100, 4, 1, 2500, 200), (1, 2000, 3, 1, 1999, 1), (2, 1500, 1, 1, 700, 300)])
def test_divided_walks(b, t, h, kv, win, sinks):
    """Few heads and long sequences: the walks of the backward are divided, those of the first tokens and those of the window."""
    gen = _gen("divided", t)
    qkv, dy = _randn(gen, b, t, h + 2 * kv, 64), _randn(gen, b, t, h, 64)
    lengths = torch.tensor([t - 700] * b, device="cuda") if b > 1 else None
    want = oracle.window(*qkv.split((h, kv, kv), 2), win, sinks, lengths, dy)
    qkv.requires_grad_()
    y = ops.window_attention_qkv(qkv, kv, win, sinks, lengths)
    oracle.within(y, *want["y"])
    grad, = torch.autograd.grad((y,), (qkv,), (dy,))
    for part, name in zip(grad.split((h, kv, kv), 2), ("dq", "dk", "dv")):
        oracle.within(part, *want[name])
    again, = torch.autograd.grad((ops.window_attention_qkv(qkv, kv, win, sinks, lengths),), (qkv,), (dy,))
    assert torch.equal(grad, again)
    nv.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("lengths,most,h,kv,d", [([20000], None, 8, 1, 128), ([5000, 1, 9000], 2000, 16, 2, 64), ([300] * 40, None, 4, 4, 64)])
def test_keys_are_shared_out(lengths, most, h, kv, d):
    """Long histories of few sequences, whose keys several thread blocks share, and a table wider than any of them."""
    gen = _gen("shares", lengths[0])
    cache = _cache(gen, lengths, 16, kv, d, most)
    q = _randn(gen, len(lengths), h, d)
    for win, sinks in ((None, 0), (3000, 100)):
        oracle.within(ops.cache_attention(q, *cache, None, win, sinks), *oracle.cached(q, *cache, None, win, sinks))
        offsets = torch.arange(len(lengths) + 1, dtype=I32, device="cuda")
        oracle.within(ops.cache_attention(q, *cache, offsets, win, sinks), *oracle.cached(q, *cache, offsets, win, sinks))


def test_a_pool_of_more_than_2_31_values():
    gen = _gen("large pool")
    k, v = (torch.zeros(1_100_000, 16, 1, 128, dtype=BF, device="cuda") for _ in range(2))
    tables = torch.tensor([[1_099_999, 3, 1_060_000], [1_050_001, 1_099_998, -1]], dtype=I32, device="cuda")
    lengths, offsets = torch.tensor([40, 30], dtype=I32, device="cuda"), torch.tensor([0, 40, 70], dtype=I32, device="cuda")
    qkv = _randn(gen, 70, 4, 128)
    q = ops.cache_append(qkv, k, v, tables, lengths, offsets)
    assert torch.equal(q, qkv[:, :2]) and torch.equal(k[1_060_000, :8, 0], qkv[32:40, 2]) and torch.equal(v[1_099_998, :14, 0], qkv[56:, 3])
    got = ops.cache_attention(q, k, v, tables, lengths, offsets)
    near = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=I32, device="cuda")
    used = tables.flatten()[:5].long()
    oracle.within(got, *oracle.cached(q, k[used], v[used], near, lengths, offsets, None, 0))


def test_heads_of_more_than_2_31_values():
    """Rows near the end of tensors of 2.3 billion values."""
    gen = _gen("large heads")
    t, h = 140_000, 128
    x = torch.zeros(1, t, h, 128, dtype=BF, device="cuda")
    tail = _randn(gen, 1, 2, h, 128)
    x[:, -2:] = tail
    positions = torch.arange(t, device="cuda")
    freqs = ops.rotary_frequencies(128)
    y = ops.rotary(x, positions, freqs)[:, -2:]
    assert torch.equal(y, ops.rotary(tail, positions[-2:], freqs))
    del x, y
    # 2 048 sequences whose 32 query heads share a key head
    q, k, v, dy = (torch.zeros(2048, 257, n, 128, dtype=BF, device="cuda") for n in (32, 1, 1, 32))
    for x in (q, k, v, dy):
        x[-1] = _randn(gen, *x.shape[1:])
    want = oracle.window(q[-1:], k[-1:], v[-1:], 8, 0, None, dy[-1:])
    for x in (q, k, v):
        x.requires_grad_()
    out = ops.window_attention(q, k, v, 8)
    oracle.within(out[-1:], *want["y"])
    for g, name in zip(torch.autograd.grad((out,), (q, k, v), (dy,)), ("dq", "dk", "dv")):
        oracle.within(g[-1:], *want[name])
        assert not g[:-1].any()
    nv.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("b,t,h,kv,d,win,sinks,padded", [
    (3, 500, 32, 32, 64, 100, 3, True), (2, 700, 28, 28, 128, None, 0, False), (5, 333, 48, 24, 128, 64, 70, True),
    (1, 2304, 17, 17, 128, None, 0, False), (2, 2200, 10, 10, 128, 2100, 5, True), (1, 2100, 20, 20, 64, 2000, 1, False)])
def test_more_tiles_than_fit_at_once(b, t, h, kv, d, win, sinks, padded):
    gen = _gen("waves", t, d)
    qkv, dy = _randn(gen, b, t, h + 2 * kv, d), _randn(gen, b, t, h, d)
    lengths = None
    if padded:
        lengths = torch.tensor([t - 129 * i for i in range(b)], device="cuda")
        for i, n in enumerate(lengths.tolist()):
            qkv[i, n:], dy[i, n:] = float("nan"), float("nan")
    want = oracle.window(*qkv.split((h, kv, kv), 2), win, sinks, lengths, dy)
    qkv.requires_grad_()
    y = ops.window_attention_qkv(qkv, kv, win, sinks, lengths)
    oracle.within(y, *want["y"])
    with torch.no_grad():
        assert torch.equal(ops.window_attention_qkv(qkv, kv, win, sinks, lengths), y)
    grad, = torch.autograd.grad((y,), (qkv,), (dy,))
    for part, name in zip(grad.split((h, kv, kv), 2), ("dq", "dk", "dv")):
        oracle.within(part, *want[name])
    nv.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("slots,most,h,kv,d,win,sinks", [(16, None, 32, 32, 64, None, 0), (64, 60, 32, 16, 128, 200, 9), (16, 200, 20, 20, 128, None, 0),
                                                         (128, 30, 20, 20, 128, 2100, 2)])
def test_new_tokens_in_waves(slots, most, h, kv, d, win, sinks):
    gen = _gen("new in waves", h, d, most)
    lengths, new = [700, 2400, 90, 33, 1000, 64, 2600], [300, 257, 90, 1, 129, 5, 700]
    cache = _cache(gen, lengths, slots, kv, d, most)
    q = _randn(gen, sum(new), h, d)
    offsets = torch.tensor([0] + new, device="cuda").cumsum(0).to(I32)
    want = oracle.cached(q, *cache, offsets, win, sinks)
    y = ops.cache_attention(q, *cache, offsets, win, sinks)
    oracle.within(y, *want)
    for _ in range(5):
        assert torch.equal(ops.cache_attention(q, *cache, offsets, win, sinks), y)
    nv.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("t,h,kv,win", [(300, 2, 1, 90), (2200, 24, 24, None), (400, 40, 40, 64)])
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_a_number_shows(t, h, kv, win, d):
    """NaN in a query or a key is in every row that sees it, and in no other."""
    gen = _gen("nan", t)
    q, k, v = _randn(gen, 1, t, h, d), _randn(gen, 1, t, kv, d), _randn(gen, 1, t, kv, d)
    clean = ops.window_attention(q, k, v, win)
    q[0, 40, 1, 5], k[0, t // 2, 0, 7] = float("nan"), float("nan")
    y = ops.window_attention(q, k, v, win)
    hurt = torch.zeros(t, h, dtype=torch.bool, device="cuda")
    hurt[40, 1] = True
    hurt[t // 2:t if win is None else t // 2 + win, :h // kv] = True
    assert y[0][hurt].isnan().all() and torch.equal(y[0][~hurt], clean[0][~hurt])
    pages, slots = -(-t // 16), 16
    padded = [torch.nn.functional.pad(x[0], (0, 0, 0, 0, 0, pages * slots - t)).view(pages, slots, kv, d) for x in (k, v)]
    tables, lengths = torch.arange(pages, dtype=I32, device="cuda")[None], torch.tensor([t], dtype=I32, device="cuda")
    got = ops.cache_attention(q[0], *padded, tables, lengths, torch.tensor([0, t], dtype=I32, device="cuda"), win)
    assert got[hurt].isnan().all() and got[~hurt].isfinite().all()
    last = ops.cache_attention(q[0, t // 2:t // 2 + 1], *padded, tables, lengths - (t - t // 2 - 1), None, win)
    assert last[0, :h // kv].isnan().all() and last[0, h // kv:].isfinite().all()
    nv.check_status(torch.device("cuda", 0))


def test_windows_beyond_the_kernels_integers():
    gen = _gen("far windows")
    qkv, dy = _randn(gen, 1, 300, 6, 64).requires_grad_(), _randn(gen, 1, 300, 2, 64)
    cache = _cache(gen, [300, 200], 16, 2, 64)
    q = _randn(gen, 2, 4, 64)

    def everything(window, sinks):
        y = ops.window_attention_qkv(qkv, 2, window, sinks)
        return [y, *torch.autograd.grad((y,), (qkv,), (dy,)), ops.cache_attention(q, *cache, None, window, sinks)]

    for window, sinks, same in ((2 ** 32 + 5, 3, (None, 0)), (2 ** 40, 2 ** 40, (None, 0)), (70, 2 ** 32 + 1, (70, 300))):
        assert all(torch.equal(a, b) for a, b in zip(everything(window, sinks), everything(*same)))
    nv.check_status(torch.device("cuda", 0))
