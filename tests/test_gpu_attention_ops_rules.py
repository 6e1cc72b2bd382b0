"""Rotary positions, windowed attention and the paged cache on the kernels: what each call promises beyond ordinary inputs."""
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


def _gradients(q, k, v, dy, window, sinks=0, lengths=None):
    """All of a call against 64 bits; the gradients are returned."""
    want = oracle.window(q, k, v, window, sinks, lengths, dy)
    at = [x.clone().requires_grad_() for x in (q, k, v)]
    y = ops.window_attention(*at, window, sinks, lengths)
    oracle.within(y, *want["y"])
    grads = torch.autograd.grad((y,), at, (dy,))
    nv.check_status(q.device)
    for g, name in zip(grads, ("dq", "dk", "dv")):
        oracle.within(g, *want[name])
    return grads


# ------------------------------------------------------------------------------------------------------------------
# gradients of a scaled loss
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128])
def test_scores_gradients_in_half_are_finite_where_the_definition_is(d):
    """Two equal scores, values of 1 and -1, a gradient of 4096 in all channels: the score's gradient is 32 d sqrt(d), 16 384 and
    46 341, and before its scale 131 072 and 262 144, which half does not have."""
    q, k, v = (torch.zeros(1, 2, 1, d, dtype=HALF, device="cuda") for _ in range(3))
    q[..., 0] = 0.5
    k[0, 0, 0, 1], k[0, 1, 0, 1] = 0.5, -0.5
    v[0, 0], v[0, 1] = 1.0, -1.0
    dy = torch.full((1, 2, 1, d), 4096.0, dtype=HALF, device="cuda")
    dq, _, _ = _gradients(q, k, v, dy, None)
    assert float(dq[0, 1, 0, 1]) == pytest.approx(2048.0 * d * d ** -0.5, rel=2.0 ** -10)


@pytest.mark.parametrize("t,h,kv,d,win,sinks", [(70, 2, 1, 64, 2, 0), (300, 4, 2, 128, 3, 0), (200, 2, 2, 96, 2, 0)])
def test_large_gradients_in_half(t, h, kv, d, win, sinks):
    gen = _gen("large", t)
    q, k = _randn(gen, 1, t, h, d, dtype=HALF, scale=0.25), _randn(gen, 1, t, kv, d, dtype=HALF, scale=0.25)
    v, dy = _randn(gen, 1, t, kv, d, dtype=HALF), _randn(gen, 1, t, h, d, dtype=HALF, scale=10000.0)
    _gradients(q, k, v, dy, win, sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_delta_has_what_rounding_took_off_the_output(d, dtype):
    """Two equal scores over equal keys: the gradient of the query is nothing at all, the two scores' gradients cancel.  The values are
    one step of the type apart, so that the output, half way between, loses as much in rounding as they differ by: with delta from the
    rounded output alone the gradient is tens of times the bound."""
    gen = _gen("residual", d)
    t, h, kv, unit = 300, 4, 2, oracle.UNIT[dtype]
    q, k = torch.zeros(1, t, h, d, dtype=dtype, device="cuda"), torch.ones(1, t, kv, d, dtype=dtype, device="cuda")
    v = (1.0 + 2 * unit * torch.randint(0, 2, (1, t, kv, d), generator=gen, device="cuda")).to(dtype)
    dy = _randn(gen, 1, t, h, d, dtype=dtype)
    dy *= torch.arange(d, device="cuda") % (d // 8) == torch.arange(t, device="cuda").view(t, 1, 1) % (d // 8)     # eight channels a token
    q.requires_grad_()
    dq, = torch.autograd.grad((ops.window_attention(q, k, v, 2),), (q,), (dy,))
    nv.check_status(q.device)
    g, two = dy[0].double(), v[0].repeat_interleave(h // kv, 1).double()
    two = torch.stack([two, torch.cat([two[:1], two[:-1]])])           # the token and the one before; the first sees itself only
    out = two.mean(0)
    dp, delta = (two * g).sum(-1), (out * g).sum(-1)
    mass = (two * g).abs().sum(-1).amax(0)
    # sums of eight products in fp32, delta from an output and a residual in 16 bits, dS rounded
    wrong = (8 + 8) * 2.0 ** -24 * 2 * mass + unit ** 2 * mass + 2.0 ** -19 * (dp - delta).abs().amax(0)
    wrong = d ** -0.5 * (wrong + unit * (dp - delta).abs().amax(0)) + 2 * oracle.FLOOR[dtype]
    assert bool((dq[0].double().abs().amax(-1) <= wrong).all())
    planted = d ** -0.5 * (dp - (out.to(dtype).double() * g).sum(-1)).mean(0).abs()
    assert int((planted > 10 * wrong).sum()) > t * h // 2


# ------------------------------------------------------------------------------------------------------------------
# the paged cache
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [0, 1])
@pytest.mark.parametrize("backend", ["auto", "torch"])
def test_append_is_seen_by_a_backward_that_saved_the_pages(page, backend):
    gen = _gen("versions")
    cache = (_randn(gen, 3, 8, 1, 64), _randn(gen, 3, 8, 1, 64), torch.tensor([[0, 1]], dtype=I32, device="cuda"),
             torch.tensor([5], dtype=I32, device="cuda"))
    weight = torch.ones(64, dtype=BF, device="cuda", requires_grad=True)
    loss = (cache[page] * weight).sum()
    ops.set_backend(backend)
    try:
        ops.cache_append(_randn(gen, 1, 4, 64), *cache)
    finally:
        ops.set_backend("auto")
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ------------------------------------------------------------------------------------------------------------------
# one tile a thread block, two thread blocks a multiprocessor
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t,h,win,sinks", [(1300, 14, None, 0), (1100, 32, 700, 130), (640, 59, 64, 0)])
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_as_many_tiles_as_thread_blocks_fit(t, h, win, sinks, dtype):
    """150 to 296 tiles of heads of 64, whose ring of keys goes round more than once."""
    assert 149 <= -(-t // 128) * h <= 296
    gen = _gen("tiles", t)
    _gradients(*(_randn(gen, 1, t, h, 64, dtype=dtype) for _ in range(4)), win, sinks)


def _cache(gen, lengths, slots, kv, d, dtype=BF):
    per = [-(-n // slots) for n in lengths]
    tables = torch.full((len(lengths), max(per)), -1, dtype=I32, device="cuda")
    order, at = torch.randperm(sum(per), generator=gen, device="cuda").to(I32), 0
    for b, n in enumerate(per):
        tables[b, :n] = order[at:at + n]
        at += n
    return (*(_randn(gen, sum(per), slots, kv, d, dtype=dtype) for _ in range(2)), tables, torch.tensor(lengths, dtype=I32, device="cuda"))


@pytest.mark.parametrize("win,sinks", [(None, 0), (100, 20)])
def test_as_many_tiles_over_a_cache_as_thread_blocks_fit(win, sinks):
    gen = _gen("cached tiles")
    cache = _cache(gen, [900] * 10, 16, 8, 64)
    q, offsets = _randn(gen, 1450, 16, 64), (torch.arange(11, device="cuda") * 145).to(I32)
    oracle.within(ops.cache_attention(q, *cache, offsets, win, sinks), *oracle.cached(q, *cache, offsets, win, sinks))
    nv.check_status(q.device)


# ------------------------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width", [64, 66])
def test_rotary_at_far_positions(width, interleaved):
    """Whole pieces and any, against the definition of the same frequencies in 64 bits."""
    gen = _gen("far", width)
    positions = torch.tensor([[0, 2 ** 31 - 1, 2 ** 38 + 5, -(2 ** 40) - 3, 2 ** 48 + 1]], device="cuda")
    freqs = ops.rotary_frequencies(64)
    x = _randn(gen, 1, 5, 3, width, dtype=HALF)
    want = ops.rotary(x.double(), positions, freqs, interleaved=interleaved)
    reach = x.double().abs().amax(-1, keepdim=True) * 2
    # the angle (32 bits of a turn, rounded to 24), its sine and cosine and three roundings in fp32, one of the result
    angle = 2 * math.pi * (2.0 ** -26 + 2.0 ** -32)
    bound = oracle.UNIT[HALF] * want.abs() + oracle.FLOOR[HALF] + (angle + 2.0 ** -20) * reach
    oracle.within(ops.rotary(x, positions, freqs, interleaved=interleaved), want, bound)


# ------------------------------------------------------------------------------------------------------------------
# rows that belong to no sequence
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lengths,new,h,kv,d", [([300, 40], [2, 5], 4, 2, 64), ([2000, 900], [1, 1], 8, 2, 128), ([700, 300], [200, 90], 6, 2, 128),
                                                ([260], [150], 40, 8, 64)])
@pytest.mark.parametrize("front", [1, 130, 300])
def test_rows_of_no_sequence_are_zeros(lengths, new, h, kv, d, front):
    """In front of the first offset and behind the last, where memory held something else."""
    gen = _gen("rows", lengths, front)
    cache = _cache(gen, lengths, 16, kv, d)
    n = front + sum(new) + 3
    q = _randn(gen, n, h, d)
    offsets = (front + torch.tensor([0] + new, device="cuda").cumsum(0)).to(I32)
    for win in (None, 100):
        want = oracle.cached(q, *cache, offsets, win, 0)
        for _ in range(3):
            spoilt = [torch.full(s, math.nan, dtype=BF, device="cuda") for s in ((n, h, d),) * 3]
            del spoilt
            y = ops.cache_attention(q, *cache, offsets, win)
            oracle.within(y, *want)
            assert not y[:front].any() and not y[front + sum(new):].any()
    nv.check_status(q.device)


def test_append_of_rows_that_offsets_go_beyond():
    """Offsets behind the last row: the rows that are there are the last ones of their sequences, as the definition has it and as the
    attention over them takes them."""
    gen = _gen("beyond")
    cache, qkv = _cache(gen, [40, 30], 16, 1, 64), _randn(gen, 5, 4, 64)
    offsets = torch.tensor([1, 3, 9], dtype=I32, device="cuda")
    freqs = ops.rotary_frequencies(64)
    got, want = ([x.clone() for x in cache[:2]] for _ in range(2))
    q = ops.cache_append(qkv, *got, *cache[2:], offsets, freqs)
    y = ops.cache_attention(q, *got, *cache[2:], offsets)
    ops.set_backend("torch")
    try:
        q_want = ops.cache_append(qkv, *want, *cache[2:], offsets, freqs)
    finally:
        ops.set_backend("auto")
    for a, b in ((q, q_want), *zip(got, want)):        # one rounding each, of fp32 values that are 2^-20 of terms of size 8 apart
        assert bool(((a.double() - b.double()).abs() <= 2 * oracle.UNIT[BF] * b.double().abs() + 2.0 ** -16).all())
    for a, b, c in zip(got, want, cache):
        assert torch.equal((a != c).any(-1), (b != c).any(-1))         # the same slots
    oracle.within(y, *oracle.cached(q, *got, *cache[2:], offsets.clamp(max=5), None, 0))
    assert not y[0].any() and not q[0].any()


# ------------------------------------------------------------------------------------------------------------------
# the decoder
# ------------------------------------------------------------------------------------------------------------------
def test_a_refused_step_leaves_the_cache_as_it_was():
    from fbamtrain_b200.models import AttentionDecoder, PagedCache
    from fbamtrain_b200.models.init_utils import SeedSequence

    def model(dim):
        return AttentionDecoder(frame_dim=24, dim=dim, layers=2, heads=4, inner=32, vocab=37, dtype=BF, seeds=SeedSequence(3), kv_heads=2,
                                window=9, sinks=2).cuda()

    decoder, gen = model(256), _gen("decoder")
    cache, frames, previous = decoder.make_cache(2, 40, slots=8), _randn(gen, 5, 24), torch.arange(5, device="cuda")
    decoder.extend(frames, previous, cache, [4, 1])
    before = [x.clone() for x in (cache.k, cache.v, cache.tables, cache.lengths)]
    for bad in (dict(frames=frames[:, :23]), dict(frames=frames.half()), dict(frames=frames.cpu()), dict(previous=previous[:4]), dict(top=99),
                dict(temperature=0.0), dict(new=[6, -1]), dict(new=[0, 5], previous=previous.cpu())):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            decoder.extend(**{"frames": frames, "previous": previous, "cache": cache, "new": [2, 3], **bad})
        assert cache._lengths == [4, 1]
    for a, b in zip(before, (cache.k, cache.v, cache.tables, cache.lengths)):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    other = model(384)                                    # 96 channels a head
    with pytest.raises(ValueError, match="64 or 128"):
        other.make_cache(2, 40)
    by_hand = PagedCache(2, 9, 8, 2, 96, 2, 40, BF, "cuda", 9, 2)
    with pytest.raises(ValueError, match="64 or 128"):
        other.extend(frames, previous, by_hand, [2, 3])
    assert by_hand.lengths.tolist() == [0, 0]
    nv.check_status(frames.device)


def test_a_step_without_frames():
    from fbamtrain_b200.models import AttentionDecoder
    from fbamtrain_b200.models.init_utils import SeedSequence
    decoder = AttentionDecoder(frame_dim=24, dim=256, layers=2, heads=4, inner=32, vocab=37, dtype=BF, seeds=SeedSequence(3), window=9).cuda()
    cache, frames, previous = decoder.make_cache(2, 40, slots=8), _randn(_gen("none"), 5, 24), torch.arange(5, device="cuda")
    decoder.extend(frames, previous, cache, [4, 1])
    nothing = decoder.extend(frames[:0], previous[:0], cache, [0, 0], top=3)
    assert nothing.entropy.shape == (0,) and nothing.top_ids.shape == nothing.top_logprobs.shape == (0, 3)
    assert cache.lengths.tolist() == [4, 1]
    with pytest.raises(ValueError):
        decoder.extend(frames[:0], previous[:0], cache, [0, 0, 0])
    nv.check_status(frames.device)


# ------------------------------------------------------------------------------------------------------------------
# lengths
# ------------------------------------------------------------------------------------------------------------------
def test_lengths_beyond_32_bits():
    gen = _gen("lengths")
    heads = [_randn(gen, 4, 150, n, 64) for n in (2, 1, 1, 2)]
    far = torch.tensor([2 ** 32 + 3, -2 ** 32 + 3, 150, 2 ** 62], device="cuda")
    for lengths in (far, far.clamp(-1, 151).to(I32), torch.tensor([150, 0, 150, 150], device="cuda")):
        _gradients(*heads, 40, 3, lengths)
