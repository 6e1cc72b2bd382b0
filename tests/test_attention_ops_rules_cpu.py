"""Rotary positions, windowed attention and the paged cache without a GPU: what each call promises beyond ordinary inputs."""
import copy
import decimal
import io
import math
import os
import pickle
import re
from fractions import Fraction

import pytest
import torch

import attention_oracle as oracle
import fbamtrain_b200
from fbamtrain_b200 import ops

BF = torch.bfloat16
I32 = torch.int32


class Library:
    """Takes the place of the kernels: every entry succeeds and does nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, entry):
        return lambda *args: self.calls.append((entry, args)) or 0


@pytest.fixture
def library(monkeypatch):
    from fbamtrain_b200.ops import native
    fake = Library()
    monkeypatch.setattr(native, "lib", lambda like=None: fake)
    monkeypatch.setattr(native, "stream", lambda: 0)
    monkeypatch.setattr(native, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    return fake


def _small_cache(dtype=torch.float32):
    k, v = torch.randn(3, 8, 1, 64).to(dtype), torch.randn(3, 8, 1, 64).to(dtype)
    return k, v, torch.tensor([[0, 1]], dtype=I32), torch.tensor([5], dtype=I32)


# ------------------------------------------------------------------------------------------------------------------
# writes into the pages
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["definition", "kernels"])
@pytest.mark.parametrize("page", [0, 1])
def test_append_is_seen_by_a_backward_that_saved_the_pages(which, page, library):
    cache = _small_cache(BF)
    weight = torch.ones(64, dtype=BF, requires_grad=True)
    loss = (cache[page] * weight).sum()                                 # saves the pages
    qkv = torch.randn(1, 4, 64).to(BF)
    if which == "definition":
        ops.cache_append(qkv, *cache)
    else:
        from fbamtrain_b200.ops.positions import cache_append
        cache_append(qkv, *cache, None, None, False, 2, 1)
        assert [entry for entry, _ in library.calls] == ["fbam_cache_append"]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_append_to_pages_that_count_no_versions(library):
    """Pages of inference mode, as a cache that is made there has them."""
    from fbamtrain_b200.ops.positions import cache_append
    with torch.inference_mode():
        cache_append(torch.randn(1, 4, 64).to(BF), *_small_cache(BF), None, None, False, 2, 1)
        ops.cache_append(torch.randn(1, 4, 64).to(BF), *_small_cache(BF))
    cache = _small_cache(BF)
    with torch.inference_mode():
        cache_append(torch.randn(1, 4, 64).to(BF), *cache, None, None, False, 2, 1)


def test_the_cache_operators_beside_tangents():
    """A level of forward differentiation is no tangent: what has none passes, what has one is refused, without gradients too."""
    from torch.autograd import forward_ad
    cache, q, qkv = _small_cache(), torch.randn(1, 2, 64), torch.randn(1, 4, 64)

    def dual(x):
        return forward_ad.make_dual(x, torch.ones_like(x))

    want = ops.cache_attention(q, *cache)
    with forward_ad.dual_level():
        assert torch.equal(ops.cache_append(qkv, *(x.clone() for x in cache)), qkv[:, :2])
        assert torch.equal(ops.cache_attention(q, *cache), want)
        for taken in (torch.enable_grad, torch.no_grad):
            with taken():
                for call in (lambda: ops.cache_attention(dual(q), *cache), lambda: ops.cache_append(dual(qkv), *cache),
                             lambda: ops.cache_attention(q, cache[0], dual(cache[1]), *cache[2:])):
                    with pytest.raises(RuntimeError, match="no gradient"):
                        call()


# ------------------------------------------------------------------------------------------------------------------
# slots that nobody sees
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,win,sinks", [(1, 10, 0), (1, 10, 5), (7, 10, 5), (20, 30, 17), (60, 3, 1), (3, None, 0)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_the_definition_of_cache_attention_reads_what_queries_see(new, win, sinks, value):
    """Slots between the first tokens and the window, and behind the sequence, of pages that are still in the table."""
    gen = torch.Generator().manual_seed(1)
    k, v = torch.randn(10, 8, 2, 6, generator=gen), torch.randn(10, 8, 2, 6, generator=gen)
    tables, lengths = torch.tensor([[3, 7, 1, 0, 9, 5, 2, 8]], dtype=I32), torch.tensor([60], dtype=I32)
    offsets, q = torch.tensor([0, new], dtype=I32), torch.randn(new, 4, 6, generator=gen)
    for j in range(64):
        if j >= 60 or (win is not None and sinks <= j <= 60 - new - win):
            k[tables[0, j // 8], j % 8] = v[tables[0, j // 8], j % 8] = value
    y = ops.cache_attention(q, k, v, tables, lengths, offsets, win, sinks)
    oracle.within(y, *oracle.cached(q, k, v, tables, lengths, offsets, win, sinks))


# ------------------------------------------------------------------------------------------------------------------
# frequencies
# ------------------------------------------------------------------------------------------------------------------
def test_frequencies_and_a_model_that_has_them_are_pickled():
    from fbamtrain_b200.models import AttentionDecoder
    from fbamtrain_b200.models.init_utils import SeedSequence
    freqs = ops.rotary_frequencies(64, factor=4.0, context=100)
    for _ in range(2):
        for other in (pickle.loads(pickle.dumps(freqs)), copy.deepcopy(freqs)):
            assert other == freqs and other.dims == 64 and list(other.table) == list(freqs.turns)      # from here on with a table of its own
    model = AttentionDecoder(frame_dim=8, dim=32, layers=1, heads=2, inner=16, vocab=5, dtype=torch.float32, seeds=SeedSequence(1))
    file = io.BytesIO()
    torch.save(model, file)
    file.seek(0)
    other = torch.load(file, weights_only=False)
    args = torch.randn(1, 4, 8), torch.tensor([[-1, 2, 3, 1]]), torch.tensor([[2, 3, 1, 0]])
    assert other.freqs == model.freqs and torch.equal(other(*args).logprob, model(*args).logprob)


def _speeds(dims, digits=45):
    """Of base 10^(dims / 2), whose pairs turn by 10^-i radians a position: that in turns, exact to ``digits``."""
    def inverse_tangent(n):                                             # of 1 / n, by its series
        total, term, i = 0, 10 ** digits // n, 1
        while term:
            total += term // i if i % 4 == 1 else -(term // i)
            term //= n * n
            i += 2
        return total
    pi = 4 * (4 * inverse_tangent(5) - inverse_tangent(239))            # Machin's formula
    return [Fraction(10 ** digits, 2 * pi * 10 ** i) for i in range(dims // 2)]


@pytest.mark.parametrize("settings", [{}, {"factor": 4.0}, {"factor": 8.0, "context": 512}, {"factor": 5.0, "context": 3000, "few": 2.0, "many": 40.0}])
def test_frequencies_fill_their_64_bits(settings):
    freqs = ops.rotary_frequencies(8, base=10000.0, **settings)
    for got, turn in zip(freqs.turns, _speeds(8)):
        factor = Fraction(settings.get("factor", 1))
        if "context" in settings:
            few, many = Fraction(settings.get("few", 1)), Fraction(settings.get("many", 32))
            kept = min(Fraction(1), max(Fraction(0), (turn * settings["context"] - few) / (many - few)))
            turn *= kept + (1 - kept) / factor
        else:
            turn /= factor
        assert abs(got - turn * 2 ** 64) <= Fraction(1, 2) + Fraction(1, 10 ** 9)


def test_frequencies_do_not_depend_on_the_callers_decimal_context():
    want = ops.rotary_frequencies(64, factor=3.0, context=50)
    with decimal.localcontext(prec=5, rounding=decimal.ROUND_UP) as around:
        around.traps[decimal.Inexact] = True
        assert ops.rotary_frequencies(64, factor=3.0, context=50) == want


def test_the_definition_of_rotary_at_far_positions():
    """In 64 bits: the angle is off by 2^-65 of a turn a position, and by the roundings of a double."""
    positions = [1, 2 ** 31 - 1, 10 ** 12 + 7, -(2 ** 44) - 3, 2 ** 50 + 1]
    x = torch.tensor([[1.0] * 4 + [0.0] * 4], dtype=torch.float64).expand(1, len(positions), 1, 8)
    y = ops.rotary(x, torch.tensor([positions]), ops.rotary_frequencies(8))
    for n, p in enumerate(positions):
        for i, turn in enumerate(_speeds(8)):
            angle = 2 * math.pi * float((p * turn) % 1)
            bound = 2 * math.pi * (abs(p) * 2.0 ** -65) + 2.0 ** -48
            assert abs(float(y[0, n, 0, i]) - math.cos(angle)) <= bound and abs(float(y[0, n, 0, 4 + i]) - math.sin(angle)) <= bound


# ------------------------------------------------------------------------------------------------------------------
# waits that run out
# ------------------------------------------------------------------------------------------------------------------
def _meetings(source):
    """Of each named barrier in CUDA source: the headers of the blocks around it and the start of its own statement."""
    code = re.sub(r"//[^\n]*", "", source)
    code = re.sub(r"^\s*#[^\n]*", "", code, flags=re.M)
    around, start, out, nested = [], 0, [], 0
    for i, c in enumerate(code):
        if code.startswith('"bar.sync', i):
            out.append(around + [code[start:i]])
        nested += (c == "(") - (c == ")")
        if c == "{" and nested == 0:
            around.append(code[start:i])
        elif c == "}" and nested == 0:
            around.pop()
        if c in "{};" and nested == 0:
            start = i + 1
    assert not around
    return out


def test_warps_meet_whether_or_not_a_wait_of_theirs_expired():
    """Warps that meet at a named barrier each have waited for themselves: one whose wait ran out has to come as well."""
    for name in ("window_attention.cu", "window_attention_bwd.cu"):
        with open(os.path.join(os.path.dirname(fbamtrain_b200.__file__), "csrc", name)) as f:
            found = _meetings(f.read())
        assert len(found) == 2
        for around in found:
            conditions = [h for h in around if re.search(r"\b(if|for|while)\b", h)]
            assert conditions and not any(re.search(r"\bok\b|mbar_wait", h) for h in conditions), conditions


@pytest.mark.parametrize("dtype", [I32, torch.int64])
def test_lengths_reach_the_kernels_as_what_they_are(dtype):
    """Beyond 32 bits too, where they are as good as the largest, or as none."""
    from fbamtrain_b200.ops.window import _lengths
    far = [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 62, -2 ** 63] if dtype == torch.int64 else []
    lengths = torch.tensor([0, 7, 2 ** 31 - 1, -5] + far, dtype=dtype)
    got = _lengths(lengths, lengths)
    assert got.dtype == I32 and [max(n, 0) for n in got.tolist()] == [0, 7, 2 ** 31 - 1, 0] + [2 ** 31 - 1, 0] * (len(far) // 2)


# ------------------------------------------------------------------------------------------------------------------
# nothing at all
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("b,t", [(0, 3), (2, 0), (0, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_gradients_of_no_tokens_are_empty(b, t, dtype):
    q, k, v = (torch.randn(b, t, n, 8).to(dtype).requires_grad_() for n in (4, 2, 2))
    lengths = torch.zeros(b, dtype=I32)
    for how in ((None, 0, None), (3, 1, lengths)):
        y = ops.window_attention(q, k, v, *how)
        assert y.shape == q.shape and y.dtype == dtype
        assert [g.shape for g in torch.autograd.grad((y.float().sum(),), (q, k, v))] == [q.shape, k.shape, v.shape]
    qkv = torch.randn(b, t, 8, 8).to(dtype).requires_grad_()
    for y in (ops.window_attention_qkv(qkv, 2, 3), ops.rotary(qkv, torch.arange(t), ops.rotary_frequencies(8))):
        assert torch.autograd.grad((y.float().sum(),), (qkv,))[0].shape == qkv.shape


# ------------------------------------------------------------------------------------------------------------------
# plans
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t,kv,group", [(13_400_064, 232, 1), (11_783_936, 150, 2), (51_025_920, 4, 4), (2_000_000, 1, 1)])
def test_workspace_of_walks_beyond_an_integer(t, kv, group):
    """Where a multiprocessor has more tiles to do than an int holds, walks are not divided: the workspace is dQ's sums, counters and
    delta only.  Where they are divided, by what one has to do."""
    from fbamtrain_b200.ops import native
    rows = 128 // group
    tiles, blocks = -(-t // rows), -(-t // 128)
    got = native.lib().fbam_window_bwd_workspace(1, t, kv, group, 64, 0, 0)
    least = kv * tiles * 128 * 64 + (kv * tiles + 1 + 3) // 4 * 4 + kv * tiles * 128
    parts = blocks * kv * 2 * 128 * 64
    share = blocks * tiles * kv // 296
    assert got == least + (0 if share >= tiles else -(-tiles // share) * parts)


# ------------------------------------------------------------------------------------------------------------------
# the decoder
# ------------------------------------------------------------------------------------------------------------------
def _decoder(heads=4, dim=256, **how):
    from fbamtrain_b200.models import AttentionDecoder
    from fbamtrain_b200.models.init_utils import SeedSequence
    how = {"layers": 2, "kv_heads": 2, "window": 9, "sinks": 2, **how}
    return AttentionDecoder(frame_dim=24, dim=dim, heads=heads, inner=32, vocab=37, dtype=torch.float32, seeds=SeedSequence(3), **how)


@pytest.mark.parametrize("heads,dim,fits", [(4, 256, True), (2, 256, True), (4, 384, False), (4, 128, False)])
def test_a_cache_that_the_kernels_do_not_take_is_refused_when_it_is_made(heads, dim, fits, monkeypatch):
    """64 and 128 channels a head; 96 and 32, which train."""
    from fbamtrain_b200.ops import dispatch
    model = _decoder(heads, dim)
    cache = model.make_cache(2, 50)
    assert cache.k.shape[-1] == dim // heads                                # the definitions take any
    monkeypatch.setattr(dispatch, "_native_inner", lambda t, dtype, family: True)
    if fits:
        model.make_cache(2, 50)
        return
    with pytest.raises(ValueError, match="64 or 128"):
        model.make_cache(2, 50)
    with pytest.raises(ValueError, match="64 or 128"):
        model.step(torch.randn(2, 24), torch.tensor([1, 2]), cache)
    assert cache.lengths.tolist() == [0, 0]


def test_a_refused_step_leaves_the_cache_as_it_was():
    """A call that raises has counted no tokens and taken no pages, so that it can be made again; with pages of another model, or of one
    that looks further back, it is refused."""
    from fbamtrain_b200.models import PagedCache
    model, gen = _decoder(), torch.Generator().manual_seed(2)
    cache = model.make_cache(2, 40, slots=8)
    frames, previous = torch.randn(5, 24, generator=gen), torch.tensor([1, 2, 3, 4, 5])
    model.extend(frames, previous, cache, [4, 1])

    def state():
        return [x.clone() for x in (cache.k, cache.v, cache.tables, cache.lengths)], list(cache._lengths), cache.free_pages

    def same(a, b):
        return all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(a[0], b[0])) and a[1:] == b[1:]

    before = state()
    for bad in (dict(frames=frames[:, :23]), dict(previous=previous[:4]), dict(previous=previous.view(1, 5)), dict(previous=previous.float()),
                dict(frames=frames.double()), dict(top=99), dict(top=-1), dict(temperature=0.0), dict(new=[6, -1]), dict(new=[2, 2]),
                dict(new=[2.5, 2.5]), dict(new=[5]), dict(new=[5, 0, 0]), dict(new=[0, 5], frames=frames[:0])):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            model.extend(**{"frames": frames, "previous": previous, "cache": cache, "new": [2, 3], **bad})
        assert same(state(), before), bad
    got = model.extend(frames, previous, cache, torch.tensor([2, 3]))
    assert got.entropy.shape == (5,) and cache.lengths.tolist() == [6, 4]

    nothing = model.extend(frames[:0], previous[:0], cache, [0, 0])
    assert nothing.entropy.shape == (0,) and nothing.top_ids.shape == (0, 1) and cache.lengths.tolist() == [6, 4]

    def of(layers=2, kv=2, d=64, dtype=torch.float32, window=9, sinks=2):
        return PagedCache(layers, 6, 8, kv, d, 2, 40, dtype, "cpu", window, sinks)

    for fits in (of(), of(window=None), of(window=20, sinks=30), of(window=9, sinks=2)):
        model.extend(frames, previous, fits, [2, 3])
    for other in (of(layers=1), of(layers=3), of(kv=4), of(d=32), of(dtype=torch.float64), of(window=8), of(sinks=1)):
        with pytest.raises(ValueError, match="model"):
            model.extend(frames, previous, other, [2, 3])
        assert other.lengths.tolist() == [0, 0]
    with pytest.raises(ValueError, match="model"):
        _decoder(window=None).extend(frames, previous, of(), [2, 3])


def test_a_cache_serves_in_and_out_of_inference_mode():
    """Wherever it was made."""
    model, gen = _decoder(), torch.Generator().manual_seed(4)
    frames, previous = torch.randn(5, 24, generator=gen), torch.tensor([1, 2, 3, 4, 5])
    answers = []
    for made in (True, False):
        with torch.inference_mode(made):
            cache = model.make_cache(2, 40, slots=8)
        for mode in (True, False, True):
            with torch.inference_mode(mode):
                r = model.extend(frames, previous, cache, [2, 3])
        cache.reset(0)
        assert cache.lengths.tolist() == [0, 9]
        answers.append(r.entropy)
    assert torch.equal(*answers)
