"""The action model with a window of frames: whole sequences against chunks and single steps over its cache, gradients, and the cache's
pages."""
import pytest
import torch

from fbamtrain_b200.models import AttentionDecoder, PagedCache
from fbamtrain_b200.models.init_utils import SeedSequence


def _model(dtype, device, **how):
    how = {"kv_heads": 2, "window": 9, "sinks": 2, **how}
    return AttentionDecoder(frame_dim=24, dim=256, layers=2, heads=4, inner=96, vocab=37, dtype=dtype, seeds=SeedSequence(3), **how).to(device)


def _batch(dtype, device, b=3, t=45):
    gen = torch.Generator().manual_seed(5)
    frames = torch.randn(b, t, 24, generator=gen).to(dtype).to(device)
    actions = torch.randint(0, 37, (b, t), generator=gen).to(device)
    previous = torch.cat([torch.full_like(actions[:, :1], -1), actions[:, :-1]], 1)
    return frames, previous, actions


def _pieces_match_the_whole(dtype, device, tolerance, **how):
    """Recordings that advance by different numbers of frames, down to single steps of all, in a cache of no spare page."""
    model, (frames, previous, actions) = _model(dtype, device, **how), _batch(dtype, device)
    b, t = actions.shape
    with torch.no_grad():
        whole = model(frames, previous, actions, top=4)
    cache = model.make_cache(b, t, slots=8, pages=b * 6)
    at = [0] * b
    for new in ([20, 0, 3], [1, 7, 2], [0, 1, 0], [3, 3, 3]) + ([1, 1, 1],) * 21:
        rows = [(i, at[i] + j) for i, n in enumerate(new) for j in range(n)]
        who, when = (torch.tensor(x, device=device) for x in zip(*rows))
        if new == [1, 1, 1]:
            got = model.step(frames[who, when], previous[who, when], cache, top=4)
        else:
            got = model.extend(frames[who, when], previous[who, when], cache, new, top=4)
        at = [a + n for a, n in zip(at, new)]
        torch.testing.assert_close(got.entropy, whole.entropy[who, when], rtol=0, atol=tolerance)
        torch.testing.assert_close(got.top_logprobs, whole.top_logprobs[who, when], rtol=0, atol=tolerance)
    assert cache.lengths.tolist() == at


def _padding_has_no_influence(dtype, device):
    model, (frames, previous, actions) = _model(dtype, device), _batch(dtype, device)
    lengths = torch.tensor([45, 17, 0], device=device)
    other, far = frames.clone(), actions.clone()
    for i, n in enumerate(lengths.tolist()):
        other[i, n:], far[i, n:] = 3.0, -1
    params = list(model.parameters())
    got = []
    for x in (frames, other):
        r = model(x, previous, far, lengths)
        keep = far >= 0
        got.append([r.logprob.detach()[keep], *torch.autograd.grad(r.logprob.sum(), params)])
    for one, two in zip(*got):
        # the padded rows take part in the gradients' products, with zeros
        torch.testing.assert_close(one, two, rtol=0, atol=1e-5 if dtype == torch.float32 else float(one.abs().max()) * 2.0 ** -8)


def test_decoder_cpu():
    _pieces_match_the_whole(torch.float32, "cpu", 1e-4)
    _pieces_match_the_whole(torch.float32, "cpu", 1e-4, window=None, sinks=0, kv_heads=4, factor=2.0, context=16)
    _padding_has_no_influence(torch.float32, "cpu")


def test_decoder_gradients_are_differences():
    """Along its own direction, against a central difference of fp32 values of size 3 (2^-21 each) over a step of 0.01: rounding
    is off by 1e-4, the third derivative by some 1e-4 more; the gradient is larger than 0.1."""
    model, (frames, previous, actions) = _model(torch.float32, "cpu"), _batch(torch.float32, "cpu")
    params = list(model.parameters())

    def value():
        r = model(frames, previous, actions)
        return r.logprob.mean() + 0.1 * r.entropy.mean()

    grads = torch.autograd.grad(value(), params)
    assert all(bool(g.any()) for g in grads)
    norm = float(sum(g.double().pow(2).sum() for g in grads).sqrt())
    assert norm > 0.1
    ends = []
    with torch.no_grad():
        for sign in (1.0, -2.0):
            for p, g in zip(params, grads):
                p += sign * 0.01 / norm * g
            ends.append(float(value()))
    assert (ends[0] - ends[1]) / 0.02 == pytest.approx(norm, rel=1e-2)


# As for the recurrent decoder: 16-bit activations of size 1 whose roundings change with the order of fp32 sums.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tolerance", [(torch.bfloat16, 8 * 2.0 ** -8), (torch.float16, 8 * 2.0 ** -11)])
def test_decoder_gpu(dtype, tolerance):
    _pieces_match_the_whole(dtype, "cuda", tolerance)
    _pieces_match_the_whole(dtype, "cuda", tolerance, window=None, sinks=0, kv_heads=1, factor=2.0, context=16)
    _padding_has_no_influence(dtype, "cuda")


@pytest.mark.gpu
def test_decoder_gpu_matches_the_definitions():
    """Values within eight roundings; gradients within sixteen of their norm, two layers' activations being rounded on the way."""
    from fbamtrain_b200 import ops
    model, (frames, previous, actions) = _model(torch.bfloat16, "cuda"), _batch(torch.bfloat16, "cuda")
    params = list(model.parameters())

    def all_of_it():
        r = model(frames, previous, actions)
        return r.logprob.detach(), torch.autograd.grad(r.logprob.mean(), params)

    got, grads = all_of_it()
    ops.set_backend("torch")
    try:
        want, want_grads = all_of_it()
    finally:
        ops.set_backend("auto")
    torch.testing.assert_close(got, want, rtol=0, atol=8 * 2.0 ** -8)
    for a, b in zip(grads, want_grads):
        assert float((a.double() - b.double()).norm()) <= 16 * 2.0 ** -8 * float(b.double().norm())


def test_pages_are_taken_and_given_back():
    cache = PagedCache(1, 6, 8, 1, 8, sequences=2, most_tokens=400, dtype=torch.float32, device="cpu", window=10, sinks=3)
    cache.make_room([20, 1])
    assert cache.free_pages == 2 and cache.lengths.tolist() == [20, 1]
    assert (cache.tables[0, :3] >= 0).all() and (cache.tables[0, 3:] == -1).all()
    for _ in range(370):                               # a window's pages and the first tokens' page, however long the recording
        cache.make_room([1, 0])
        assert cache.free_pages >= 1
    held = (cache.tables[0] >= 0).nonzero().flatten().tolist()
    assert held[0] == 0 and held[1:] == [47, 48] and cache.lengths.tolist() == [390, 1]
    assert len(set(cache.tables[cache.tables >= 0].tolist())) == 4
    with pytest.raises(RuntimeError, match="full"):
        cache.make_room([0, 40])
    assert cache.lengths.tolist() == [390, 1] and cache.free_pages == 2       # nothing was taken
    with pytest.raises(ValueError, match="do not fit"):
        cache.make_room([11, 0])
    with pytest.raises(ValueError, match="sequences"):
        cache.make_room([1])
    with pytest.raises(ValueError, match="do not fit"):
        cache.make_room([-1, 0])
    cache.reset(0)
    assert cache.free_pages == 5 and cache.lengths.tolist() == [0, 1]
    cache.make_room([0, 39])
    with pytest.raises(ValueError, match="multiple of 8"):
        PagedCache(1, 6, 12, 1, 8, 2, 400, torch.float32, "cpu")
    with pytest.raises(ValueError, match="new frames"):
        _model(torch.float32, "cpu").extend(torch.randn(2, 24), torch.tensor([1, 2]), cache, [1, 2])
    with pytest.raises(ValueError, match="share"):
        _model(torch.float32, "cpu", kv_heads=3)
