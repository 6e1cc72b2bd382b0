"""The action model that reads its earlier actions: whole sequences against single steps, and a few training steps."""
import pytest
import torch

from fbamtrain_b200.models import RecurrentDecoder
from fbamtrain_b200.models.init_utils import SeedSequence


def _model(dtype, device):
    return RecurrentDecoder(frame_dim=24, dim=64, layers=2, inner=96, vocab=37, dtype=dtype, seeds=SeedSequence(3)).to(device)


def _batch(dtype, device, b=3, t=21):
    gen = torch.Generator().manual_seed(5)
    frames = torch.randn(b, t, 24, generator=gen).to(dtype).to(device)
    actions = torch.randint(0, 37, (b, t), generator=gen).to(device)
    previous = torch.cat([torch.full_like(actions[:, :1], -1), actions[:, :-1]], 1)
    return frames, previous, actions


def _steps_match_sequence(dtype, device, tolerance):
    model, (frames, previous, actions) = _model(dtype, device), _batch(dtype, device)
    with torch.no_grad():
        whole = model(frames, previous, actions, top=4)
        state = None
        for t in range(frames.shape[1]):
            got, state = model.step(frames[:, t], previous[:, t], state, top=4)
            torch.testing.assert_close(got.entropy, whole.entropy[:, t], rtol=0, atol=tolerance)
            torch.testing.assert_close(got.top_logprobs, whole.top_logprobs[:, t], rtol=0, atol=tolerance)
    assert whole.logprob.shape == actions.shape and whole.top_ids.shape == (*actions.shape, 4)


def _resets_separate_recordings(dtype, device, tolerance):
    """Two recordings in a row with a reset between them are two sequences."""
    model, (frames, previous, actions) = _model(dtype, device), _batch(dtype, device)
    cut = 8
    previous = previous.clone()
    previous[:, cut] = -1
    resets = torch.zeros_like(actions, dtype=torch.bool)
    resets[:, cut] = True
    with torch.no_grad():
        joined = model(frames, previous, actions, resets).logprob
        first = model(frames[:, :cut], previous[:, :cut], actions[:, :cut]).logprob
        second = model(frames[:, cut:], previous[:, cut:], actions[:, cut:]).logprob
    torch.testing.assert_close(joined, torch.cat([first, second], 1), rtol=0, atol=tolerance)


def _learns(dtype, device):
    """Gradient steps on one batch raise the log probability of its actions and reach every parameter."""
    model, (frames, previous, actions) = _model(dtype, device), _batch(dtype, device)
    values = []
    for _ in range(8):
        r = model(frames, previous, actions)
        objective = r.logprob.mean() + 0.01 * r.entropy.mean()
        values.append(float(r.logprob.detach().mean()))
        grads = torch.autograd.grad(objective, list(model.parameters()))
        with torch.no_grad():
            for p, g in zip(model.parameters(), grads):
                assert bool(g.isfinite().all())
                p += (0.5 * g).to(p.dtype)
    assert values[-1] > values[0] + 0.1
    assert all(bool(g.any()) for g in grads)


def test_decoder_cpu():
    _steps_match_sequence(torch.float32, "cpu", 1e-4)
    _resets_separate_recordings(torch.float32, "cpu", 1e-4)
    _learns(torch.float32, "cpu")


# Sequence and steps differ by the order of fp32 sums, which changes roundings of 16-bit activations: some of 8 (11) bits in
# four layers' values of size 1, on logits of size 1.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tolerance", [(torch.bfloat16, 8 * 2.0 ** -8), (torch.float16, 8 * 2.0 ** -11)])
def test_decoder_gpu(dtype, tolerance):
    _steps_match_sequence(dtype, "cuda", tolerance)
    _resets_separate_recordings(dtype, "cuda", tolerance)
    _learns(dtype, "cuda")


@pytest.mark.gpu
def test_decoder_gpu_matches_the_definitions():
    from fbamtrain_b200 import ops
    model, (frames, previous, actions) = _model(torch.bfloat16, "cuda"), _batch(torch.bfloat16, "cuda")
    with torch.no_grad():
        got = model(frames, previous, actions)
        ops.set_backend("torch")
        try:
            want = model(frames, previous, actions)
        finally:
            ops.set_backend("auto")
    torch.testing.assert_close(got.logprob, want.logprob, rtol=0, atol=8 * 2.0 ** -8)
    torch.testing.assert_close(got.entropy, want.entropy, rtol=0, atol=8 * 2.0 ** -8)
