"""The token operators on the CPU: their plain definitions against 64 bits, and what they refuse."""
import math

import pytest
import torch

import token_oracle as oracle
from fbamtrain_b200 import ops

F32 = torch.float32


def test_definitions_match_the_oracle():
    torch.manual_seed(0)
    ids = torch.tensor([[0, 3, -1], [5, 3, 7]])
    table = torch.randn(6, 4).requires_grad_()
    out = ops.embed_tokens(ids, table, 0.5)
    oracle.within(out.detach(), oracle.embed(ids, table.detach(), 0.5), F32, 1e-6)
    d = torch.randn(2, 3, 4)
    grad, = torch.autograd.grad((out,), (table,), (d,))
    oracle.within(grad, oracle.embed_grad(ids, d, 6, 0.5)[0], F32, 1e-6)

    zgo, state = torch.randn(2, 9, 3, 5).requires_grad_(), torch.randn(2, 5).requires_grad_()
    resets = torch.rand(2, 9) < 0.2
    y, last = ops.gated_recurrence(zgo, state, resets)
    want_y, want_last, _, _ = oracle.recurrence(zgo.detach(), state.detach(), resets)
    oracle.within(y.detach(), want_y, F32, 1e-5)
    oracle.within(last.detach(), want_last, F32, 1e-5)
    dy, d_last = torch.randn(2, 9, 5), torch.randn(2, 5)
    grads = torch.autograd.grad((y, last), (zgo, state), (dy, d_last))
    for got, want in zip(grads, oracle.recurrence_grad(zgo.detach(), state.detach(), resets, dy, d_last)):
        oracle.within(got, want, F32, 1e-5)

    x, w_in, w_out = torch.randn(4, 6), torch.randn(10, 6), torch.randn(3, 5)
    b_in, b_out, res, dy = torch.randn(10), torch.randn(3), torch.randn(4, 3), torch.randn(4, 3)
    named = {"x": x, "w_in": w_in, "w_out": w_out, "b_in": b_in, "b_out": b_out, "residual": res}
    for v in named.values():
        v.requires_grad_()
    for act in ("gelu", "silu"):
        y = ops.gated_mlp(x, w_in, w_out, b_in, b_out, act, res)
        grads = torch.autograd.grad((y,), list(named.values()), (dy,))
        with torch.no_grad():
            want, size = oracle.mlp(x, w_in, w_out, b_in, b_out, act, res, dy)
        for name, got in [("y", y.detach())] + list(zip(named, grads)):
            oracle.within(got, want[name], F32, 1e-4)

    logits = torch.randn(5, 11)
    logits[1, 3:] = -math.inf
    logits[2] = -math.inf
    logits.requires_grad_()
    t = torch.tensor([0, 5, 1, -1, 10])
    r = ops.token_logprobs(logits, t, 4, 0.7)
    lp, entropy, logp, _ = oracle.logprobs(logits.detach(), t, 0.7)
    oracle.within(r.logprob.detach(), lp, F32, 1e-5)
    oracle.within(r.entropy.detach(), entropy, F32, 1e-5)
    assert torch.equal(r.top_ids, oracle.alternatives(logits.detach(), 4))
    oracle.within(r.top_logprobs, logp.gather(1, r.top_ids), F32, 1e-5)
    dl, dh = torch.randn(5), torch.randn(5)
    grad, = torch.autograd.grad((r.logprob, r.entropy), (logits,), (dl, dh))
    oracle.within(grad, oracle.logprobs_grad(logits.detach(), t, 0.7, dl, dh), F32, 1e-5)


def test_oracle_gradients_are_the_forms_derivatives():
    """The formulas against central differences in 64 bits."""
    torch.manual_seed(1)
    h = 1e-6

    def check(f, grad, *at):
        for x, g in zip(at, grad):
            v = torch.randn_like(x)
            diff = (f(*[a + h * v if a is x else a for a in at]) - f(*[a - h * v if a is x else a for a in at])) / (2 * h)
            assert float((g * v).sum()) == pytest.approx(float(diff), rel=1e-6, abs=1e-7)

    zgo, state = torch.randn(2, 6, 3, 4).double(), torch.randn(2, 4).double()
    resets, dy, dl = torch.rand(2, 6) < 0.3, torch.randn(2, 6, 4).double(), torch.randn(2, 4).double()

    def rec(z, s):
        y, last, _, _ = oracle.recurrence(z, s, resets)
        return (y * dy).sum() + (last * dl).sum()

    check(rec, oracle.recurrence_grad(zgo, state, resets, dy, dl), zgo, state)
    logits, t = torch.randn(3, 9).double(), torch.tensor([1, -1, 8])
    a, b = torch.randn(3).double(), torch.randn(3).double()

    def lps(x):
        lp, entropy, _, _ = oracle.logprobs(x, t, 0.6)
        return (lp * a + entropy * b).sum()

    check(lps, (oracle.logprobs_grad(logits, t, 0.6, a, b),), logits)
    x, w1, w2, d = torch.randn(3, 4).double(), torch.randn(10, 4).double(), torch.randn(2, 5).double(), torch.randn(3, 2).double()
    for act in ("gelu", "silu"):
        g = oracle.mlp(x, w1, w2, None, None, act, None, d)[0]
        check(lambda *a: (oracle.mlp(*a, None, None, act, None, d)[0]["y"] * d).sum(), (g["x"], g["w_in"], g["w_out"]), x, w1, w2)


def test_refusals():
    table, ids = torch.randn(4, 8), torch.tensor([1, 2])
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.embed_tokens(ids.float(), table)
    with pytest.raises(ValueError, match="rows, width"):
        ops.embed_tokens(ids, table[0])
    with pytest.raises(TypeError, match="own type"):
        ops.embed_tokens(ids, table.to(torch.bfloat16), 1.0, torch.float32)

    zgo = torch.randn(2, 5, 3, 4)
    with pytest.raises(ValueError, match="projections"):
        ops.gated_recurrence(zgo[:, :, :2])
    with pytest.raises(ValueError, match="projections"):
        ops.gated_recurrence(zgo[0])
    with pytest.raises(ValueError, match="state"):
        ops.gated_recurrence(zgo, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="state"):
        ops.gated_recurrence(zgo, torch.zeros(2, 4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="resets"):
        ops.gated_recurrence(zgo, None, torch.zeros(2, 5))
    with pytest.raises(ValueError, match="resets"):
        ops.gated_recurrence(zgo, None, torch.zeros(5, 2, dtype=torch.bool))

    x, w_in, w_out = torch.randn(3, 4), torch.randn(12, 4), torch.randn(5, 6)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_mlp(x, w_in, w_out, act="relu")
    for a, b in ((w_in[:10], w_out), (w_in[:, :3], w_out), (w_in, w_out[:, :5]), (w_in[0], w_out)):
        with pytest.raises(ValueError, match="gated block"):
            ops.gated_mlp(x, a, b)
    with pytest.raises(ValueError, match="b_in"):
        ops.gated_mlp(x, w_in, w_out, torch.zeros(6))
    with pytest.raises(ValueError, match="b_out"):
        ops.gated_mlp(x, w_in, w_out, None, torch.zeros(4))
    with pytest.raises(ValueError, match="residual"):
        ops.gated_mlp(x, w_in, w_out, residual=torch.zeros(3, 4))

    logits, t = torch.randn(3, 6), torch.tensor([0, 1, 2])
    with pytest.raises(ValueError, match="targets"):
        ops.token_logprobs(logits, t[:2])
    with pytest.raises(ValueError, match="targets"):
        ops.token_logprobs(logits, t.float())
    for top in (-1, 7):
        with pytest.raises(ValueError, match="alternatives"):
            ops.token_logprobs(logits, t, top)
    with pytest.raises(ValueError, match="alternatives"):
        ops.token_logprobs(torch.randn(1, 100), None, 33)
    for temperature in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_logprobs(logits, t, 0, temperature)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.token_logprobs(torch.empty(3, 0))
