"""The token operators in 64 bits, written from their definitions: what the tests compare with."""
import math

import torch

# Largest relative error of one rounding to the type.
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def within(got, want, dtype, computed=0.0):
    """One rounding to ``dtype`` of a value that was computed in fp32 with an absolute error of ``computed`` (a number, or
    one for each value); infinities and NaN in the same places."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape
    finite = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~finite & ~want.isnan()], want[~finite & ~want.isnan()])
    bound = UNIT[dtype] * want.abs() + computed + 2.0 ** -25     # the last term: half a step of half's subnormals
    over = ((got - want).abs() - bound)[finite]
    assert over.numel() == 0 or float(over.max()) <= 0.0, float(over.max())


def embed(ids, table, scale):
    out = torch.zeros(*ids.shape, table.shape[1], dtype=torch.float64, device=table.device)
    valid = (ids >= 0) & (ids < table.shape[0])
    out[valid] = table.double()[ids[valid].long()] * scale
    return out


def embed_grad(ids, d_out, vocab, scale):
    """The gradient and, for bounds, the sum of its terms' absolute values."""
    valid = (ids >= 0) & (ids < vocab)
    at, rows = ids[valid].long(), d_out[valid].double() * scale
    zero = torch.zeros(vocab, d_out.shape[-1], dtype=torch.float64, device=d_out.device)
    return zero.index_add(0, at, rows), zero.index_add(0, at, rows.abs())


def recurrence(zgo, state, resets):
    """y, the last state, and h before and after each step (T, B, D)."""
    z, g, o = (x.transpose(0, 1) for x in zgo.double().unbind(2))
    f, s = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(-o))
    h = torch.zeros_like(z[0]) if state is None else state.double()
    before, after = [], []
    for t in range(z.shape[0]):
        if resets is not None:
            h = torch.where(resets[:, t].unsqueeze(1), torch.zeros_like(h), h)
        before.append(h)
        h = f[t] * h + (1 - f[t]) * z[t]
        after.append(h)
    before, after = torch.stack(before), torch.stack(after)
    return (s * after).transpose(0, 1), h, before, after


def recurrence_grad(zgo, state, resets, dy, d_state):
    z, g, o = (x.transpose(0, 1) for x in zgo.double().unbind(2))
    f, s = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(-o))
    _, _, before, after = recurrence(zgo, state, resets)
    dy = dy.double().transpose(0, 1)
    carry = torch.zeros_like(z[0]) if d_state is None else d_state.double()
    grads = []
    for t in range(z.shape[0] - 1, -1, -1):
        dh = carry + dy[t] * s[t]
        grads.append(torch.stack([dh * (1 - f[t]), dh * (before[t] - z[t]) * f[t] * (1 - f[t]),
                                  dy[t] * after[t] * s[t] * (1 - s[t])], 1))
        carry = dh * f[t]
        if resets is not None:
            carry = torch.where(resets[:, t].unsqueeze(1), torch.zeros_like(carry), carry)
    return torch.stack(grads[::-1], 1), carry


def gate(g, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def mlp(x, w_in, w_out, b_in, b_out, act, residual, dy):
    """Every output, and for bounds the sum of the absolute values of the terms of each product."""
    x, w_in, w_out, dy = (t.double() for t in (x, w_in, w_out, dy))
    vg = x @ w_in.t() + (0 if b_in is None else b_in.double())
    v, g = vg.chunk(2, 1)
    a, da = gate(g, act)
    h = v * a
    y = h @ w_out.t() + (0 if b_out is None else b_out.double()) + (0 if residual is None else residual.double())
    dh = dy @ w_out
    dvg = torch.cat([dh * a, dh * v * da], 1)
    out = {"y": y, "x": dvg @ w_in, "w_in": dvg.t() @ x, "w_out": dy.t() @ h, "b_in": dvg.sum(0), "b_out": dy.sum(0),
           "residual": dy}
    size = {"y": h.abs() @ w_out.abs().t(), "x": dvg.abs() @ w_in.abs(), "w_in": dvg.abs().t() @ x.abs(),
            "w_out": dy.abs().t() @ h.abs(), "b_in": dvg.abs().sum(0), "b_out": dy.abs().sum(0), "residual": 0 * dy}
    return out, size


def logprobs(logits, targets, temperature):
    x = logits.double() / temperature
    nothing = (x == -math.inf).all(-1)
    top = x.amax(-1, keepdim=True).masked_fill(nothing.unsqueeze(-1), 0.0)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True).masked_fill(nothing.unsqueeze(-1), 1.0)
    logp = (x - top - torch.log(total))
    p = e / total
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    valid = (targets >= 0) & (targets < logits.shape[-1])
    at = targets.long().clamp(0, logits.shape[-1] - 1).unsqueeze(-1)
    return torch.where(valid, logp.gather(-1, at).squeeze(-1), 0.0), entropy, logp, p


def logprobs_grad(logits, targets, temperature, d_logprob, d_entropy):
    lp, entropy, logp, p = logprobs(logits, targets, temperature)
    valid = (targets >= 0) & (targets < logits.shape[-1]) & (p.sum(-1) != 0)
    dl = torch.where(valid, d_logprob.double(), 0.0).unsqueeze(-1)
    dx = -p * dl - d_entropy.double().unsqueeze(-1) * torch.where(p == 0, torch.zeros_like(p), p * (logp + entropy.unsqueeze(-1)))
    at = targets.long().clamp(0, logits.shape[-1] - 1).unsqueeze(-1)
    return dx.scatter_add(-1, at, dl) / temperature


def alternatives(logits, top):
    """The first ``top`` by (value falling, index rising), a NaN as -inf."""
    x = logits.double()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    return x.sort(dim=-1, descending=True, stable=True)[1][..., :top]
