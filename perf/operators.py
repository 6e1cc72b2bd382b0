"""Operators of token models that are measured on their own: what an action model that reads its earlier actions trains
on and answers with.

* ``embed``     the vectors of token ids from a table, scaled, and the table's gradient (``ops.embed_tokens``);
* ``recur``     a gated linear recurrence over a sequence with its backward pass, and one step of it
                (``ops.gated_recurrence``);
* ``mlp``       a gated feed-forward block with its backward pass (``ops.gated_mlp``);
* ``logprobs``  log probabilities of given tokens, the entropy and the most likely alternatives
                (``ops.token_logprobs``), with the gradient of the first two.

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One action for each of eight terminals: the choice, how sure the model is, and the five most likely actions.
        {"name": "logprobs_act", "kind": "logprobs", "rows": 8, "vocab": 4096, "dtype": "bf16", "top": 5, "temperature": 1.0,
         "masked": 0.0, "ignored": 0.0, "grad": False},
        # A batch of the headline configuration (8 sequences of 1024 frames, 4096 actions) under an objective of log
        # probabilities and entropy.
        {"name": "logprobs_train", "kind": "logprobs", "rows": 8192, "vocab": 4096, "dtype": "bf16", "top": 0,
         "temperature": 1.0, "masked": 0.0, "ignored": 0.02, "grad": True},
        # Scoring of recorded text with a large vocabulary of no round size, with masked tokens and alternatives.
        {"name": "logprobs_score", "kind": "logprobs", "rows": 1001, "vocab": 100003, "dtype": "fp32", "top": 20,
         "temperature": 0.7, "masked": 0.3, "ignored": 0.1, "grad": True},
        # The earlier actions of a batch of the headline configuration: a table of 4096 rows, a few actions very common.
        {"name": "embed_train", "kind": "embed", "tokens": 8192, "vocab": 4096, "dim": 1024, "table": "bf16", "out": "bf16",
         "skew": 1.1, "invalid": 0.0, "grad": True},
        # A large vocabulary with fp32 master rows and 16-bit activations, as the cell embedding keeps its tables.
        {"name": "embed_text", "kind": "embed", "tokens": 65536, "vocab": 100003, "dim": 2048, "table": "fp32", "out": "bf16",
         "skew": 1.0, "invalid": 0.01, "grad": True},
        # One step for each of eight terminals from a carried state.
        {"name": "recur_act", "kind": "recur", "batch": 8, "steps": 1, "dim": 1024, "dtype": "bf16", "state": True,
         "resets": 0.0, "time_major": False, "grad": False},
        # A batch of the headline configuration with several recordings in a row.
        {"name": "recur_train", "kind": "recur", "batch": 8, "steps": 1024, "dim": 1024, "dtype": "bf16", "state": False,
         "resets": 0.004, "time_major": False, "grad": True},
        # One long recording, time-major as the LSTM takes its sequences.
        {"name": "recur_long", "kind": "recur", "batch": 1, "steps": 30011, "dim": 2048, "dtype": "fp16", "state": True,
         "resets": 0.0, "time_major": True, "grad": True},
        # One step for each of eight terminals: the weights are read for a few rows.
        {"name": "mlp_act", "kind": "mlp", "rows": 8, "width": 1024, "inner": 4096, "dtype": "bf16", "act": "gelu",
         "bias": True, "residual": True, "grad": False},
        # A batch of the headline configuration.
        {"name": "mlp_train", "kind": "mlp", "rows": 8192, "width": 1024, "inner": 4096, "dtype": "bf16", "act": "gelu",
         "bias": True, "residual": True, "grad": True},
        # A batch of the one-billion-parameter configuration.
        {"name": "mlp_train_2048", "kind": "mlp", "rows": 8192, "width": 2048, "inner": 8192, "dtype": "fp16", "act": "silu",
         "bias": False, "residual": False, "grad": True},
        # A short odd batch through sizes that are no multiples of a tile.
        {"name": "mlp_ragged", "kind": "mlp", "rows": 1001, "width": 1000, "inner": 2730, "dtype": "bf16", "act": "silu",
         "bias": False, "residual": True, "grad": True},
    ]


# ---------------------------------------------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size as models have them: mostly a multiple of 64 (or 8, when small), sometimes any number."""
    n = _log_int(rng, lo, hi)
    if rng.random() < 0.7:
        unit = 64 if n >= 128 else 8
        n = max(lo, n // unit * unit)
    return n


def draw(rng):
    kind = rng.choice(["logprobs", "embed", "recur", "mlp"])
    if kind == "logprobs":
        vocab = _log_int(rng, 17, 262144)
        rows = _log_int(rng, 1, max(1, min(16384, 100_000_000 // vocab)))
        return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "top": min(vocab, rng.choice([0, 1, 5, 20, 32])), "temperature": rng.choice([1.0, 0.7]),
                "masked": rng.choice([0.0, 0.3]), "ignored": rng.choice([0.0, 0.05]), "grad": rng.random() < 0.6}
    if kind == "embed":
        dim = _size(rng, 8, 4096)
        table, out = rng.choice([("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "bf16"), ("fp32", "fp32")])
        return {"kind": kind, "tokens": _log_int(rng, 1, max(1, min(131072, 134_000_000 // dim))),
                "vocab": _log_int(rng, 16, max(16, min(262144, 204_000_000 // dim))), "dim": dim, "table": table, "out": out,
                "skew": rng.choice([0.0, 1.0, 1.3]), "invalid": rng.choice([0.0, 0.01]), "grad": rng.random() < 0.7}
    if kind == "recur":
        dim = _size(rng, 8, 4096)
        batch = _log_int(rng, 1, 64)
        return {"kind": kind, "batch": batch, "steps": _log_int(rng, 1, max(1, min(65536, 61_000_000 // (dim * batch)))), "dim": dim,
                "dtype": rng.choice(["bf16", "fp16"]), "state": rng.random() < 0.5, "resets": rng.choice([0.0, 0.005]),
                "time_major": rng.random() < 0.5, "grad": rng.random() < 0.7}
    return {"kind": kind, "rows": _log_int(rng, 1, 8192), "width": _size(rng, 64, 2048), "inner": _size(rng, 64, 8192),
            "dtype": rng.choice(["bf16", "fp16"]), "act": rng.choice(["gelu", "silu"]), "bias": rng.random() < 0.5,
            "residual": rng.random() < 0.5, "grad": rng.random() < 0.6}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _frequencies(vocab, skew):
    """How often each id comes up: by its rank to the power ``-skew``."""
    p = torch.arange(1, vocab + 1, dtype=torch.float64).pow(-skew)
    return p / p.sum()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype="fp32"):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(DTYPES[dtype])

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    st = {"case": case}
    kind = case["kind"]
    if kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # The head's width is padded to a multiple of 8 columns; the logits are the view without the padding.
        full = normal(rows, (vocab + 7) // 8 * 8, scale=3.0, dtype=case["dtype"])
        if case["masked"]:
            full.masked_fill_(uniform(*full.shape) < case["masked"], -math.inf)
            full[rows // 2] = -math.inf              # a row in which nothing is allowed
        st["logits"] = full[:, :vocab].requires_grad_(case["grad"])
        st["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        if case["ignored"]:
            st["targets"].masked_fill_(uniform(rows) < case["ignored"], -1)
        st["d_logprob"], st["d_entropy"] = normal(rows), normal(rows, scale=0.1)
    elif kind == "embed":
        n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        st["table"] = normal(vocab, dim, dtype=case["table"]).requires_grad_(case["grad"])
        edges = _frequencies(vocab, case["skew"]).cumsum(0).float().cuda()
        ranks = torch.searchsorted(edges, uniform(n)).clamp_(max=vocab - 1)
        st["ids"] = torch.randperm(vocab, generator=gen, device="cuda")[ranks]
        if case["invalid"]:
            st["ids"].masked_fill_(uniform(n) < case["invalid"], -1)
        st["d_out"] = normal(n, dim, dtype=case["out"])
        st["scale"] = math.sqrt(dim)
    elif kind == "recur":
        b, t, d = case["batch"], case["steps"], case["dim"]

        def sequence(*inner):
            if case["time_major"]:
                return normal(t, b, *inner, dtype=case["dtype"]).transpose(0, 1)
            return normal(b, t, *inner, dtype=case["dtype"])

        zgo = sequence(3, d)
        zgo[:, :, 1] += 3.0                          # gates that remember some twenty steps, with a bias of the projection
        st["zgo"] = zgo.requires_grad_(case["grad"])
        st["state"] = normal(b, d).requires_grad_(case["grad"]) if case["state"] else None
        st["resets"] = uniform(b, t) < case["resets"] if case["resets"] else None
        st["d_y"], st["d_state"] = sequence(d), normal(b, d)
    else:
        rows, width, inner, dt = case["rows"], case["width"], case["inner"], case["dtype"]
        st["x"] = normal(rows, width, dtype=dt)
        st["w_in"] = normal(2 * inner, width, scale=width ** -0.5, dtype=dt)
        st["w_out"] = normal(width, inner, scale=inner ** -0.5, dtype=dt)
        st["b_in"] = normal(2 * inner, scale=0.1, dtype=dt) if case["bias"] else None
        st["b_out"] = normal(width, scale=0.1, dtype=dt) if case["bias"] else None
        st["residual"] = normal(rows, width, dtype=dt) if case["residual"] else None
        st["d_y"] = normal(rows, width, scale=0.1, dtype=dt)
        for name in _MLP_INPUTS:
            if case["grad"] and st[name] is not None:
                st[name].requires_grad_()
    return st


_MLP_INPUTS = ("x", "w_in", "w_out", "b_in", "b_out", "residual")


def run(st):
    return globals()[("_own_" if own else "_plain_") + st["case"]["kind"]](st)


# ---------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------
def _own_logprobs(st):
    from fbamtrain_b200 import ops
    case = st["case"]
    r = ops.token_logprobs(st["logits"], st["targets"], top=case["top"], temperature=case["temperature"])
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if case["top"]:
        out.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
    if case["grad"]:
        out["d_logits"], = torch.autograd.grad((r.logprob, r.entropy), (st["logits"],), (st["d_logprob"], st["d_entropy"]))
    return out


def _own_embed(st):
    from fbamtrain_b200 import ops
    out = {"out": ops.embed_tokens(st["ids"], st["table"], st["scale"], DTYPES[st["case"]["out"]])}
    if st["case"]["grad"]:
        out["d_table"], = torch.autograd.grad((out["out"],), (st["table"],), (st["d_out"],))
    return out


def _own_recur(st):
    from fbamtrain_b200 import ops
    y, state = ops.gated_recurrence(st["zgo"], st["state"], st["resets"])
    out = {"y": y, "state": state}
    if st["case"]["grad"]:
        into = (st["zgo"],) if st["state"] is None else (st["zgo"], st["state"])
        grads = torch.autograd.grad((y, state), into, (st["d_y"], st["d_state"]))
        out.update(zip(("d_zgo", "d_state"), grads))
    return out


def _own_mlp(st):
    from fbamtrain_b200 import ops
    y = ops.gated_mlp(st["x"], st["w_in"], st["w_out"], st["b_in"], st["b_out"], st["case"]["act"], st["residual"])
    out = {"y": y}
    if st["case"]["grad"]:
        names = [n for n in _MLP_INPUTS if st[n] is not None]
        grads = torch.autograd.grad((y,), [st[n] for n in names], (st["d_y"],))
        out.update(("d_" + n, g) for n, g in zip(names, grads))
    return out


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def _plain_logprobs(st):
    """With x = logits / temperature: log p = x - log sum exp x, entropy = -sum p log p; a row in which nothing is
    allowed has entropy 0, log probabilities of -inf and no gradient; a target outside the vocabulary counts 0."""
    case = st["case"]
    x = st["logits"].float() / case["temperature"]
    top = x.amax(1, keepdim=True)
    some = top > -math.inf
    e = (x - top.where(some, torch.zeros_like(top))).exp()
    total = e.sum(1, keepdim=True)
    logp = (x - top - total.log()).masked_fill(~some, -math.inf)
    p = (e / total).masked_fill(~some, 0.0)
    plogp = (p * logp).masked_fill(p == 0, 0.0)
    entropy = -plogp.sum(1)
    valid = (st["targets"] >= 0) & (st["targets"] < case["vocab"])
    at = st["targets"].clamp(0, case["vocab"] - 1).unsqueeze(1)
    logprob = logp.gather(1, at).squeeze(1).masked_fill(~valid, 0.0)
    out = {"logprob": logprob, "entropy": entropy}
    if case["top"]:
        ids = st["logits"].float().sort(dim=1, descending=True, stable=True)[1][:, :case["top"]]
        out.update(top_logprobs=logp.gather(1, ids), top_ids=ids)
    if case["grad"]:
        dl = (st["d_logprob"] * valid).unsqueeze(1)
        dx = -p * dl - st["d_entropy"].unsqueeze(1) * (plogp + p * entropy.unsqueeze(1))
        dx.scatter_add_(1, at, dl * some)
        out["d_logits"] = (dx / case["temperature"]).to(st["logits"].dtype)
    return out


@torch.no_grad()
def _plain_embed(st):
    case, ids, table = st["case"], st["ids"], st["table"]
    valid = ((ids >= 0) & (ids < case["vocab"])).unsqueeze(1)
    at = ids.clamp(0, case["vocab"] - 1)
    out = {"out": (table[at].float() * st["scale"] * valid).to(DTYPES[case["out"]])}
    if case["grad"]:
        order = at.sort(stable=True)[1]              # equal ids one after the other, so that their sums have one order
        rows = (st["d_out"].float() * valid)[order]
        total = torch.zeros(case["vocab"], case["dim"], device="cuda")
        total.index_put_((at[order],), rows, accumulate=True)
        out["d_table"] = (total * st["scale"]).to(table.dtype)
    return out


def _scan(a, b):
    """``h[t] = a[t] h[t - 1] + b[t]`` along dimension 1 by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


@torch.no_grad()
def _plain_recur(st):
    """``f = sigmoid(g)``, ``h[t] = f h[t - 1] + (1 - f) z``, ``y = sigmoid(o) h``; a reset drops ``h[t - 1]``."""
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    z, g, o = st["zgo"].float().unbind(2)
    f, f1, s = g.sigmoid(), (-g).sigmoid(), o.sigmoid()
    keep = f if st["resets"] is None else f.masked_fill(st["resets"].unsqueeze(2), 0.0)
    h0 = torch.zeros_like(z[:, 0]) if st["state"] is None else st["state"]
    b = f1 * z
    b[:, 0] += keep[:, 0] * h0
    h = _scan(keep, b)
    out = {"y": (s * h).to(dt), "state": h[:, -1].clone()}
    if case["grad"]:
        dy = st["d_y"].float()
        b = dy * s
        b[:, -1] += st["d_state"]
        after = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
        dh = _scan(after.flip(1), b.flip(1)).flip(1)
        before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
        if st["resets"] is not None:
            before = before.masked_fill(st["resets"].unsqueeze(2), 0.0)
        out["d_zgo"] = torch.stack([dh * f1, dh * (before - z) * f * f1, dy * h * s * (1 - s)], 2).to(dt)
        if st["state"] is not None:
            out["d_state"] = keep[:, 0] * dh[:, 0]
    return out


def _act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        s = g.sigmoid()
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _mlp_formula(st):
    """``y = (v * act(g)) w_out^T + b_out + residual`` with ``(v, g) = x w_in^T + b_in``, and its gradients."""
    x, w_in, w_out, dy = (st[n].float() for n in ("x", "w_in", "w_out", "d_y"))
    vg = x @ w_in.t()
    if st["b_in"] is not None:
        vg = vg + st["b_in"].float()
    v, g = vg.chunk(2, dim=1)
    a, da = _act(g, st["case"]["act"])
    h = v * a
    y = h @ w_out.t()
    if st["b_out"] is not None:
        y = y + st["b_out"].float()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    out = {"y": y}
    if st["case"]["grad"]:
        dh = dy @ w_out
        dvg = torch.cat([dh * a, dh * v * da], 1)
        out.update(d_x=dvg @ w_in, d_w_in=dvg.t() @ x, d_w_out=dy.t() @ h)
        if st["b_in"] is not None:
            out.update(d_b_in=dvg.sum(0), d_b_out=dy.sum(0))
        if st["residual"] is not None:
            out["d_residual"] = dy
    return out


@torch.no_grad()
def _plain_mlp(st):
    dt = DTYPES[st["case"]["dtype"]]
    return {k: v.to(dt) for k, v in _mlp_formula(st).items()}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    kind, g = case["kind"], case["grad"]
    if kind == "logprobs":
        n, e = case["rows"] * case["vocab"], SIZE[case["dtype"]]
        per_row = 8 + 8 + 12 * case["top"] + (8 if g else 0)
        return {"bytes": n * e * (2 if g else 1) + case["rows"] * per_row, "flops": n * (12 if g else 5)}
    if kind == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        seen = float((1 - (1 - _frequencies(v, case["skew"])).pow(n)).sum())
        there = n * (1 - case["invalid"])
        size = n * 8 + seen * d * SIZE[case["table"]] + n * d * SIZE[case["out"]]
        if g:
            size += there * d * SIZE[case["out"]] + v * d * SIZE[case["table"]]
        return {"bytes": int(size), "flops": int(n * d * (2 if g else 1))}
    if kind == "recur":
        n = case["batch"] * case["steps"] * case["dim"]
        states = case["batch"] * case["dim"] * 4 * (1 + case["state"]) * (2 if g else 1)
        flags = case["batch"] * case["steps"] if case["resets"] else 0
        return {"bytes": n * 2 * (8 if g else 4) + states + flags, "flops": n * (40 if g else 14)}
    r, w, f = case["rows"], case["width"], case["inner"]
    ends = 2 + case["residual"]
    size = 2 * (ends * r * w + 3 * w * f + (2 * f + w) * case["bias"])
    if g:
        size += 2 * (2 * r * w + 3 * w * f + (2 * f + w) * case["bias"])
    return {"bytes": size, "flops": r * w * f * (18 if g else 6)}


# ---------------------------------------------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](st, case)


def _exact_logprobs(st, case):
    x = st["logits"].double() / case["temperature"]
    nothing = (x == -math.inf).all(1)
    logp = x.masked_fill(nothing.unsqueeze(1), 0.0).log_softmax(1)
    logp[nothing] = -math.inf
    p = logp.exp()
    finite = logp.masked_fill(logp == -math.inf, 0.0)
    entropy = -(p * finite).sum(1)
    rows = torch.arange(case["rows"], device="cuda")
    valid = st["targets"] >= 0
    t = st["targets"].clamp(min=0)
    out = {"logprob": torch.where(valid, logp[rows, t], 0.0), "entropy": entropy}
    if case["top"]:
        out.update(top_logprobs=logp.topk(case["top"], dim=1)[0], top_ids=None)
    if case["grad"]:
        dl = torch.where(valid & ~nothing, st["d_logprob"].double(), 0.0)
        dx = -p * (dl.unsqueeze(1) + st["d_entropy"].double().unsqueeze(1) * (finite + entropy.unsqueeze(1)))
        dx[rows, t] += dl
        out["d_logits"] = dx / case["temperature"]
    return out


def _exact_embed(st, case):
    ids, scale = st["ids"], st["scale"]
    valid = ids >= 0
    rows = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
    rows[valid] = st["table"][ids[valid]].double() * scale
    out = {"out": rows}
    if case["grad"]:
        grad = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        out["d_table"] = grad.index_add_(0, ids[valid], st["d_out"][valid].double() * scale)
    return out


def _exact_recur(st, case):
    b, t, d = case["batch"], case["steps"], case["dim"]
    z, g, o = (st["zgo"][:, :, k].transpose(0, 1).double() for k in range(3))
    f, s = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(-o))
    go = torch.ones(t, b, 1, dtype=torch.float64, device="cuda")
    if st["resets"] is not None:
        go = (~st["resets"]).t().unsqueeze(2).double()
    h = torch.zeros(b, d, dtype=torch.float64, device="cuda") if st["state"] is None else st["state"].double()
    before, after = torch.empty_like(z), torch.empty_like(z)
    into = (1 - f) * z
    kept = f * go
    for k in range(t):
        before[k] = h
        h = torch.addcmul(into[k], kept[k], h)
        after[k] = h
    out = {"y": (s * after).transpose(0, 1), "state": h}
    if case["grad"]:
        dy = st["d_y"].transpose(0, 1).double()
        out_grad = dy * s
        dh = torch.empty_like(z)
        carry = st["d_state"].double()
        for k in range(t - 1, -1, -1):
            dh[k] = carry + out_grad[k]
            carry = dh[k] * kept[k]
        dz, do = dh * (1 - f), dy * after * s * (1 - s)
        dg = dh * (before * go - z) * f * (1 - f)
        out["d_zgo"] = torch.stack([dz, dg, do], 2).transpose(0, 1)
        if st["state"] is not None:
            out["d_state"] = carry
    return out


def _exact_mlp(st, case):
    names = [n for n in _MLP_INPUTS if st[n] is not None]
    with torch.enable_grad():
        at = {n: st[n].detach().double().requires_grad_() for n in names}
        v, g = torch.nn.functional.linear(at["x"], at["w_in"], at.get("b_in")).split(case["inner"], dim=1)
        gate = torch.nn.functional.silu(g) if case["act"] == "silu" else torch.nn.functional.gelu(g)
        y = torch.nn.functional.linear(v * gate, at["w_out"], at.get("b_out"))
        if "residual" in at:
            y = y + at["residual"]
    out = {"y": y.detach()}
    if case["grad"]:
        grads = torch.autograd.grad((y,), [at[n] for n in names], (st["d_y"].double(),))
        out.update(("d_" + n, w) for n, w in zip(names, grads))
    return out
