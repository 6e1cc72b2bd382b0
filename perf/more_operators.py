"""Operators of attention models that are measured on their own: what an action model with a bounded or cached memory trains on
and answers with.

* ``rotary``   rotation of query and key heads by their positions, and its gradient (``ops.rotary``);
* ``window``   causal attention over a sliding window and a few first tokens that stay visible, with its backward pass
               (``ops.window_attention_qkv``);
* ``append``   new tokens into a paged cache: queries and keys rotated, keys and values written (``ops.cache_append``);
* ``cache``    attention of new tokens over a paged cache (``ops.cache_attention``).

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits (angles in 64), rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # Queries and keys of a batch of the headline configuration (8 sequences of 1024 frames, 16 heads of 64), with gradient.
        {"name": "rotary_train", "kind": "rotary", "batch": 8, "steps": 1024, "heads": 48, "turned": 32, "dim": 64, "rotated": 64,
         "interleaved": False, "base": 10000.0, "factor": 1.0, "context": 0, "from": 0, "dtype": "bf16", "grad": True},
        # A long recording far from its start: interleaved pairs in a part of each head, frequencies scaled for a long context.
        {"name": "rotary_far", "kind": "rotary", "batch": 1, "steps": 30011, "heads": 24, "turned": 20, "dim": 128, "rotated": 96,
         "interleaved": True, "base": 500000.0, "factor": 8.0, "context": 8192, "from": 1000000, "dtype": "fp16", "grad": True},
        # A batch of the headline configuration that looks back 256 frames.
        {"name": "window_train", "kind": "window", "batch": 8, "steps": 1024, "heads": 16, "kv_heads": 16, "dim": 64, "window": 256,
         "sinks": 4, "padded": False, "dtype": "bf16", "grad": True},
        # One long recording with shared heads: four query heads to a key head, in the width of the billion-parameter configuration.
        {"name": "window_long", "kind": "window", "batch": 1, "steps": 30011, "heads": 16, "kv_heads": 4, "dim": 128,
         "window": 2048, "sinks": 16, "padded": False, "dtype": "bf16", "grad": True},
        # Scoring of a padded batch of recordings of any length, three query heads to a key head.
        {"name": "window_score", "kind": "window", "batch": 6, "steps": 777, "heads": 12, "kv_heads": 4, "dim": 128, "window": 200,
         "sinks": 1, "padded": True, "dtype": "fp16", "grad": False},
        # One new frame for each of eight terminals.
        {"name": "append_act", "kind": "append", "batch": 8, "new": 1, "cached": 1000, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 16, "ragged": False, "interleaved": False, "dtype": "bf16"},
        # Prompts of several users at once.
        {"name": "append_prompt", "kind": "append", "batch": 5, "new": 2100, "cached": 4000, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "ragged": True, "interleaved": True, "dtype": "bf16"},
        # One new frame for each of eight terminals over what they have seen so far.
        {"name": "cache_act", "kind": "cache", "batch": 8, "new": 1, "cached": 1000, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 16, "window": 0, "sinks": 0, "ragged": False, "dtype": "bf16"},
        # Many users with long histories, one token each, eight query heads to a key head in small pages.
        {"name": "cache_serve", "kind": "cache", "batch": 64, "new": 1, "cached": 16384, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 16, "window": 0, "sinks": 0, "ragged": False, "dtype": "bf16"},
        # Prompts in chunks over long histories.
        {"name": "cache_prompt", "kind": "cache", "batch": 2, "new": 4096, "cached": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "sinks": 0, "ragged": False, "dtype": "bf16"},
        # A mixed batch: chunks of any length and single tokens, each over its window and the first tokens.
        {"name": "cache_mixed", "kind": "cache", "batch": 13, "new": 333, "cached": 9001, "heads": 20, "kv_heads": 4, "dim": 64,
         "page": 32, "window": 1500, "sinks": 4, "ragged": True, "dtype": "fp16"},
    ]


# ---------------------------------------------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _groups(rng):
    """Query heads and key heads: up to eight of the one to one of the other."""
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    return kv * rng.choice([g for g in (1, 1, 2, 3, 4, 5, 8) if g * kv <= 32]), kv


def draw(rng):
    kind = rng.choice(["rotary", "window", "append", "cache"])
    dim, dtype = rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    if kind == "rotary":
        heads, batch = rng.randint(1, 48), _log_int(rng, 1, 16)
        steps = _log_int(rng, 1, max(1, min(32768, 90_000_000 // (heads * batch * dim))))
        factor = rng.choice([1.0, 1.0, 4.0, 8.0])
        return {"kind": kind, "batch": batch, "steps": steps, "heads": heads, "turned": rng.randint(1, heads), "dim": dim,
                "rotated": rng.choice([dim, dim, dim // 2, dim // 4, 32]), "interleaved": rng.random() < 0.5,
                "base": rng.choice([10000.0, 500000.0]), "factor": factor, "context": rng.choice([0, 8192]) if factor > 1 else 0,
                "from": rng.choice([0, 0, 8000, 1000000]), "dtype": dtype, "grad": rng.random() < 0.6}
    heads, kv = _groups(rng)
    if kind == "window":
        grad = rng.random() < 0.7
        batch = _log_int(rng, 1, 16)
        steps = _log_int(rng, 1, max(1, min(30000, 60_000_000 // (batch * heads * dim))))
        most = int(1.7e12 / ((14 if grad else 4) * dim * heads * batch * steps))
        window = _log_int(rng, 1, max(1, min(most - 100, 2 * steps)))
        return {"kind": kind, "batch": batch, "steps": steps, "heads": heads, "kv_heads": kv, "dim": dim, "window": window,
                "sinks": rng.choice([0, 0, 1, 4, 100]), "padded": rng.random() < 0.3, "dtype": dtype, "grad": grad}
    batch, page = _log_int(rng, 1, 64), rng.choice([16, 16, 32, 64, 128])
    case = {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv, "dim": dim, "page": page, "dtype": dtype}
    if kind == "append":
        new = _log_int(rng, 1, max(1, min(4096, 30_000_000 // (batch * (heads + 2 * kv) * dim))))
        cached = new + _log_int(rng, 1, max(2, min(16384, 30_000_000 // (batch * kv * dim))))
        return {**case, "new": new, "cached": cached, "ragged": batch > 1 and rng.random() < 0.5, "interleaved": rng.random() < 0.5}
    new = 1 if rng.random() < 0.5 else _log_int(rng, 1, max(1, min(4096, 60_000_000 // (batch * heads * dim))))
    most = min(int(3e12 / (4 * dim * heads * batch * new)), 500_000_000 // (batch * kv * dim), 65536)
    cached = _log_int(rng, new, max(new, most))
    window = rng.choice([0, _log_int(rng, 1, cached)])
    return {**case, "new": new, "cached": cached, "window": window, "sinks": rng.choice([0, 4, 100]) if window else 0,
            "ragged": batch > 1 and new > 1 and rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------
# the batch of a case
# ---------------------------------------------------------------------------------------------------------------
def _new_tokens(case):
    """New tokens of each sequence: all alike, or every third one only a single token and the others fewer and fewer."""
    if not case["ragged"]:
        return [case["new"]] * case["batch"]
    return [1 if b % 3 == 2 else max(1, case["new"] - case["new"] * b // (2 * case["batch"])) for b in range(case["batch"])]


def _cache_lengths(case):
    """Tokens of each sequence, the new ones among them: from the longest down to about a half; a serving batch of single tokens
    has an idle place where there are more than four of them."""
    new = _new_tokens(case)
    out = [max(n, case["cached"] - case["cached"] * b // (2 * case["batch"])) for b, n in enumerate(new)]
    if case["new"] == 1 and case["batch"] > 4:
        out[3] = 0
    return out


def _padded_lengths(case):
    if not case["padded"]:
        return [case["steps"]] * case["batch"]
    return [case["steps"] - case["steps"] * b // case["batch"] for b in range(case["batch"])]


def _visible(first, last, window, sinks):
    """How many pairs of a query and a key it sees there are for the queries ``first <= i < last`` of one sequence."""
    i = torch.arange(max(first, 0), max(last, 0), dtype=torch.int64)
    if not window:
        return int((i + 1).sum())
    near = (i + 1).clamp(max=window)
    return int((near + (i + 1 - near).clamp(max=sinks)).sum())


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dt)

    st = {"case": case}
    kind, d = case["kind"], case["dim"]
    if kind == "rotary":
        b, t, h = case["batch"], case["steps"], case["heads"]
        st["x"] = normal(b, t, h, d).requires_grad_(case["grad"])
        st["positions"] = torch.arange(t, device="cuda") + case["from"] + torch.randint(0, 100, (b, 1), generator=gen, device="cuda")
        st["d_y"] = normal(b, t, h, d)
    elif kind == "window":
        b, t, h, kv = case["batch"], case["steps"], case["heads"], case["kv_heads"]
        st["qkv"] = normal(b, t, h + 2 * kv, d).requires_grad_(case["grad"])
        st["lengths"] = torch.tensor(_padded_lengths(case), dtype=torch.int32, device="cuda") if case["padded"] else None
        st["d_y"] = normal(b, t, h, d)
    else:
        h, kv, page = case["heads"], case["kv_heads"], case["page"]
        new, lengths = _new_tokens(case), _cache_lengths(case)
        n = sum(new)
        per = [(x + page - 1) // page for x in lengths]
        pages = sum(per) + 3
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        tables = torch.full((case["batch"], max(per)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, count in enumerate(per):
            tables[b, :count] = order[at:at + count]
            at += count
        st["k_pages"], st["v_pages"] = normal(pages, page, kv, d), normal(pages, page, kv, d)
        st["tables"] = tables
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        starts = [0]
        for x in new:
            starts.append(starts[-1] + x)
        st["offsets"] = None if case["new"] == 1 else torch.tensor(starts, dtype=torch.int32, device="cuda")
        st["plan"] = (starts, lengths)               # what the program that makes the batch knows of it
        if kind == "append":
            st["qkv"] = normal(n, h + 2 * kv, d)
        else:
            st["q"] = normal(n, h, d)
    if own and kind in ("rotary", "append"):
        _plan(st)
    return st


def _plan(st):
    """The frequencies, which a program makes once."""
    if "frequencies" not in st:
        from fbamtrain_b200 import ops
        c = st["case"]
        st["frequencies"] = ops.rotary_frequencies(c.get("rotated", c["dim"]), base=c.get("base", 10000.0),
                                                   factor=c.get("factor", 1.0), context=c.get("context") or None)
    return st["frequencies"]


def run(st):
    return globals()[("_own_" if own else "_plain_") + st["case"]["kind"]](st)


# ---------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------
def _own_rotary(st):
    from fbamtrain_b200 import ops
    case = st["case"]
    out = {"y": ops.rotary(st["x"], st["positions"], _plan(st), heads=case["turned"], interleaved=case["interleaved"])}
    if case["grad"]:
        out["d_x"], = torch.autograd.grad((out["y"],), (st["x"],), (st["d_y"],))
    return out


def _own_window(st):
    from fbamtrain_b200 import ops
    case = st["case"]
    out = {"y": ops.window_attention_qkv(st["qkv"], case["kv_heads"], case["window"], case["sinks"], st["lengths"])}
    if case["grad"]:
        out["d_qkv"], = torch.autograd.grad((out["y"],), (st["qkv"],), (st["d_y"],))
    return out


def _own_append(st):
    from fbamtrain_b200 import ops
    q = ops.cache_append(st["qkv"], st["k_pages"], st["v_pages"], st["tables"], st["lengths"], st["offsets"], _plan(st),
                         interleaved=st["case"]["interleaved"])
    return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _own_cache(st):
    from fbamtrain_b200 import ops
    case = st["case"]
    return {"y": ops.cache_attention(st["q"], st["k_pages"], st["v_pages"], st["tables"], st["lengths"], st["offsets"],
                                     window=case["window"] or None, sinks=case["sinks"])}


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _angles(positions, rotated, base, factor, context):
    """``cos`` and ``sin`` of each position's angles, and the factor on what is rotated.  A pair turns by
    ``base^(-2 i / rotated)`` a position; scaled, by that over ``factor``, or, with the context that the model was trained on,
    by less of it the more often the pair turned around within that context."""
    i = torch.arange(rotated // 2, dtype=torch.float64, device=positions.device)
    theta = torch.exp(i * (-2.0 / rotated * math.log(base)))
    magnitude = 1.0
    if factor > 1.0:
        kept = torch.zeros_like(theta)
        if context:
            kept = ((context * theta / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
            magnitude = 1.0 + 0.1 * math.log(factor)
        theta = theta * (kept + (1.0 - kept) / factor)
    angle = positions.double().unsqueeze(-1) * theta
    return angle.cos().float(), angle.sin().float(), magnitude


def _turn(x, cos, sin, magnitude, rotated, interleaved):
    """``x`` ``(..., heads, dim)`` in 32 bits, turned by the angles ``(..., rotated / 2)``."""
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    r = x[..., :rotated]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r.chunk(2, dim=-1)
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r * magnitude, x[..., rotated:]], -1)


@torch.no_grad()
def _plain_rotary(st):
    case, n = st["case"], st["case"]["turned"]
    cos, sin, m = _angles(st["positions"], case["rotated"], case["base"], case["factor"], case["context"])

    def turned(x, sin):
        part = _turn(x[:, :, :n].float(), cos, sin, m, case["rotated"], case["interleaved"])
        return torch.cat([part.to(x.dtype), x[:, :, n:]], 2)

    out = {"y": turned(st["x"], sin)}
    if case["grad"]:
        out["d_x"] = turned(st["d_y"], -sin)
    return out


def _mask(i, j, window, sinks):
    """Which keys at positions ``j`` the queries at positions ``i`` see."""
    seen = j <= i.unsqueeze(-1)
    if window:
        seen &= (i.unsqueeze(-1) - j < window) | (j < sinks)
    return seen


def _attend(q, k, v, seen):
    """``softmax(q k^T / sqrt(D)) v`` with its probabilities: ``q`` ``(..., n, D)``, ``k``, ``v`` ``(..., m, D)``; a row that
    sees nothing gives zeros."""
    s = (q @ k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0.0, 1.0)
    return p @ v, p


def _pieces(first, last, window, sinks, size):
    """Queries ``first <= i < last`` in pieces, each with the keys that it needs: two ranges."""
    for lo in range(first, last, size):
        hi = min(last, lo + size)
        k0 = max(0, lo - window + 1) if window else 0
        s1 = min(sinks, k0) if window else 0
        yield lo, hi, s1, k0


@torch.no_grad()
def _plain_window(st):
    case, qkv = st["case"], st["qkv"]
    b, t, h, kv, d = case["batch"], case["steps"], case["heads"], case["kv_heads"], case["dim"]
    g = h // kv
    x = qkv.float().transpose(1, 2)
    q, k, v = x[:, :h].reshape(b * kv, g, t, d), x[:, h:h + kv].reshape(b * kv, 1, t, d), x[:, h + kv:].reshape(b * kv, 1, t, d)
    dy = st["d_y"].float().transpose(1, 2).reshape(b * kv, g, t, d)
    lengths = torch.full((b,), t, device="cuda") if st["lengths"] is None else st["lengths"]
    lengths = lengths.repeat_interleave(kv).view(-1, 1, 1, 1)
    y = torch.zeros_like(q)
    if case["grad"]:
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k[:, 0]), torch.zeros_like(v[:, 0])
    for lo, hi, s1, k0 in _pieces(0, t, case["window"], case["sinks"], max(256, min(1024, case["window"]))):
        i, at = torch.arange(lo, hi, device="cuda"), torch.cat([torch.arange(s1, device="cuda"), torch.arange(k0, hi, device="cuda")])
        seen = _mask(i, at, case["window"], case["sinks"]) & (i.unsqueeze(-1) < lengths)
        kk, vv = k[:, :, at], v[:, :, at]
        o, p = _attend(q[:, :, lo:hi], kk, vv, seen)
        y[:, :, lo:hi] = o
        if case["grad"]:
            up = dy[:, :, lo:hi]
            dp = up @ vv.transpose(2, 3)
            ds = p * (dp - (p * dp).sum(3, keepdim=True)) * d ** -0.5
            dq[:, :, lo:hi] = ds @ kk
            for total, part in ((dk, (ds.transpose(2, 3) @ q[:, :, lo:hi]).sum(1)), (dv, (p.transpose(2, 3) @ up).sum(1))):
                total[:, :s1] += part[:, :s1]
                total[:, k0:hi] += part[:, s1:]
    out = {"y": y.view(b, h, t, d).transpose(1, 2).to(qkv.dtype)}
    if case["grad"]:
        grad = torch.cat([dq.view(b, h, t, d), dk.view(b, kv, t, d), dv.view(b, kv, t, d)], 1)
        out["d_qkv"] = grad.transpose(1, 2).to(qkv.dtype)
    return out


def _sequences(st):
    """Of each sequence with anything in it: its number, its new tokens' rows and its length."""
    starts, lengths = st["plan"]
    return [(b, starts[b], starts[b + 1], x) for b, x in enumerate(lengths) if x > 0]


@torch.no_grad()
def _plain_append(st):
    case, qkv = st["case"], st["qkv"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q = torch.zeros(qkv.shape[0], h, d, dtype=qkv.dtype, device="cuda")
    for b, lo, hi, length in _sequences(st):
        at = torch.arange(length - (hi - lo), length, device="cuda")
        cos, sin, m = _angles(at, d, 10000.0, 1.0, 0)
        turned = _turn(qkv[lo:hi, :h + kv].float(), cos, sin, m, d, case["interleaved"]).to(qkv.dtype)
        q[lo:hi] = turned[:, :h]
        where = st["tables"][b, at // page].long()
        st["k_pages"][where, at % page] = turned[:, h:]
        st["v_pages"][where, at % page] = qkv[lo:hi, h + kv:]
    return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


@torch.no_grad()
def _plain_cache(st):
    case, q = st["case"], st["q"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    y = torch.zeros(q.shape, device="cuda")
    for b, lo, hi, length in _sequences(st):
        used = st["tables"][b, :(length + page - 1) // page].long()
        k, v = (x[used].reshape(-1, kv, d)[:length].float().transpose(0, 1) for x in (st["k_pages"], st["v_pages"]))
        first = length - (hi - lo)
        for p0, p1, s1, k0 in _pieces(first, length, case["window"], case["sinks"], 512):
            at = torch.cat([torch.arange(s1, device="cuda"), torch.arange(k0, p1, device="cuda")])
            part = q[lo + p0 - first:lo + p1 - first].float()
            n, g = part.shape[0], h // kv
            rows = part.view(n, kv, g, d).permute(1, 2, 0, 3).reshape(kv, g * n, d)
            seen = _mask(torch.arange(p0, p1, device="cuda"), at, case["window"], case["sinks"]).repeat(g, 1)
            o, _ = _attend(rows, k[:, at], v[:, at], seen)
            y[lo + p0 - first:lo + p1 - first] = o.view(kv, g, n, d).permute(2, 0, 1, 3).reshape(n, h, d)
    return {"y": y.to(q.dtype)}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    kind, d = case["kind"], case["dim"]
    if kind == "rotary":
        n = case["batch"] * case["steps"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * 2 * n * case["heads"] * d + 8 * n), "flops": passes * n * case["turned"] * case["rotated"] * 3}
    h, kv = case["heads"], case["kv_heads"]
    if kind == "window":
        pairs = sum(_visible(0, x, case["window"], case["sinks"]) for x in _padded_lengths(case))
        rows = sum(_padded_lengths(case))
        size = 2 * d * (rows * (h + 2 * kv) + case["batch"] * case["steps"] * h)
        if case["grad"]:
            size += 2 * d * (rows * h + case["batch"] * case["steps"] * (h + 2 * kv))
        return {"bytes": size, "flops": pairs * h * d * (14 if case["grad"] else 4)}
    n, new, lengths = sum(_new_tokens(case)), _new_tokens(case), _cache_lengths(case)
    if kind == "append":
        there = sum(x for x, length in zip(new, lengths) if length)
        return {"bytes": 2 * d * (there * (h + 2 * kv) * 2 + (n - there) * h), "flops": there * (h + kv) * d * 3}
    window, sinks = case["window"], case["sinks"]
    pairs = sum(_visible(x - y, x, window, sinks) for y, x in zip(new, lengths) if x)
    keys = 0
    for y, x in zip(new, lengths):
        first = max(0, x - y - window + 1) if window else 0
        keys += x - first + min(sinks, first)
    return {"bytes": 2 * d * (2 * n * h + 2 * keys * kv) + 4 * keys // case["page"], "flops": 4 * d * h * pairs}


# ---------------------------------------------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](st, case)


def _exact_turned(x, positions, rotated, base=10000.0, factor=1.0, context=0, interleaved=False, back=False):
    """The pairs as complex numbers, times ``magnitude * e^(i angle)``; ``x`` ``(n, heads, dim)``, ``positions`` ``(n,)``."""
    speed = torch.tensor([base ** (-2.0 * i / rotated) for i in range(rotated // 2)], dtype=torch.float64, device=x.device)
    size = 1.0
    if factor > 1.0 and context:
        share = torch.clamp((context * speed / (2 * math.pi) - 1) / 31, 0, 1)
        speed, size = share * speed + (1 - share) * speed / factor, 0.1 * math.log(factor) + 1
    elif factor > 1.0:
        speed = speed / factor
    angle = torch.outer(positions.double(), -speed if back else speed)
    wheel = torch.polar(torch.full_like(angle, size), angle).unsqueeze(1)
    out = x.double().clone()
    half = rotated // 2
    first = slice(0, rotated, 2) if interleaved else slice(0, half)
    second = slice(1, rotated, 2) if interleaved else slice(half, rotated)
    pair = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * wheel
    out[..., first], out[..., second] = pair.real, pair.imag
    return out


def _exact_rotary(st, case):
    n = case["turned"]
    at = st["positions"].reshape(-1)

    def turned(x, back):
        flat = x.double().flatten(0, 1)
        flat[:, :n] = _exact_turned(flat[:, :n], at, case["rotated"], case["base"], case["factor"], case["context"], case["interleaved"], back)
        return flat.view(x.shape)

    out = {"y": turned(st["x"], False)}
    if case["grad"]:
        out["d_x"] = turned(st["d_y"], True)
    return out


def _exact_rows(q, k, v, first, window, sinks):
    """Attention of one head in 64 bits: queries ``(n, D)`` at positions from ``first`` on, all keys ``(m, D)`` from 0 on."""
    out = []
    for lo in range(0, q.shape[0], 256):
        i = torch.arange(lo, min(lo + 256, q.shape[0]), device="cuda")[:, None] + first
        m = int(first + min(lo + 256, q.shape[0]))
        near = max(0, first + lo - window + 1) if window else 0
        keep = torch.arange(m, device="cuda")
        if near > sinks:
            keep = torch.cat([keep[:sinks], keep[near:]])
        hidden = keep > i
        if window:
            hidden = hidden | ((i - keep >= window) & (keep >= sinks))
        s = torch.einsum("nd,md->nm", q[lo:lo + 256], k[keep]) / math.sqrt(q.shape[1])
        out.append(torch.softmax(s.masked_fill(hidden, -math.inf), dim=1) @ v[keep])
    return torch.cat(out)


def _exact_window(st, case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    x = st["qkv"].detach()
    y = torch.zeros(*x.shape[:2], h, d, dtype=torch.float64, device="cuda")
    grad = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(_padded_lengths(case)):
        for n in range(h):
            c = n // (h // kv)
            three = [x[b, :length, r].double().requires_grad_(case["grad"]) for r in (n, h + c, h + kv + c)]
            with torch.set_grad_enabled(case["grad"]):
                o = _exact_rows(*three, 0, case["window"], case["sinks"])
            y[b, :length, n] = o.detach()
            if case["grad"]:
                got = torch.autograd.grad((o,), three, (st["d_y"][b, :length, n].double(),))
                for r, g in zip((n, h + c, h + kv + c), got):
                    grad[b, :length, r] += g
    return {"y": y, "d_qkv": grad} if case["grad"] else {"y": y}


def _exact_append(st, case):
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    starts, lengths = st["plan"]
    q = torch.zeros(starts[-1], h, d, dtype=torch.float64, device="cuda")
    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    tables = st["tables"].tolist()
    for b, length in enumerate(lengths):
        if not length:
            continue
        rows = st["qkv"][starts[b]:starts[b + 1]]
        first = length - rows.shape[0]
        turned = _exact_turned(rows[:, :h + kv], torch.arange(first, length, device="cuda"), d, interleaved=case["interleaved"])
        q[starts[b]:starts[b + 1]] = turned[:, :h]
        p = first
        while p < length:
            stop = min(length, (p // page + 1) * page)
            at, s = tables[b][p // page], p % page
            k_pages[at, s:s + stop - p] = turned[p - first:stop - first, h:]
            v_pages[at, s:s + stop - p] = rows[p - first:stop - first, h + kv:].double()
            p = stop
    return {"q": q, "k_pages": k_pages, "v_pages": v_pages}


def _exact_cache(st, case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    starts, lengths = st["plan"]
    y = torch.zeros(starts[-1], h, d, dtype=torch.float64, device="cuda")
    tables = st["tables"].tolist()
    for b, length in enumerate(lengths):
        if not length:
            continue
        used = tables[b][:-(-length // case["page"])]
        for c in range(kv):
            k, v = (torch.cat([x[p, :, c] for p in used])[:length].double() if len(used) < 64 else
                    x[torch.tensor(used, device="cuda"), :, c].flatten(0, 1)[:length].double() for x in (st["k_pages"], st["v_pages"]))
            for n in range(c * h // kv, (c + 1) * h // kv):
                rows = st["q"][starts[b]:starts[b + 1], n].double()
                y[starts[b]:starts[b + 1], n] = _exact_rows(rows, k, v, length - rows.shape[0], case["window"], case["sinks"])
    return {"y": y}
