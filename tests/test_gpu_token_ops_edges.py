"""The token operators where steps of one call overlap, and at values, layouts and settings beside the usual ones."""
import math
import zlib

import pytest
import torch

import token_oracle as oracle
from fbamtrain_b200 import ops

pytestmark = pytest.mark.gpu
BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------------------------------------------------------
# embedding
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,dim,dtype", [(32 * 33, 8, F32), (32 * 65 + 1, 3, F32), (32 * 129, 72, BF), (20_001, 40, F32), (70_001, 24, HALF)])
def test_embedding_sums_follow_one_another_in_used_memory(n, dim, dtype):
    """Each step of the sums reads the list and the partial sums that the one before it has just written, in memory of earlier
    calls with other tokens (odd counts of pieces: where one region ends the next begins in the same sector).  Gradients of
    whole numbers are exact."""
    gen = _gen("overlap", n, dim)
    table = torch.zeros(50, dim, dtype=dtype, device="cuda").requires_grad_()
    for turn in range(30):
        vocab = (1, 3, 50)[turn % 3]
        ids = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
        d_out = torch.randint(0, 2, (n, dim), generator=gen, device="cuda").to(dtype)
        grad, = torch.autograd.grad((ops.embed_tokens(ids, table),), (table,), (d_out,))
        want = torch.zeros(50, dim, dtype=torch.float64, device="cuda").index_add(0, ids, d_out.double())
        assert torch.equal(grad, want.to(dtype))


# ------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ------------------------------------------------------------------------------------------------------------------
def _mlp_check(rows, width, inner, out, dtype, act, extras, make=lambda t: t):
    """All outputs against 64 bits, with the bound of test_gated_mlp; `make` lays an input out."""
    gen = _gen("mlp", rows, width, inner, out, act)
    named = {"x": _randn(gen, rows, width, dtype=dtype), "w_in": _randn(gen, 2 * inner, width, dtype=dtype, scale=width ** -0.5),
             "w_out": _randn(gen, out, inner, dtype=dtype, scale=inner ** -0.5),
             "b_in": _randn(gen, 2 * inner, dtype=dtype, scale=0.1) if extras else None,
             "b_out": _randn(gen, out, dtype=dtype, scale=0.1) if extras else None,
             "residual": _randn(gen, rows, out, dtype=dtype) if extras else None}
    dy = make(_randn(gen, rows, out, dtype=dtype, scale=0.5))
    named = {k: make(v) if v is not None and v.dim() == 2 else v for k, v in named.items()}
    for v in named.values():
        if v is not None:
            v.requires_grad_()
    y = ops.gated_mlp(*(named[k] for k in ("x", "w_in", "w_out", "b_in", "b_out")), act, named["residual"])
    names = [k for k, v in named.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad((y,), [named[k] for k in names], (dy,))))
    with torch.no_grad():
        want, size = oracle.mlp(*(named[k] for k in ("x", "w_in", "w_out", "b_in", "b_out")), act, named["residual"], dy)
    relative = 1.01 * oracle.UNIT[dtype] + 8 * (rows + width + inner + 64) * 2.0 ** -24
    for name, got in [("y", y)] + list(grads.items()):
        oracle.within(got, want[name], dtype, relative * size[name] + 1e-6)


@pytest.mark.parametrize("rows,width,inner,out", [(1, 1000, 40, 1000), (1, 64, 1, 8), (4, 64, 24, 1), (1, 77, 51, 35), (1, 8, 8, 1)])
def test_gated_mlp_rows_of_any_pitch(rows, width, inner, out):
    """Slices of rows of odd lengths.  A single row counts as dense whatever its pitch is."""
    def sliced(t):
        wide = torch.zeros(t.shape[0] + 1, t.shape[1] + 1, dtype=t.dtype, device="cuda")
        wide[:-1, :-1] = t
        return wide[:-1, :-1].detach()
    _mlp_check(rows, width, inner, out, BF, "gelu", True, sliced)
    _mlp_check(rows, width, inner, out, HALF, "silu", False, sliced)


def test_gated_mlp_one_row_in_front_of_an_odd_width():
    """The gradient of a row that is joined with an odd number of columns comes as a slice of the joined row."""
    gen = _gen("joined")
    x, w_in, w_out = _randn(gen, 1, 64, dtype=BF), _randn(gen, 96, 64, dtype=BF, scale=0.1), _randn(gen, 40, 48, dtype=BF, scale=0.1)
    d = _randn(gen, 1, 43, dtype=BF)
    y = ops.gated_mlp(x.requires_grad_(), w_in, w_out)
    joined = torch.cat([y, torch.zeros(1, 3, dtype=BF, device="cuda")], 1)
    grad, = torch.autograd.grad((joined,), (x,), (d,))
    with torch.no_grad():
        want, size = oracle.mlp(x, w_in, w_out, None, None, "gelu", None, d[:, :40])
    oracle.within(grad, want["x"], BF, (1.01 * 2.0 ** -8 + 1e-4) * size["x"] + 1e-6)


def test_gated_mlp_refuses_weights_on_the_host():
    gen = _gen("host")
    x, w_in, w_out = _randn(gen, 4, 8, dtype=BF), _randn(gen, 32, 8, dtype=BF), _randn(gen, 8, 16, dtype=BF)
    for args in ((x, w_in.cpu(), w_out), (x, w_in, w_out.cpu())):
        with pytest.raises(ValueError, match="one device"):
            ops.gated_mlp(*args)
    with pytest.raises(ValueError, match="one device"):
        ops.linear(x, w_in.cpu())


def _block(rows, width, inner, out, needs=("x", "w_in", "w_out")):
    gen = _gen("block", rows, width)
    named = {"x": _randn(gen, rows, width, dtype=BF), "w_in": _randn(gen, 2 * inner, width, dtype=BF, scale=width ** -0.5),
             "w_out": _randn(gen, out, inner, dtype=BF, scale=inner ** -0.5)}
    for k in needs:
        named[k].requires_grad_()
    dy = _randn(gen, rows, out, dtype=BF)

    def step():
        y = ops.gated_mlp(**named)
        return y, torch.autograd.grad((y,), [named[k] for k in needs], (dy,))
    return step


@pytest.mark.parametrize("needs", [("x", "w_in", "w_out"), ("x",), ("w_in",), ("w_out",)])
def test_gated_mlp_counts_its_operations_once(needs):
    """2 rows inner (2 width + out) forward; of the backward what is wanted.  The same with a table of tuned tiles."""
    from fbamtrain_b200.ops import tuning
    from fbamtrain_b200.utils import flops
    rows, width, inner, out = 100, 48, 80, 24
    step = _block(rows, width, inner, out, needs)
    counted = []
    for table in (None, {}):
        tuning.set_table(table)
        try:
            flops.reset()
            step()
            counted.append(flops.snapshot()[0])
        finally:
            tuning.set_table(None)
    unit = 2.0 * rows * inner
    gating, dx, dw_in, dw_out = unit * out, unit * 2 * width, unit * 2 * width, unit * out
    want = unit * (2 * width + out) + ("x" in needs or "w_in" in needs) * gating + ("x" in needs) * dx + ("w_in" in needs) * dw_in + \
        ("w_out" in needs) * dw_out
    assert counted == [want, want]


def test_gated_mlp_splits_its_weight_gradients_with_a_tile_table_too():
    """What is split along the rows is not looked up in a table, as for linear layers."""
    from fbamtrain_b200.ops import tuning
    step = _block(4104, 64, 72, 56)
    y, plain = step()
    with tuning.recording() as noted:
        _, tuned = step()
    assert sorted(noted) == [tuning.gemm_key(4104, 56, 72, False, False), tuning.gemm_key(4104, 64, 144, False, True)]
    for a, b in zip(plain, tuned):
        oracle.within(a, b.double(), BF, 2.0 ** -8 * b.double().abs() + 1e-3)


@pytest.mark.parametrize("rows", [1, 8, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("width,inner,out", [(8, 8, 3), (24, 40, 17), (40, 264, 12), (100, 130, 61), (1000, 2056, 1000)])
@pytest.mark.parametrize("act,extras", [("gelu", True), ("silu", False), ("silu", True)])
def test_gated_mlp_answers_of_a_few_rows(rows, width, inner, out, act, extras):
    """Up to 32 rows the weights are streamed past the rows: both halves of 16 rows, parts of K that end inside a warp's run, columns
    behind the last eight."""
    _mlp_answer(rows, width, inner, out, BF, act, extras)
    _mlp_answer(rows, width, inner, out, HALF, act, extras)


# tiles of 64, of 128 and of pairs of CTAs with 256 columns of the accumulator, with whole and partial last ones of both sides
@pytest.mark.parametrize("rows,width,inner,out", [(64, 136, 1000, 72), (1100, 64, 1032, 40), (1300, 72, 1992, 64), (2561, 320, 2072, 136),
                                                  (4096, 128, 1288, 64)])
@pytest.mark.parametrize("act,extras", [("gelu", True), ("silu", False)])
def test_gated_mlp_answers_of_many_rows(rows, width, inner, out, act, extras):
    _mlp_answer(rows, width, inner, out, BF, act, extras)
    _mlp_answer(rows, width, inner, out, HALF, act, extras)


def _mlp_answer(rows, width, inner, out, dtype, act, extras):
    """y without gradients, with the bound of test_gated_mlp."""
    gen = _gen("mlp answer", rows, width, inner, out, act)
    x, residual = _randn(gen, rows, width, dtype=dtype), _randn(gen, rows, out, dtype=dtype) if extras else None
    w_in, w_out = _randn(gen, 2 * inner, width, dtype=dtype, scale=width ** -0.5), _randn(gen, out, inner, dtype=dtype, scale=inner ** -0.5)
    b_in, b_out = (_randn(gen, 2 * inner, dtype=dtype, scale=0.1), _randn(gen, out, dtype=dtype, scale=0.1)) if extras else (None, None)
    with torch.no_grad():
        y = ops.gated_mlp(x, w_in, w_out, b_in, b_out, act, residual)
    want, size = oracle.mlp(x, w_in, w_out, b_in, b_out, act, residual, torch.zeros(rows, out, device="cuda"))
    relative = 1.01 * oracle.UNIT[dtype] + 8 * (width + inner + 64) * 2.0 ** -24
    oracle.within(y, want["y"], dtype, relative * size["y"] + 1e-6)


@pytest.mark.parametrize("switch", [("TWO_CTA", False), ("TWO_CTA", True), ("USE_MN_MAJOR", False), ("DEBUG_KERNEL_LAUNCH", True),
                                    ("SYNC_EVERY_OP", True), ("PROFILE_LABELS", True), ("POISON_ALLOC", True)])
@pytest.mark.parametrize("rows,width,inner,out", [(20, 72, 90, 66), (2600, 256, 2048, 256)])
def test_gated_mlp_with_the_switches_of_the_other_products(switch, rows, width, inner, out, monkeypatch, capsys):
    from fbamtrain_b200.ops import native_ops
    from fbamtrain_b200.utils import debug
    name, value = switch
    monkeypatch.setattr(native_ops if hasattr(native_ops, name) else debug, name, value)
    if value is True and name == "TWO_CTA" and rows < 256:
        pytest.skip("pairs want tiles of 256 columns")
    _mlp_check(rows, width, inner, out, BF, "gelu", True)
    _mlp_answer(rows, width, inner, out, BF, "gelu", True)
    lines = [line.split("(")[0] for line in capsys.readouterr().out.splitlines() if line.startswith("[launch]")]
    if name == "DEBUG_KERNEL_LAUNCH":
        block = ["[launch] gated_few_rows"] if rows <= 32 else ["[launch] gated_block_fwd", "[launch] gemm"]
        assert lines == ["[launch] gated_block_fwd", "[launch] gemm", "[launch] gated_block_bwd"] + 3 * ["[launch] gemm"] + block


# ------------------------------------------------------------------------------------------------------------------
# all
# ------------------------------------------------------------------------------------------------------------------
def _calls():
    """Every operator as a function of one input, and that input."""
    gen = _gen("calls")
    ids = torch.randint(0, 20, (30,), generator=gen, device="cuda")
    w_in, w_out = _randn(gen, 96, 32, dtype=BF), _randn(gen, 24, 48, dtype=BF)
    return {"embed_tokens": (lambda t: ops.embed_tokens(ids, t), _randn(gen, 20, 16, dtype=BF)),
            "gated_recurrence": (lambda z: ops.gated_recurrence(z)[0], _randn(gen, 2, 30, 3, 16, dtype=BF)),
            "gated_mlp": (lambda x: ops.gated_mlp(x, w_in, w_out), _randn(gen, 40, 32, dtype=BF)),
            "token_logprobs": (lambda x: ops.token_logprobs(x, ids, 2).logprob, _randn(gen, 30, 64, dtype=BF))}


@pytest.mark.parametrize("name", ["embed_tokens", "gated_recurrence", "gated_mlp", "token_logprobs"])
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(name, grad):
    """Forward-mode differentiation has no formula here, and an answer without its tangent would be a wrong one."""
    call, x = _calls()[name]
    with torch.set_grad_enabled(grad):
        plain = call(x)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="jvp"):
                call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
            inside = call(x)
        oracle.within(inside, plain.double(), BF if plain.dtype == BF else F32, 2.0 ** -8 * plain.double().abs())
        assert torch.equal(call(x), plain)


@pytest.mark.parametrize("shape", [(40, 32, 48, 24), (40, 30, 50, 21)])
@pytest.mark.parametrize("name", ["x", "w_in", "w_out", "b_in"])
def test_a_second_derivative_of_the_block_is_refused(name, shape):
    gen = _gen("second", shape)
    rows, width, inner, out = shape
    named = {"x": _randn(gen, 5, rows // 5, width, dtype=BF), "w_in": _randn(gen, 2 * inner, width, dtype=BF),
             "w_out": _randn(gen, out, inner, dtype=BF), "b_in": _randn(gen, 2 * inner, dtype=BF)}
    for v in named.values():
        v.requires_grad_()
    y = ops.gated_mlp(**named)
    first, = torch.autograd.grad((y,), (named["w_in"],), (torch.ones_like(y),), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad((first.float().sum() + named[name].float().sum(),), (named[name],))


@pytest.mark.parametrize("name", ["embed_tokens", "gated_recurrence", "gated_mlp", "token_logprobs"])
def test_a_second_derivative_is_refused(name):
    """Of the gradient by what it depends on: the input (but for the embedding, whose gradient does not) and the gradient that
    comes in; alone and in a sum with what has a derivative."""
    call, x = _calls()[name]
    x.requires_grad_()
    y = call(x)
    up = torch.ones_like(y).requires_grad_()
    first, = torch.autograd.grad((y,), (x,), (up.detach(),), retain_graph=True)
    again, = torch.autograd.grad((y,), (x,), (up,), create_graph=True)
    assert torch.equal(first, again) and again.requires_grad
    for of in (up,) if name == "embed_tokens" else (up, x):
        for value in (again.float().square().sum(), again.float().sum() + of.float().sum()):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad((value,), (of,), retain_graph=True)


# ------------------------------------------------------------------------------------------------------------------
# log probabilities
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,vocab,dtype", [(400, 2_000_003, BF), (2, 15_000_001, BF), (1, 30_000_000, F32), (200, 3_600_007, F32)])
def test_logprobs_alternatives_of_any_vocabulary(rows, vocab, dtype):
    """A vocabulary of more batches than shared memory has room for the best of.  A sum in fp32 takes some 260 additions one after
    the other: that many units of 2^-24, of the logarithm and of differences of up to 6."""
    gen = _gen("vocabulary", rows, vocab)
    logits = torch.empty(rows, vocab, dtype=dtype, device="cuda").normal_(generator=gen)
    logits[0, vocab // 3::7] = 6.0                           # more equal values than candidates
    r = ops.token_logprobs(logits, None, 32)
    for i in {0, rows // 2, rows - 1}:
        ids = oracle.alternatives(logits[i:i + 1], 32)
        assert torch.equal(r.top_ids[i:i + 1], ids)
        _, entropy, logp, _ = oracle.logprobs(logits[i:i + 1], torch.zeros(1, dtype=torch.int64, device="cuda"), 1.0)
        oracle.within(r.entropy[i:i + 1], entropy, F32, 3e-4)
        oracle.within(r.top_logprobs[i:i + 1], logp.gather(1, ids), F32, 3e-4)


@pytest.mark.parametrize("width,out", [(1001, 8), (8, 1001)])
def test_gated_mlp_beyond_32_bit_counts(width, out):
    """More than 2^31 values of rows of an odd width, padded on the way in and cut on the way out."""
    rows, some = 2_200_000, slice(-100, None)
    gen = _gen("many rows", width)

    def at_the_end(n, scale):
        t = torch.zeros(rows, n, dtype=BF, device="cuda")
        t[some] = _randn(gen, 100, n, dtype=BF, scale=scale)
        return t

    named = {"x": at_the_end(width, 1.0), "w_in": _randn(gen, 16, width, dtype=BF, scale=width ** -0.5),
             "w_out": _randn(gen, out, 8, dtype=BF, scale=0.3), "b_in": _randn(gen, 16, dtype=BF), "b_out": _randn(gen, out, dtype=BF)}
    dy = at_the_end(out, 0.5)
    for v in named.values():
        v.requires_grad_()
    y = ops.gated_mlp(**named)
    grads = dict(zip(named, torch.autograd.grad((y,), list(named.values()), (dy,))))
    with torch.no_grad():
        want, size = oracle.mlp(named["x"][some], *(named[k] for k in ("w_in", "w_out", "b_in", "b_out")), "gelu", None, dy[some])
        relative = 1.01 * 2.0 ** -8 + 8 * (100 + width + 72) * 2.0 ** -24
        oracle.within(y[some], want["y"], BF, relative * size["y"] + 1e-6)
        oracle.within(grads["x"][some], want["x"], BF, relative * size["x"] + 1e-6)
        for name in ("w_in", "w_out", "b_in", "b_out"):
            oracle.within(grads[name], want[name], BF, relative * size[name] + 1e-6)
        assert not grads["x"][:-100].any()


def test_gated_mlp_without_outputs():
    """No output columns: an empty result and gradients of zeros, as on the CPU."""
    for device in ("cpu", "cuda"):
        x, w_in, w_out = (torch.ones(*s, dtype=BF, device=device).requires_grad_() for s in ((3, 8), (12, 8), (0, 6)))
        y = ops.gated_mlp(x, w_in, w_out)
        assert y.shape == (3, 0) and y.dtype == BF
        for g, of in zip(torch.autograd.grad((y,), (x, w_in, w_out), (torch.zeros_like(y),)), (x, w_in, w_out)):
            assert g.shape == of.shape and not g.any()


# ------------------------------------------------------------------------------------------------------------------
# gated recurrence
# ------------------------------------------------------------------------------------------------------------------
UNIT = 2.0 ** -24


def _scan_bounds(zgo, state, resets, dy, d_state, drop=None):
    """In 64 bits, time first: y, the last state, d_zgo and d_state, and for each a bound of the absolute error of its fp32 value.

    Every quantity goes through the scan three times: its value, the sum A of its terms' absolute values and its error E.  An
    exponential's argument is rounded once and its value is off by 2 units, the reciprocal by one: (|g| + 8) units of min(f, 1 - f),
    which is what moves the state; where f is small, but not far out (g >= -5), 1 - f may do.  So a step adds (|g| + 8) units of
    q A with q = 1 - f where g >= -5 and f below, and 4 units of A for its sums and the product of gates that carries the same
    value through a link; folding links adds 32 units of A at the end.
    `drop`: a step in front of which what the steps behind it hand on is lost (a mistake, for the test of the bounds)."""
    z, g, o = (x.transpose(0, 1) for x in zgo.detach().double().unbind(2))
    f, f1, s, s1 = torch.sigmoid(g), torch.sigmoid(-g), torch.sigmoid(o), torch.sigmoid(-o)
    q = torch.where(g >= -5, f1, f)
    off_g, off_o = UNIT * (g.abs() + 8), UNIT * (o.abs() + 8)
    steps = z.shape[0]
    h = torch.zeros_like(z[0]) if state is None else state.detach().double()
    size, err = h.abs(), torch.zeros_like(h)
    before, after, e_before, e_after, a_after = [], [], [], [], []
    for t in range(steps):
        if resets is not None:
            gone = resets[:, t].unsqueeze(1)
            h, size, err = (torch.where(gone, torch.zeros_like(v), v) for v in (h, size, err))
        before.append(h)
        e_before.append(err + 32 * UNIT * size)
        h = f[t] * h + f1[t] * z[t]
        add = off_g[t] * q[t] * (size + z[t].abs())
        size = f[t] * size + f1[t] * z[t].abs()
        err = f[t] * err + add + 4 * UNIT * size
        after.append(h)
        e_after.append(err + 32 * UNIT * size)
        a_after.append(size)
    before, after, e_before, e_after, a_after = (torch.stack(v) for v in (before, after, e_before, e_after, a_after))
    out = {"y": (s * after).transpose(0, 1), "last": h}
    bound = {"y": (s * e_after + 2 * off_o * s * a_after).transpose(0, 1), "last": e_after[-1]}
    d = dy.detach().double().transpose(0, 1)
    e = torch.zeros_like(z[0]) if d_state is None else d_state.detach().double()
    size, err = e.abs(), torch.zeros_like(e)
    grads, bounds = [], []
    for t in range(steps - 1, -1, -1):
        if t + 1 == drop:
            e = torch.zeros_like(e)
        dh = d[t] * s[t] + e
        a = d[t].abs() * s[t] + size
        eh = err + 32 * UNIT * size + 2 * off_o[t] * d[t].abs() * s[t] + UNIT * a
        step = before[t] - z[t]
        e_step = e_before[t] + UNIT * (before[t].abs() + z[t].abs())
        grads.append(torch.stack([dh * f1[t], dh * step * f[t] * f1[t], d[t] * after[t] * s[t] * s1[t]], 1))
        bounds.append(torch.stack([f1[t] * (eh + 2 * off_g[t] * a),
                                   f[t] * f1[t] * (step.abs() * eh + a * e_step + 4 * off_g[t] * a * (step.abs() + e_step)),
                                   d[t].abs() * s[t] * s1[t] * (e_after[t] + 4 * off_o[t] * a_after[t])], 1))
        add = off_g[t] * q[t] * a + 4 * UNIT * f[t] * a
        e, size, err = f[t] * dh, f[t] * a, f[t] * (err + 2 * off_o[t] * d[t].abs() * s[t] + UNIT * a) + add
        if resets is not None:
            gone = resets[:, t].unsqueeze(1)
            e, size, err = (torch.where(gone, torch.zeros_like(v), v) for v in (e, size, err))
    out.update(d_zgo=torch.stack(grads[::-1], 1), d_state=e)
    bound.update(d_zgo=torch.stack(bounds[::-1], 1), d_state=err + 32 * UNIT * size)
    return out, bound


def _recurrence_case(b, t, d, dtype, kind, extras, time_major):
    gen = _gen("recurrence", b, t, d, kind, extras)
    zgo = _randn(gen, t, b, 3, d, dtype=dtype).transpose(0, 1) if time_major else _randn(gen, b, t, 3, d, dtype=dtype)
    if kind == "long":                      # memories of some twenty steps
        zgo[:, :, 1] += 3.0
    elif kind == "short":                   # of one or two
        pass
    elif kind == "closed":                  # most gates far out on either side, and values of very different sizes
        zgo[:, :, 1] = (torch.rand(b, t, d, generator=gen, device="cuda") * 60 - 30).to(dtype)
        zgo[:, :, 0] *= torch.tensor([1.0, 1000.0, 0.01, 30.0], device="cuda").to(dtype).repeat(d // 4 + 1)[:d]
    state = _randn(gen, b, d, scale=1e4 if kind == "closed" else 1.0) if "state" in extras else None
    resets = torch.rand(b, t, generator=gen, device="cuda") < 0.01 if "resets" in extras else None
    return zgo, state, resets, _randn(gen, b, t, d, dtype=dtype), _randn(gen, b, d)


def _recurrence_run(zgo, state, resets, dy, d_state):
    zgo = zgo.detach().requires_grad_()
    state = None if state is None else state.detach().requires_grad_()
    y, last = ops.gated_recurrence(zgo, state, resets)
    grads = torch.autograd.grad((y, last), (zgo,) if state is None else (zgo, state), (dy, d_state))
    return {"y": y, "last": last, "d_zgo": grads[0], "d_state": grads[1] if state is not None else None}


# whole chunks and parts, one round and several of one CTA and of clusters, tiled and plain
RECURRENCE = [(2, 1, 64), (3, 5, 40), (2, 8, 33), (2, 128, 64), (1, 129, 130), (2, 257, 96), (1, 1025, 72), (1, 4100, 64), (1, 2100, 1300),
              (3, 700, 1024), (2, 900, 1416), (1, 2500, 65), (93, 200, 64)]


# (the oracle of a long one takes seconds: one of the extras each)
@pytest.mark.parametrize("b,t,d,extras", [(*s, e) for i, s in enumerate(RECURRENCE) for j, e in enumerate(["", "state", "state resets"])
                                          if s[1] < 500 or (i + j) % 3 == 0])
@pytest.mark.parametrize("kind", ["long", "short", "closed"])
def test_recurrence_values_and_gradients(b, t, d, kind, extras):
    """Each value against its own bound."""
    dtype = HALF if extras == "state" else BF
    case = _recurrence_case(b, t, d, dtype, kind, extras, time_major=extras == "state")
    want, bound = _scan_bounds(*case)
    for name, got in _recurrence_run(*case).items():
        if got is not None:
            oracle.within(got, want[name], F32 if name in ("last", "d_state") else dtype, bound[name])


@pytest.mark.parametrize("b,t,d", [(2, 128, 64), (1, 1025, 72), (3, 700, 1024)])
def test_recurrence_bounds_see_what_is_missing(b, t, d):
    """A gradient of zeros is outside the bounds nearly everywhere, and one that lost what is handed on in front of any chunk is
    outside in the steps before."""
    case = _recurrence_case(b, t, d, BF, "long", "state", False)
    want, bound = _scan_bounds(*case)
    allowed = bound["d_zgo"] + 2.0 ** -8 * want["d_zgo"].abs() + 2.0 ** -25
    assert float((allowed < want["d_zgo"].abs()).double().mean()) > 0.99
    for drop in (8, t // 2 // 8 * 8, (t - 1) // 8 * 8):
        wrong, _ = _scan_bounds(*case, drop=drop)
        over = (wrong["d_zgo"] - want["d_zgo"]).abs() > allowed
        assert bool(over[:, drop - 1, 0].any())


def _oracle_equal(got, want, dtype, finite_slack):
    """Infinities and NaN in the same places, what is finite within the type's rounding and a share of its row's size."""
    oracle.within(got, want, dtype, finite_slack * want.abs().nan_to_num(0.0, 0.0, 0.0) + finite_slack)


@pytest.mark.parametrize("b,t,d", [(2, 1, 64), (3, 7, 33), (2, 40, 64), (2, 300, 65), (1, 1500, 72), (1, 700, 1030), (1, 3000, 64)])
@pytest.mark.parametrize("where", ["z", "state", "z and state", "dy", "d_state", "all"])
@pytest.mark.parametrize("resets", [False, True])
def test_recurrence_infinities(b, t, d, where, resets):
    """An infinite candidate or state is what the definition makes of it: f inf + (1 - f) z is infinite until a reset, and of
    both signs together NaN; the same for gradients."""
    gen = _gen("infinities", b, t, d, where, resets)
    zgo = _randn(gen, b, t, 3, d, dtype=BF)
    zgo[:, :, 1] = zgo[:, :, 1] * 2 - 1                      # closed often: products of gates fall below the smallest number
    zgo[:, :, 1, : d // 2] += 4
    state, dy, d_state = _randn(gen, b, d), _randn(gen, b, t, d, dtype=BF), _randn(gen, b, d)
    marks = torch.rand(b, t, generator=gen, device="cuda") < 0.01 if resets else None

    def some(shape, share):
        sign = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.5, -INF, INF)
        return torch.rand(shape, generator=gen, device="cuda") < share, sign

    if "z" in where or where == "all":
        at, sign = some((b, t, d), 0.6 / t)
        zgo[:, :, 0] = torch.where(at, sign.to(BF), zgo[:, :, 0])
    if where in ("state", "z and state", "all"):
        at, sign = some((b, d), 0.3)
        state = torch.where(at, sign, state)
    if where in ("dy", "all"):
        at, sign = some((b, t, d), 0.6 / t)
        dy = torch.where(at, sign.to(BF), dy)
    if where in ("d_state", "all"):
        at, sign = some((b, d), 0.3)
        d_state = torch.where(at, sign, d_state)
    got = _recurrence_run(zgo, state, marks, dy, d_state)
    want_y, want_last, _, _ = oracle.recurrence(zgo, state, marks)
    want_zgo, want_state = oracle.recurrence_grad(zgo, state, marks, dy, d_state)
    # what is finite: 64 units of the largest value of each, over memories of up to some hundred steps
    _oracle_equal(got["y"], want_y, BF, 1e-3)
    _oracle_equal(got["last"], want_last, F32, 1e-3)
    _oracle_equal(got["d_zgo"], want_zgo, BF, 1e-2)
    _oracle_equal(got["d_state"], want_state, F32, 1e-2)


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gated_mlp_gradients_of_large_gates(act, dtype):
    """Far out the activation's derivative is 1 or 0.  Gates from rows of the identity, values of 1: no sum has a second term, so
    each gradient is a product of a few factors of 8 units each, and roundings of the type."""
    far = [300.0, 3e3, 3e4, 6e4] + ([1e8, 3e30] if dtype == BF else [5e4, 100.0]) + [20.0, 8.0]
    gates = torch.tensor(far + [-g for g in far] + [0.0, -0.0] + [3.0, -3.0] * 7, device="cuda").repeat(2)
    x = torch.eye(64, device="cuda").to(dtype)
    w_in = torch.zeros(128, 64, device="cuda")
    w_in[:64].fill_diagonal_(1.0)
    w_in[64:] = torch.diag(gates)
    w_in, w_out, dy = w_in.to(dtype).requires_grad_(), torch.eye(64, device="cuda").to(dtype), torch.eye(64, device="cuda").to(dtype)
    b_in = torch.zeros(128, dtype=dtype, device="cuda").requires_grad_()
    y = ops.gated_mlp(x, w_in, w_out, b_in, None, act)
    d_w, d_b = torch.autograd.grad((y,), (w_in, b_in), (dy,))
    with torch.no_grad():
        want, size = oracle.mlp(x, w_in, w_out, b_in, None, act, None, dy)
    unit = oracle.UNIT[dtype]
    # erf is approximated to 1.5e-7; the gates at which that shows are some units of 1
    slack = 1e-6
    oracle.within(d_w, want["w_in"], dtype, (1.01 * unit + 64 * 2.0 ** -24) * size["w_in"] + slack)
    oracle.within(d_b, want["b_in"], dtype, (1.01 * unit + 64 * 2.0 ** -24) * size["b_in"] + slack)


@pytest.mark.parametrize("needs,kept", [(("w_out", "b_out", "residual"), False), (("x",), True), (("w_in",), True), (("b_in",), True)])
@pytest.mark.parametrize("rows", [20, 300])
def test_gated_mlp_keeps_its_factors_where_they_are_needed(needs, kept, rows):
    """The fp32 factors, 8 bytes a hidden value, are for the gradients in front of the gating only."""
    gen = _gen("kept")
    named = {"x": _randn(gen, rows, 44, dtype=BF), "w_in": _randn(gen, 2 * 30, 44, dtype=BF, scale=0.1),
             "w_out": _randn(gen, 20, 30, dtype=BF, scale=0.1), "b_in": _randn(gen, 60, dtype=BF), "b_out": _randn(gen, 20, dtype=BF),
             "residual": _randn(gen, rows, 20, dtype=BF)}
    dy = _randn(gen, rows, 20, dtype=BF)
    want, size = oracle.mlp(*(named[k] for k in ("x", "w_in", "w_out", "b_in", "b_out")), "gelu", named["residual"], dy)
    for k in needs:
        named[k].requires_grad_()
    y = ops.gated_mlp(**named)
    assert any(t is not None and t.dtype == F32 for t in y.grad_fn.saved_tensors) == kept
    for k, g in zip(needs, torch.autograd.grad((y,), [named[k] for k in needs], (dy,))):
        oracle.within(g, want[k], BF, (1.01 * 2.0 ** -8 + 1e-4) * size[k] + 1e-6)


def test_recurrence_of_more_sequences_than_clusters_of_sixteen_could_have():
    b = 140_000_000
    gen = _gen("very many")
    zgo = torch.zeros(b, 1, 3, 1, dtype=BF, device="cuda")
    tail = _randn(gen, 100, 1, 3, 1, dtype=BF)
    zgo[-100:] = tail
    y, last = ops.gated_recurrence(zgo)
    want_y, want_last, _, _ = oracle.recurrence(tail, None, None)
    oracle.within(y[-100:], want_y, BF, 1e-5)
    oracle.within(last[-100:], want_last, F32, 1e-5)
    assert not y[:-100].any()


def test_inputs_that_the_gradients_do_not_read_may_be_overwritten():
    """A carried state in its place, and a bias, between the forward and the backward."""
    gen = _gen("overwritten")
    zgo, buffer, dy = _randn(gen, 2, 9, 3, 16, dtype=BF).requires_grad_(), _randn(gen, 2, 16), _randn(gen, 2, 9, 16, dtype=BF)
    want, = torch.autograd.grad(ops.gated_recurrence(zgo, buffer.clone())[:1], (zgo,), (dy,))
    y, last = ops.gated_recurrence(zgo, buffer)
    buffer.copy_(last.detach())
    assert torch.equal(torch.autograd.grad((y,), (zgo,), (dy,))[0], want)
    x, w_in, w_out, b_in = _randn(gen, 40, 30, dtype=BF), _randn(gen, 20, 30, dtype=BF), _randn(gen, 24, 10, dtype=BF), _randn(gen, 20, dtype=BF)
    w_in.requires_grad_()
    b_in.requires_grad_()
    dy = _randn(gen, 40, 24, dtype=BF)
    want = torch.autograd.grad((ops.gated_mlp(x, w_in, w_out, b_in),), (w_in, b_in), (dy,))
    y = ops.gated_mlp(x, w_in, w_out, b_in)
    with torch.no_grad():
        b_in.zero_()
    for a, b in zip(torch.autograd.grad((y,), (w_in, b_in), (dy,)), want):
        assert torch.equal(a, b)
