"""The token operators against their definitions in 64 bits: embedding, gated recurrence, gated feed-forward block and log
probabilities, at the sizes, strides and masks where they can go wrong."""
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
EMBED = [(1, 1, 1), (1, 17, 8), (7, 5, 3), (31, 100, 64), (33, 2, 40), (64, 1, 128), (1000, 1000, 250), (4097, 4096, 1024),
         (8193, 300, 72), (20000, 50021, 16), (70001, 1023, 24), (300, 262144, 8), (513, 8, 2056), (129, 40, 1029)]


@pytest.mark.parametrize("n,vocab,dim", EMBED)
@pytest.mark.parametrize("table_dtype,out_dtype", [(BF, BF), (HALF, HALF), (F32, BF), (F32, HALF), (F32, F32)])
def test_embedding(n, vocab, dim, table_dtype, out_dtype):
    gen = _gen("embed", n, vocab, dim)
    table = _randn(gen, vocab, dim, dtype=table_dtype).requires_grad_()
    # half of the positions share a few ids; some ids are outside the table
    ids = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    common = torch.rand(n, generator=gen, device="cuda") < 0.5
    ids[common] = ids[common] % 3 % vocab
    ids[torch.rand(n, generator=gen, device="cuda") < 0.05] = -1
    ids[torch.rand(n, generator=gen, device="cuda") < 0.05] = vocab
    scale = 1.7
    out = ops.embed_tokens(ids, table, scale, out_dtype)
    assert out.dtype == out_dtype
    want = oracle.embed(ids, table.detach(), scale)
    oracle.within(out, want, out_dtype, 2 ** -23 * want.abs())          # the scale's rounding and the product's
    d_out = _randn(gen, n, dim, dtype=out_dtype)
    grad, = torch.autograd.grad((out,), (table,), (d_out,))
    assert grad.dtype == table_dtype
    want, size = oracle.embed_grad(ids, d_out, vocab, scale)
    # a sum of k terms in fp32 is off by k units of its terms' sum at most; two more for the scale
    count = torch.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=vocab).unsqueeze(1)
    oracle.within(grad, want, table_dtype, (count + 2) * 2.0 ** -24 * size)
    again, = torch.autograd.grad((ops.embed_tokens(ids, table, scale, out_dtype),), (table,), (d_out,))
    assert torch.equal(grad, again)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_embedding_shapes_and_strides(ids_dtype):
    gen = _gen("strides")
    whole = _randn(gen, 50, 96, dtype=BF)
    ids = torch.randint(0, 50, (12, 9), generator=gen, device="cuda").to(ids_dtype)
    for table in (whole[:, :64], whole[:, 1:65], whole.t()[:40].t(), whole[::2]):
        rows = table.shape[0]
        out = ops.embed_tokens(ids.t(), table, 1.0)
        assert out.shape == (9, 12, table.shape[1])
        oracle.within(out, oracle.embed(ids.t(), table, 1.0), BF)
        assert rows == 50 or bool((out[(ids.t() >= rows)] == 0).all())
    table = whole.clone().requires_grad_()
    out = ops.embed_tokens(ids, table)
    d = _randn(gen, 9, 12, 96, dtype=BF).transpose(0, 1)
    grad, = torch.autograd.grad((out,), (table,), (d,))
    want, size = oracle.embed_grad(ids.reshape(-1), d.reshape(-1, 96), 50, 1.0)
    oracle.within(grad, want, BF, 110 * 2.0 ** -24 * size)


def test_embedding_without_tokens():
    table = torch.randn(5, 8, device="cuda").requires_grad_()
    out = ops.embed_tokens(torch.empty(3, 0, dtype=torch.int64, device="cuda"), table, 2.0, BF)
    assert out.shape == (3, 0, 8)
    assert torch.equal(torch.autograd.grad((out,), (table,), (out.detach(),))[0], torch.zeros(5, 8, device="cuda"))


def test_embedding_of_one_token_only():
    """Every piece is one run: its partial sums are joined over all pieces."""
    table = torch.zeros(3, 64, device="cuda").requires_grad_()
    for n in (32, 33, 64, 32 * 257, 32 * 600 + 5):
        ids = torch.ones(n, dtype=torch.int64, device="cuda")
        grad, = torch.autograd.grad((ops.embed_tokens(ids, table, 1.0),), (table,), (torch.ones(n, 64, device="cuda"),))
        assert torch.equal(grad[1], torch.full((64,), float(n), device="cuda"))
        assert not grad[0].any() and not grad[2].any()


@pytest.mark.parametrize("n,vocab,dim,dtype", [(700, 300_007, 5, BF), (5000, 2_000_003, 3, F32), (20_000, 2_000_003, 9, HALF),
                                               (3000, 100_003, 1029, BF)])
@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_embedding_writes_every_row_of_the_gradient(n, vocab, dim, dtype, ids_dtype):
    """Large tables of which few rows come up, in memory that held something else; rows of no whole number of 16-byte pieces."""
    gen = _gen("absent", n, vocab, dim)
    table = torch.zeros(vocab, dim, dtype=dtype, device="cuda").requires_grad_()
    ids = torch.randint(0, vocab, (n,), generator=gen, device="cuda").to(ids_dtype)
    ids[:2] = torch.tensor([0, vocab - 1])
    d_out = _randn(gen, n, dim, dtype=dtype)
    out = ops.embed_tokens(ids, table)
    stale = torch.full_like(table, math.nan)
    del stale
    grad, = torch.autograd.grad((out,), (table,), (d_out,))
    want, size = oracle.embed_grad(ids.long(), d_out, vocab, 1.0)
    count = torch.bincount(ids.long(), minlength=vocab).unsqueeze(1)
    oracle.within(grad, want, dtype, (count + 2) * 2.0 ** -24 * size)
    assert not grad[count[:, 0] == 0].any()


def test_embedding_table_beyond_32_bit_offsets():
    vocab, dim = 600_000, 4096                                # 2.5e9 values
    table = torch.zeros(vocab, dim, dtype=BF, device="cuda").requires_grad_()
    ids = torch.tensor([vocab - 1, 0, vocab - 1, vocab // 2], device="cuda")
    with torch.no_grad():
        table[vocab - 1] = 3.0
    out = ops.embed_tokens(ids, table, 2.0)
    assert torch.equal(out.detach()[:, 0].float().cpu(), torch.tensor([6.0, 0.0, 6.0, 0.0]))
    d = torch.ones(4, dim, dtype=BF, device="cuda")
    grad, = torch.autograd.grad((out,), (table,), (d,))
    assert bool((grad[vocab - 1] == 4.0).all()) and bool((grad[0] == 2.0).all()) and bool((grad[vocab // 2] == 2.0).all())
    assert int(torch.count_nonzero(grad[:, 0])) == 3


# ------------------------------------------------------------------------------------------------------------------
# gated recurrence
# ------------------------------------------------------------------------------------------------------------------
def _recurrence_bounds(zgo, state, resets, dy, d_state):
    """Absolute errors of the fp32 values before their rounding.  A gate is off by a few units of its size; the state moves
    towards z by (1 - f), so that of a value in [-m, m] an error of some 8 units of m comes in per step of memory and 1 / (1 - f)
    steps are remembered: 1 / (1 - f) * 8 * 2^-24 * m / (1 - f)^-1 ... = 64 units of m bound it with the carry's."""
    m = float(zgo[:, :, 0].abs().max()) + (float(state.abs().max()) if state is not None else 0.0)
    d = float(dy.abs().max()) + (float(d_state.abs().max()) if d_state is not None else 0.0)
    g = zgo[:, :, 1].double()
    memory = min(zgo.shape[1], float((1 / (1 - torch.sigmoid(g.clamp(max=20.0)))).max()))
    return 64 * 2.0 ** -24 * m * max(1.0, memory), 64 * 2.0 ** -24 * d * m * max(1.0, memory) ** 2


@pytest.mark.parametrize("b,t,d", [(1, 1, 1), (2, 1, 64), (8, 1, 1000), (3, 2, 33), (2, 15, 64), (2, 16, 66), (2, 17, 30), (1, 127, 130),
                                   (2, 128, 64), (2, 129, 65), (1, 1000, 40), (5, 257, 96), (1, 4100, 64)])
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("time_major", [False, True])
@pytest.mark.parametrize("extras", ["", "state", "state resets"])
def test_recurrence(b, t, d, dtype, time_major, extras):
    gen = _gen("recurrence", b, t, d, extras)
    zgo = _randn(gen, t, b, 3, d, dtype=dtype).transpose(0, 1) if time_major else _randn(gen, b, t, 3, d, dtype=dtype)
    zgo[:, :, 1] += 2.0
    zgo.requires_grad_()
    state = _randn(gen, b, d).requires_grad_() if "state" in extras else None
    resets = torch.rand(b, t, generator=gen, device="cuda") < 0.05 if "resets" in extras else None
    dy, d_state = _randn(gen, b, t, d, dtype=dtype), _randn(gen, b, d)
    y, last = ops.gated_recurrence(zgo, state, resets)
    into = (zgo,) if state is None else (zgo, state)
    grads = torch.autograd.grad((y, last), into, (dy, d_state))
    held = [x.detach() if x is not None else None for x in (zgo, state)]
    fwd, bwd = _recurrence_bounds(held[0], held[1], resets, dy, d_state)
    want_y, want_last, _, _ = oracle.recurrence(*held, resets)
    oracle.within(y, want_y, dtype, fwd)
    oracle.within(last, want_last, F32, fwd)
    want = oracle.recurrence_grad(*held, resets, dy, d_state)
    oracle.within(grads[0], want[0], dtype, bwd)
    if state is not None:
        oracle.within(grads[1], want[1], F32, bwd)


# From one CTA to as many as a cluster has, whole and partial rounds of it
@pytest.mark.parametrize("b,t,d", [(93, 200, 64), (1, 2100, 1300), (3, 700, 1024), (1, 600, 2368), (2, 900, 1416), (1, 2500, 960),
                                   (1, 2500, 65), (1, 1025, 72), (300, 100, 40), (7, 260, 500)])
def test_recurrence_over_clusters(b, t, d):
    gen = _gen("clusters", b, t, d)
    zgo, state = _randn(gen, b, t, 3, d, dtype=BF).requires_grad_(), _randn(gen, b, d).requires_grad_()
    resets = torch.rand(b, t, generator=gen, device="cuda") < 0.01
    dy, d_state = _randn(gen, b, t, d, dtype=BF), _randn(gen, b, d)
    y, last = ops.gated_recurrence(zgo, state, resets)
    grads = torch.autograd.grad((y, last), (zgo, state), (dy, d_state))
    held = zgo.detach(), state.detach()
    fwd, bwd = _recurrence_bounds(*held, resets, dy, d_state)
    want_y, want_last, _, _ = oracle.recurrence(*held, resets)
    oracle.within(y, want_y, BF, fwd)
    oracle.within(last, want_last, F32, fwd)
    want = oracle.recurrence_grad(*held, resets, dy, d_state)
    oracle.within(grads[0], want[0], BF, bwd)
    oracle.within(grads[1], want[1], F32, bwd)


def test_recurrence_in_pieces_is_the_whole():
    """The carried state of one call starts the next, down to single steps."""
    gen = _gen("pieces")
    zgo = _randn(gen, 3, 200, 3, 70, dtype=BF)
    whole, last = ops.gated_recurrence(zgo)
    state, ys = None, []
    for lo, hi in ((0, 1), (1, 2), (2, 50), (50, 187), (187, 200)):
        y, state = ops.gated_recurrence(zgo[:, lo:hi], state)
        ys.append(y)
    bound = 64 * 2.0 ** -24 * float(zgo[:, :, 0].abs().max()) * 200
    # two roundings of two values that differ by the bound
    oracle.within(torch.cat(ys, 1), whole.double(), BF, bound + 2.0 ** -8 * whole.double().abs())
    oracle.within(state, last.double(), F32, bound)


@pytest.mark.parametrize("value", [math.nan, INF])
def test_recurrence_reset_keeps_the_sequence_before_out(value):
    gen = _gen("reset")
    zgo = _randn(gen, 2, 300, 3, 64, dtype=BF)
    resets = torch.zeros(2, 300, dtype=torch.bool, device="cuda")
    resets[:, 150] = True
    clean = zgo.clone().requires_grad_()
    dirty = zgo.clone()
    dirty[:, 20, 0] = value
    dirty.requires_grad_()
    dy = _randn(gen, 2, 300, 64, dtype=BF)
    (y, last), (y2, last2) = ops.gated_recurrence(clean, None, resets), ops.gated_recurrence(dirty, None, resets)
    assert torch.equal(y[:, 150:], y2[:, 150:]) and torch.equal(last, last2) and torch.equal(y[:, :20], y2[:, :20])
    g, = torch.autograd.grad((y,), (clean,), (dy,))
    g2, = torch.autograd.grad((y2,), (dirty,), (dy,))
    assert torch.equal(g[:, 150:], g2[:, 150:])
    # and backwards: what a gradient behind the reset brings does not reach the steps before it
    bad = dy.clone()
    bad[:, 200] = value
    g3, = torch.autograd.grad(ops.gated_recurrence(clean, None, resets)[:1], (clean,), (bad,))
    assert torch.equal(g[:, :150], g3[:, :150])


def test_recurrence_extreme_gates():
    """Gates at the ends of the type: 0 and 1 exactly, and 1 - f far below one unit of 1."""
    zgo = torch.randn(2, 40, 3, 64, device="cuda").to(BF)
    zgo[:, :, 1] = torch.tensor([-INF, -200.0, -100.0, -20.0, 0.0, 20.0, 100.0, INF], device="cuda").to(BF).repeat(8)
    zgo[:, :, 2] = torch.tensor([INF, -INF, 50.0, -50.0], device="cuda").to(BF).repeat(16)
    state = torch.randn(2, 64, device="cuda")
    y, last = ops.gated_recurrence(zgo, state)
    want_y, want_last, _, _ = oracle.recurrence(zgo, state, None)
    oracle.within(y, want_y, BF, 1e-5)
    oracle.within(last, want_last, F32, 1e-5)


def test_recurrence_of_many_sequences():
    """More sequences than one dimension of a grid has places, of one step each."""
    b, d = 70_000, 24
    gen = _gen("many")
    zgo, state = _randn(gen, b, 1, 3, d, dtype=BF).requires_grad_(), _randn(gen, b, d)
    y, last = ops.gated_recurrence(zgo, state)
    want_y, want_last, _, _ = oracle.recurrence(zgo.detach(), state, None)
    oracle.within(y, want_y, BF, 1e-5)
    oracle.within(last, want_last, F32, 1e-5)
    dy = _randn(gen, b, 1, d, dtype=BF)
    g, = torch.autograd.grad((y,), (zgo,), (dy,))
    oracle.within(g, oracle.recurrence_grad(zgo.detach(), state, None, dy, None)[0], BF, 1e-4)


def test_recurrence_without_steps():
    state = torch.randn(3, 8, device="cuda")
    y, last = ops.gated_recurrence(torch.empty(3, 0, 3, 8, dtype=BF, device="cuda"), state)
    assert y.shape == (3, 0, 8) and torch.equal(last, state)


@pytest.mark.parametrize("dy_kind", ["none", "expanded", "strided"])
def test_recurrence_gradients_of_other_layouts(dy_kind):
    gen = _gen("layouts")
    base = _randn(gen, 2, 50, 4, 80, dtype=BF)
    zgo = base[:, :, 1:, 5:69].requires_grad_()               # odd start: no 4-byte pairs
    y, last = ops.gated_recurrence(zgo)
    want_y, want_last, _, _ = oracle.recurrence(zgo.detach(), None, None)
    fwd = 64 * 2.0 ** -24 * 6 * 50
    oracle.within(y, want_y, BF, fwd)
    if dy_kind == "none":
        dy, d_last = torch.zeros(2, 50, 64, dtype=BF, device="cuda"), _randn(gen, 2, 64)
        grad, = torch.autograd.grad((last,), (zgo,), (d_last,))
    else:
        d_last = None
        dy = torch.ones(1, 1, 1, dtype=BF, device="cuda").expand(2, 50, 64) if dy_kind == "expanded" else _randn(gen, 2, 50, 2, 64, dtype=BF)[:, :, 1]
        grad, = torch.autograd.grad((y,), (zgo,), (dy,))
    want, _ = oracle.recurrence_grad(zgo.detach(), None, None, dy, d_last)
    oracle.within(grad, want, BF, 64 * 2.0 ** -24 * 6 * 5 * 50 ** 2)


def test_recurrence_beyond_32_bit_offsets():
    t, d = 180_000, 4096                                      # 2.2e9 values of projections
    zgo = torch.zeros(1, t, 3, d, dtype=BF, device="cuda")
    tail = torch.randn(1, 100, 3, d, device="cuda").to(BF)
    zgo[:, -100:] = tail
    resets = torch.zeros(1, t, dtype=torch.bool, device="cuda")
    resets[:, -100] = True
    zgo.requires_grad_()
    y, last = ops.gated_recurrence(zgo, None, resets)
    small = tail.clone().requires_grad_()
    y2, last2 = ops.gated_recurrence(small)
    # another division into chunks: equal but for fp32 roundings, and the rounding of each
    oracle.within(y[:, -100:], y2.double(), BF, 1e-4 + 2.0 ** -8 * y2.double().abs())
    oracle.within(last, last2.double(), F32, 1e-4)
    dy = torch.zeros(1, t, d, dtype=BF, device="cuda")
    dy[:, -100:] = 1.0
    g, = torch.autograd.grad((y,), (zgo,), (dy,))
    g2, = torch.autograd.grad((y2,), (small,), (dy[:, -100:],))
    oracle.within(g[:, -100:], g2.double(), BF, 1e-3 + 2.0 ** -8 * g2.double().abs())
    assert not g[:, :-100].any()


# ------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,width,inner,out", [(1, 64, 64, 64), (3, 8, 8, 8), (8, 256, 1024, 256), (17, 40, 24, 72), (129, 136, 200, 136),
                                                  (256, 128, 128, 128), (300, 100, 130, 60), (33, 77, 51, 35), (1000, 320, 1032, 320),
                                                  (2500, 256, 2048, 256)])
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("act,extras", [("gelu", True), ("silu", False)])
def test_gated_mlp(rows, width, inner, out, dtype, act, extras):
    gen = _gen("mlp", rows, width, inner, act)
    x = _randn(gen, rows, width, dtype=dtype)
    w_in, w_out = _randn(gen, 2 * inner, width, dtype=dtype, scale=width ** -0.5), _randn(gen, out, inner, dtype=dtype, scale=inner ** -0.5)
    b_in, b_out, residual = ((_randn(gen, 2 * inner, dtype=dtype, scale=0.1), _randn(gen, out, dtype=dtype, scale=0.1),
                              _randn(gen, rows, out, dtype=dtype)) if extras else (None, None, None))
    dy = _randn(gen, rows, out, dtype=dtype, scale=0.5)
    named = {"x": x, "w_in": w_in, "w_out": w_out, "b_in": b_in, "b_out": b_out, "residual": residual}
    for v in named.values():
        if v is not None:
            v.requires_grad_()
    y = ops.gated_mlp(x, w_in, w_out, b_in, b_out, act, residual)
    names = [k for k, v in named.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad((y,), [named[k] for k in names], (dy,))))
    with torch.no_grad():
        want, size = oracle.mlp(x, w_in, w_out, b_in, b_out, act, residual, dy)
    unit = oracle.UNIT[dtype]
    # h and the gradients of (v, g) are rounded once to the type before the second product: at most one unit of the sum of
    # the terms.  fp32 sums of the longest of the products, of `width` behind them and of the gate: that many units of 2^-24,
    # times 8 for the factors by which the gate's derivative and the value pass an error of the first product on.
    relative = 1.01 * unit + 8 * (rows + width + inner + 64) * 2.0 ** -24
    for name, got in [("y", y)] + list(grads.items()):
        oracle.within(got, want[name], dtype, relative * size[name] + 1e-6)


def test_gated_mlp_shapes_and_strides():
    gen = _gen("mlp strides")
    x = _randn(gen, 5, 7, 3, 64, dtype=BF)[:, :, 1].transpose(0, 1)
    w_in, w_out = _randn(gen, 2 * 96, 128, dtype=BF, scale=0.1)[:, :64], _randn(gen, 96, 72, dtype=BF, scale=0.1).t()
    res = _randn(gen, 1, 1, 72, dtype=BF).expand(7, 5, 72)
    y = ops.gated_mlp(x, w_in, w_out, act="silu", residual=res)
    assert y.shape == (7, 5, 72)
    want, size = oracle.mlp(x.reshape(35, 64), w_in, w_out, None, None, "silu", res.reshape(35, 72), torch.zeros(35, 72, device="cuda"))
    oracle.within(y.reshape(35, 72), want["y"], BF, (1.01 * 2.0 ** -8 + 1e-4) * size["y"] + 1e-6)
    assert ops.gated_mlp(x[:0], w_in, w_out, act="silu").shape == (0, 5, 72)


def test_gated_mlp_large_gates():
    """Gates of both signs far out: the activation is the gate itself or 0."""
    x = torch.eye(64, device="cuda").to(BF)
    w_in = torch.zeros(128, 64, device="cuda").to(BF)
    w_in[:64] = 1.0
    w_in[64:] = torch.tensor([-3e4, -200.0, -90.0, 90.0, 200.0, 3e4, 0.0, -0.0], device="cuda").repeat(8).to(BF)[None, :]
    w_out = torch.eye(64, device="cuda").to(BF)
    for act in ("gelu", "silu"):
        y = ops.gated_mlp(x, w_in, w_out, act=act)
        want, size = oracle.mlp(x, w_in, w_out, None, None, act, None, torch.zeros(64, 64, device="cuda"))
        oracle.within(y, want["y"], BF, (2.0 ** -8 + 1e-4) * size["y"] + 1e-6)


# ------------------------------------------------------------------------------------------------------------------
# log probabilities
# ------------------------------------------------------------------------------------------------------------------
def _logprob_bound(logits, temperature):
    """Absolute error of an fp32 log probability: differences and products of some 8 units of their sizes, 2^-22 of the
    exponential's approximation, and the logarithm's."""
    x = logits.double() / temperature
    spread = torch.where(x.isfinite(), x.amax(-1, keepdim=True) - x, 0.0).amax(-1)
    return 16 * 2.0 ** -24 * (spread + 16)


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 7, 7), (5, 17, 0), (300, 64, 5), (4, 255, 3), (4, 256, 32), (9, 257, 32),
                                            (2, 1000, 20), (33, 1025, 5), (2, 4096, 5), (2, 9000, 32), (1, 50021, 20), (1, 262144, 32)])
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("padded", [False, True])
def test_logprobs(rows, vocab, top, dtype, masked, padded):
    gen = _gen("logprobs", rows, vocab, top, masked)
    full = _randn(gen, rows, (vocab + 7) // 8 * 8 if padded else vocab, dtype=dtype, scale=3.0)
    if masked:
        full[torch.rand(full.shape, generator=gen, device="cuda") < 0.4] = -INF
        full[rows // 2] = -INF
    logits = full[:, :vocab].requires_grad_()
    targets = torch.randint(-2, vocab + 1, (rows,), generator=gen, device="cuda")
    for temperature in (1.0, 0.3):
        r = ops.token_logprobs(logits, targets, top, temperature)
        held = logits.detach()
        lp, entropy, logp, p = oracle.logprobs(held, targets, temperature)
        bound = _logprob_bound(held, temperature)
        oracle.within(r.logprob, lp, F32, bound)
        oracle.within(r.entropy, entropy, F32, bound)
        if top:
            ids = oracle.alternatives(held, top)
            assert torch.equal(r.top_ids, ids)
            oracle.within(r.top_logprobs, logp.gather(1, ids), F32, bound.unsqueeze(1))
        else:
            assert r.top_ids is None and r.top_logprobs is None
        dl, dh = _randn(gen, rows), _randn(gen, rows)
        grad, = torch.autograd.grad((r.logprob, r.entropy), (logits,), (dl, dh))
        want = oracle.logprobs_grad(held, targets, temperature, dl, dh)
        # p is off by the log probability's error times itself, and the entropy's term by the size of log p once more
        size = (dl.abs() + dh.abs() * (1 + bound + entropy)).unsqueeze(1).double() / temperature
        term = p * torch.where(p == 0, torch.zeros_like(p), logp.abs() + 1)
        oracle.within(grad, want, dtype, 4 * bound.unsqueeze(1) * size * (term + p) + 2.0 ** -22 * size)


@pytest.mark.parametrize("dtype", [BF, HALF, F32])
def test_logprobs_equal_values(dtype):
    """Ties go to the lowest id: rows of one value, of two, of zeros with both signs, of the type's lowest value."""
    logits = torch.zeros(5, 5000, dtype=dtype, device="cuda")
    logits[1, 777:] = 1.0
    logits[2, ::2] = -0.0
    logits[3] = torch.finfo(dtype).min
    logits[4, 4990:] = torch.finfo(dtype).max / 4
    r = ops.token_logprobs(logits, torch.full((5,), 4995, device="cuda"), 32)
    assert torch.equal(r.top_ids, oracle.alternatives(logits, 32))
    lp, entropy, _, _ = oracle.logprobs(logits, torch.full((5,), 4995, device="cuda"), 1.0)
    oracle.within(r.logprob, lp, F32, 1e-5)
    oracle.within(r.entropy, entropy, F32, 1e-5)


@pytest.mark.parametrize("vocab", [50, 3000])
def test_logprobs_not_numbers(vocab):
    logits = torch.randn(3, vocab, device="cuda")
    logits[0, 7] = math.nan
    logits[1, :] = math.nan
    logits[2, 11] = -INF
    t = torch.tensor([3, 3, 11], device="cuda")
    r = ops.token_logprobs(logits.requires_grad_(), t, 8)
    assert r.logprob[:2].isnan().all() and r.entropy[:2].isnan().all() and r.top_logprobs[:2].isnan().all()
    assert float(r.logprob[2]) == -INF and bool(r.entropy[2].isfinite())
    assert torch.equal(r.top_ids, oracle.alternatives(logits.detach(), 8))
    g, = torch.autograd.grad((r.logprob.sum() + r.entropy.sum(),), (logits,))
    assert g[:2].isnan().any(1).all() and g[2].isfinite().all()


def test_logprobs_shapes_and_parts():
    gen = _gen("shapes")
    logits = _randn(gen, 4, 6, 100, dtype=BF).transpose(0, 1).requires_grad_()
    t = torch.randint(0, 100, (6, 4), generator=gen, device="cuda", dtype=torch.int32)
    r = ops.token_logprobs(logits, t, 3)
    assert r.logprob.shape == (6, 4) and r.top_ids.shape == (6, 4, 3)
    lp, entropy, _, _ = oracle.logprobs(logits.detach(), t, 1.0)
    oracle.within(r.logprob, lp, F32, 1e-5)
    # one output alone has the gradient of that output
    g, = torch.autograd.grad((r.entropy,), (logits,), (torch.ones(6, 4, device="cuda"),))
    zeros, ones = torch.zeros(6, 4, device="cuda"), torch.ones(6, 4, device="cuda")
    oracle.within(g, oracle.logprobs_grad(logits.detach(), t, 1.0, zeros, ones), BF, 1e-5)
    r = ops.token_logprobs(logits, None, 2)
    assert r.logprob is None
    g2, = torch.autograd.grad((r.entropy,), (logits,), (torch.ones(6, 4, device="cuda"),))
    assert torch.equal(g, g2)
    assert ops.token_logprobs(logits[:0], t[:0], 2).top_ids.shape == (0, 4, 2)


@pytest.mark.parametrize("vocab", [1, 5, 8, 31, 257, 4099, 50257])
@pytest.mark.parametrize("start", [0, 1, 3])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_rows_that_start_anywhere(vocab, start, dtype):
    """Dense rows of odd lengths and views at odd starts: 16-byte pieces of a row begin in front of it."""
    gen = _gen("starts", vocab, start)
    rows, top = 7, min(vocab, 4)
    flat = _randn(gen, rows * vocab + 8, dtype=dtype, scale=3.0)
    flat[:start] = flat[start + rows * vocab:] = 1e4                  # neighbours that must not count
    logits = flat[start:start + rows * vocab].view(rows, vocab).requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    r = ops.token_logprobs(logits, t, top)
    held = logits.detach()
    lp, entropy, logp, _ = oracle.logprobs(held, t, 1.0)
    oracle.within(r.logprob, lp, F32, 1e-5)
    oracle.within(r.entropy, entropy, F32, 1e-5)
    assert torch.equal(r.top_ids, oracle.alternatives(held, top))
    dl, dh = _randn(gen, rows), _randn(gen, rows)
    g, = torch.autograd.grad((r.logprob, r.entropy), (logits,), (dl, dh))
    oracle.within(g, oracle.logprobs_grad(held, t, 1.0, dl, dh), dtype, 1e-4)


def test_logprobs_gradient_against_differences():
    """Along a direction, the 64-bit values' central difference against the kernel's gradient in fp32: the difference is off
    by h^2 times a third derivative, the gradient by fp32 roundings of a sum over the vocabulary."""
    gen = _gen("differences")
    logits, v = _randn(gen, 6, 333, scale=2.0), _randn(gen, 6, 333)
    t = torch.randint(0, 333, (6,), generator=gen, device="cuda")
    dl, dh = _randn(gen, 6).double(), _randn(gen, 6).double()

    def value(x):
        lp, entropy, _, _ = oracle.logprobs(x, t, 0.8)
        return float((lp * dl + entropy * dh).sum())

    r = ops.token_logprobs(logits.requires_grad_(), t, 0, 0.8)
    grad, = torch.autograd.grad((r.logprob, r.entropy), (logits,), (dl.float(), dh.float()))
    h = 1e-5
    base = logits.detach().double()
    assert float((grad.double() * v.double()).sum()) == pytest.approx((value(base + h * v) - value(base - h * v)) / (2 * h), abs=1e-4)


def test_recurrence_and_mlp_gradients_against_differences():
    """The same for the other operators, whose gradients come rounded to the type: one unit of the sum of the terms."""
    gen = _gen("differences 2")
    zgo, state, v = _randn(gen, 2, 37, 3, 20, dtype=HALF), _randn(gen, 2, 20), _randn(gen, 2, 37, 3, 20).double()
    resets = torch.rand(2, 37, generator=gen, device="cuda") < 0.1
    dy, d_last = _randn(gen, 2, 37, 20, dtype=HALF), _randn(gen, 2, 20)
    y, last = ops.gated_recurrence(zgo.requires_grad_(), state, resets)
    grad, = torch.autograd.grad((y, last), (zgo,), (dy, d_last))

    def value(x):
        y, last, _, _ = oracle.recurrence(x, state, resets)
        return float((y * dy.double()).sum() + (last * d_last.double()).sum())

    base, h = zgo.detach().double(), 1e-5
    slack = 2.0 ** -11 * float((grad.double().abs() * v.abs()).sum()) + 1e-3
    assert abs(float((grad.double() * v).sum()) - (value(base + h * v) - value(base - h * v)) / (2 * h)) < slack

    x, w_in, w_out = _randn(gen, 20, 24, dtype=HALF), _randn(gen, 64, 24, dtype=HALF, scale=0.3), _randn(gen, 24, 32, dtype=HALF, scale=0.3)
    d, v = _randn(gen, 20, 24, dtype=HALF), _randn(gen, 64, 24).double()
    for act in ("gelu", "silu"):
        y = ops.gated_mlp(x, w_in.requires_grad_(), w_out, act=act)
        grad, = torch.autograd.grad((y,), (w_in,), (d,))

        def mlp_value(w):
            return float((oracle.mlp(x, w, w_out, None, None, act, None, d)[0]["y"] * d.double()).sum())

        base = w_in.detach().double()
        with torch.no_grad():
            size = oracle.mlp(x, w_in, w_out, None, None, act, None, d)[1]["w_in"]
        slack = 2 * 2.0 ** -11 * float((size * v.abs()).sum()) + 1e-3
        with torch.no_grad():
            assert abs(float((grad.double() * v).sum()) - (mlp_value(base + h * v) - mlp_value(base - h * v)) / (2 * h)) < slack


def test_logprobs_beyond_32_bit_offsets():
    rows, vocab = 36_000, 65_536                              # 2.4e9 logits
    logits = torch.zeros(rows, vocab, dtype=BF, device="cuda")
    logits[-1] = torch.randn(vocab, device="cuda").to(BF)
    logits.requires_grad_()
    t = torch.full((rows,), 5, device="cuda")
    r = ops.token_logprobs(logits, t, 2)
    last = logits.detach()[-1:]
    lp, entropy, _, _ = oracle.logprobs(last, t[-1:], 1.0)
    oracle.within(r.logprob[-1:], lp, F32, 1e-5)
    assert torch.equal(r.top_ids[-1:], oracle.alternatives(last, 2))
    dl = torch.ones(rows, device="cuda")
    g, = torch.autograd.grad((r.logprob,), (logits,), (dl,))
    oracle.within(g[-1:], oracle.logprobs_grad(last, t[-1:], 1.0, dl[-1:], 0 * dl[-1:]), BF, 1e-6)


# ------------------------------------------------------------------------------------------------------------------
# all
# ------------------------------------------------------------------------------------------------------------------
def test_operators_on_another_stream_and_twice():
    """On a side stream, the same bits twice, and the same as on the default stream."""
    gen = _gen("streams")
    ids = torch.randint(0, 200, (3000,), generator=gen, device="cuda")
    table = _randn(gen, 200, 64, dtype=BF).requires_grad_()
    zgo = _randn(gen, 2, 700, 3, 64, dtype=BF).requires_grad_()
    x, w_in, w_out = _randn(gen, 300, 64, dtype=BF), _randn(gen, 256, 64, dtype=BF, scale=0.1).requires_grad_(), _randn(gen, 64, 128, dtype=BF, scale=0.1)
    logits = _randn(gen, 50, 3000, dtype=BF).requires_grad_()
    t = torch.randint(0, 3000, (50,), generator=gen, device="cuda")

    def all_of_them():
        out = ops.embed_tokens(ids, table)
        y, last = ops.gated_recurrence(zgo)
        m = ops.gated_mlp(x, w_in, w_out, act="gelu")
        r = ops.token_logprobs(logits, t, 4)
        grads = torch.autograd.grad((out, y, m, r.logprob, r.entropy), (table, zgo, w_in, logits),
                                    (out.detach(), y.detach(), m.detach(), r.logprob.detach(), r.entropy.detach()))
        return [v.detach().clone() for v in (out, y, last, m, *r, *grads)]

    first = all_of_them()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = all_of_them()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_operators_are_captured_in_a_graph():
    gen = _gen("graph")
    ids = torch.randint(0, 20, (100,), generator=gen, device="cuda")
    table = _randn(gen, 20, 64, dtype=BF)
    zgo, state = _randn(gen, 2, 1, 3, 64, dtype=BF), _randn(gen, 2, 64)
    x, w_in, w_out = _randn(gen, 2, 64, dtype=BF), _randn(gen, 256, 64, dtype=BF), _randn(gen, 64, 128, dtype=BF)
    logits = _randn(gen, 2, 300, dtype=BF)

    def step():
        y, h = ops.gated_recurrence(zgo, state)
        return [ops.embed_tokens(ids, table), y, h, ops.gated_mlp(x, w_in, w_out), *ops.token_logprobs(logits, ids[:2], 3)]

    with torch.no_grad():
        want = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("vocab", [300, 4096, 70001, 262144])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_more_equal_values_than_candidates(vocab, dtype):
    """A few allowed tokens among masked ones, plateaus, and large values that all lie where one thread reads them."""
    logits = torch.full((5, vocab), -INF, dtype=dtype, device="cuda")
    logits[0, [vocab - 1, 3, vocab // 2]] = torch.tensor([1.0, 2.0, 1.0], device="cuda").to(dtype)
    logits[1] = 0.5
    logits[1, vocab // 3::7] = 0.75
    logits[2, -40:] = -3.0
    logits[3] = torch.arange(vocab, device="cuda") % 3
    logits[4] = torch.randn(vocab, device="cuda").to(dtype)
    logits[4].view(-1)[::128] += 10.0                         # stride of a few threads' vectors
    for top in (1, 5, 32):
        r = ops.token_logprobs(logits, None, top)
        ids = oracle.alternatives(logits, top)
        assert torch.equal(r.top_ids, ids)
        _, _, logp, _ = oracle.logprobs(logits, torch.zeros(5, dtype=torch.int64, device="cuda"), 1.0)
        oracle.within(r.top_logprobs, logp.gather(1, ids), F32, 1e-5)


def test_logprobs_values_of_one_thread_only():
    """More values above the k-th best thread's best than the list of candidates has room for."""
    vocab = 262144
    logits = torch.randn(1, vocab, device="cuda")
    for dtype, vec in ((BF, 8), (F32, 4)):
        x = logits.to(dtype)
        for threads in (32, 128, 512, 4096):                  # of a row, in the launches that there are
            y = x.clone().view(1, -1)
            wide = y[:, : vocab // (threads * vec) * threads * vec].view(1, -1, threads, vec)
            wide[:, :, 0] += 20.0
            r = ops.token_logprobs(y, None, 32)
            assert torch.equal(r.top_ids, oracle.alternatives(y, 32))


def test_gated_mlp_with_a_tile_table():
    """A table of tuned tiles is used for the block's plain products, and nothing else changes."""
    from fbamtrain_b200.ops import tuning
    gen = _gen("tuned")
    x, w_in, w_out = _randn(gen, 260, 72, dtype=BF), _randn(gen, 2 * 90, 72, dtype=BF, scale=0.1), _randn(gen, 66, 90, dtype=BF, scale=0.1)
    dy = _randn(gen, 260, 66, dtype=BF)
    named = [t.requires_grad_() for t in (x, w_in, w_out)]

    def both():
        y = ops.gated_mlp(x, w_in, w_out)
        return [y.detach(), *torch.autograd.grad((y,), named, (dy,))]

    plain = both()
    with tuning.recording() as noted:
        tuned = both()
    assert len(noted) >= 3
    for a, b in zip(plain, tuned):
        # other tiles, other order of fp32 sums: at most one unit of the type apart
        oracle.within(a, b.double(), BF, 2.0 ** -8 * b.double().abs() + 1e-3)


@pytest.mark.parametrize("needs", ["x", "w_in", "w_out", "b_in", "b_out", "residual"])
def test_gated_mlp_one_gradient_at_a_time(needs):
    gen = _gen("needs")
    named = {"x": _randn(gen, 50, 44, dtype=BF), "w_in": _randn(gen, 2 * 30, 44, dtype=BF, scale=0.1),
             "w_out": _randn(gen, 20, 30, dtype=BF, scale=0.1), "b_in": _randn(gen, 60, dtype=BF), "b_out": _randn(gen, 20, dtype=BF),
             "residual": _randn(gen, 50, 20, dtype=BF)}
    dy = _randn(gen, 50, 20, dtype=BF)
    want, size = oracle.mlp(*(named[k] for k in ("x", "w_in", "w_out", "b_in", "b_out")), "gelu", named["residual"], dy)
    named[needs].requires_grad_()
    y = ops.gated_mlp(named["x"], named["w_in"], named["w_out"], named["b_in"], named["b_out"], "gelu", named["residual"])
    g, = torch.autograd.grad((y,), (named[needs],), (dy,))
    oracle.within(g, want[needs], BF, (1.01 * 2.0 ** -8 + 1e-4) * size[needs] + 1e-6)
