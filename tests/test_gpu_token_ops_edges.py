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
