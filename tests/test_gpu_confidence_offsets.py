"""Token log probabilities of logits that share a large offset: only distances
from the maximum count, in the kernel of few rows and in that of many."""
import pytest
import torch

import voxcuda as V
from rows_ref import TORCH, U32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def bound(vocab, n, dtype):
    """Relative error of a sum of e^(x - m), u = 2^-24: ex2's 2 ulp (4 u), a
    thread's additions (8 of a batch of 64 bytes, one for each batch, 2 to
    join), and 7 u (ex2, two products, an addition) each time that a
    running maximum moves - once a batch at most - and for each of the at most
    12 levels (5 in a warp, 3 over warps, 4 over shares) that join the sums."""
    per = 64 // torch.finfo(TORCH[dtype]).bits * 8 * (256 if n <= 148 else 128)
    batches = -(-vocab // per)
    return (4 + 10 + batches + 7 * (batches + 12)) * U32


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("offset", [0.0, 100.0, -100.0, 1000.0, -1000.0, 5000.0, -5000.0, 30000.0, -30000.0])
@pytest.mark.parametrize("n,vocab", [(3, 9001), (200, 4099)])
def test_a_common_offset_changes_nothing(dtype, offset, n, vocab):
    """A distance d = x - m and its product with log2 e are each off by half a
    step, the constant by a quarter of u: e^d by 2.25 u |d| beyond `bound`."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(n, vocab, generator=g, device="cuda") * 3 + offset).to(TORCH[dtype])
    tok = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    ids, top = torch.empty(n, 5, dtype=torch.int32, device="cuda"), torch.empty(n, 5, device="cuda")
    V.token_logprobs_dev(x.data_ptr(), dtype, n, vocab, 0, tok.data_ptr(), 5, lp.data_ptr(), ent.data_ptr(), ids.data_ptr(),
                         top.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    x = x.double()
    d = x - x.amax(-1, keepdim=True)
    lz = torch.logsumexp(d, -1)
    w = (d - lz[:, None]).exp()
    mean, square = (w * -d).sum(-1), (w * d * d).sum(-1)
    e = bound(vocab, n, dtype)
    tol_z = e + 2.25 * U32 * mean + 2 * U32 * lz + U32
    at = d.gather(1, tok[:, None].long()).squeeze(1)
    # the token's distance and the difference: half a step each
    assert bool(((lp - (at - lz)).abs() <= tol_z + U32 * (at.abs() + (at - lz).abs())).all())
    # H = ln Z + sum of w |d|: that sum's terms are off as the weights, by e^d's own error times |d|, and their
    # products and the quotient by Z by 4 u and Z's error
    tol_h = tol_z + (2 * e + 4 * U32) * mean + 2.25 * U32 * (square + mean * mean) + 2 * U32 * (lz + mean)
    assert bool(((ent - (lz + mean)).abs() <= tol_h).all())
    order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :5]
    assert torch.equal(ids.long(), order)
    at = d.gather(1, order)
    assert bool(((top - (at - lz[:, None])).abs() <= tol_z[:, None] + U32 * (at.abs() + lz[:, None])).all())
