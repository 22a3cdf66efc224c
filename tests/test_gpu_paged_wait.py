"""A wait of the paged attention that runs out: the rows are NaN and the thread is
told, once.  The wait is one that a diagnostic call makes for what never comes."""
import pytest
import torch

import voxcuda as V
from paged_ref import Case

pytestmark = pytest.mark.gpu

# one tile, two tiles, in shares
CASES = [dict(heads=8, kv=2, dim=128, page=16, positions=[200, -1, 3], counts=[40, 2, 33], tail=2),
         dict(heads=8, kv=4, dim=128, page=64, positions=[15 + i for i in range(12)], counts=[300] * 12),
         dict(heads=8, kv=2, dim=128, page=32, positions=[2600], counts=[300])]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def held_up(c, out, lse, wait_ms=20, stream=V.STREAM_LEGACY):
    return V.lib().vox_cuda_selftest_attention_paged_timeout(c.cache(V), c.layer, c.rows(V), c.dq.data_ptr(), V.TYPES[c.dtype], c.heads,
                                                             out.data_ptr(), lse.data_ptr(), wait_ms, stream)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kw", CASES)
def test_void_rows_are_nan_and_the_thread_is_told(dtype, kw):
    c = Case(dtype, seed=31, **kw)
    want, want_lse = c.run(V)
    out, lse = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    assert held_up(c, out, lse) == V.OK
    torch.cuda.synchronize()
    for s, (p, n) in enumerate(zip(c.positions, c.counts)):
        a, b = c.start[s], c.start[s + 1]
        void = (out[a:b] == 7.0) & (p < 0) | torch.isnan(out[a:b]) & (p >= 0)
        assert bool(void.all()) and (p < 0 or bool(torch.isnan(lse[a:b]).all())), s
    assert bool((out[c.n:] == 7.0).all())
    out.fill_(7.0)
    with pytest.raises(V.VoxCudaError, match="timed out"):
        c.run(V, out=out)
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())          # not enqueued
    got, got_lse = c.run(V)                  # once
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


def test_few_rows_have_no_waits():
    c = Case("bf16", 8, 2, 128, 16, [300], [1], seed=5)
    assert held_up(c, c.dq, torch.zeros(1, 8).cuda()) == V.ERR_ARG and "no waits" in V.last_error()
    big = Case("bf16", 8, 2, 128, 16, [300], [100], seed=5)
    for ms in (0, 10001):
        assert held_up(big, torch.empty_like(big.dq), torch.zeros(100, 8).cuda(), ms) == V.ERR_ARG
