"""A wait of the row attention that runs out: the rows that it held up are NaN,
the thread whose call it was is told, others are not disturbed.  The self-test
call waits, its work done, for what never comes: the GPU does not fault."""
import threading

import pytest
import torch

import voxcuda as V
from rows_ref import Case

pytestmark = pytest.mark.gpu

# one token (shares of a long stream), a chunk, a tile of 128 rows, two tiles' worth: heads of 64 and 128
CASES = [dict(heads=8, kv_heads=2, dim=128, cap=2100, n_sink=2, positions=[5000, 30], counts=[1, 1]),
         dict(heads=8, kv_heads=2, dim=64, cap=700, n_sink=0, positions=[600, 20], counts=[40, 17], tail=3),
         dict(heads=8, kv_heads=2, dim=128, cap=400, n_sink=0, positions=[300, -1], counts=[70, 5])]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def held_up(c, out, lse, stream=V.STREAM_LEGACY, wait_ms=20):
    return V.lib().vox_cuda_selftest_attention_timeout(c.cache(V), c.layer, c.rows(V), c.dq.data_ptr(), c.heads, out.data_ptr(),
                                                       lse.data_ptr(), wait_ms, stream)


def buffers(c):
    return torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")


def all_void(c, out, lse):
    for s, (p, n) in enumerate(zip(c.positions, c.counts)):
        a, b = c.start[s], c.start[s + 1]
        if p < 0:
            assert bool((out[a:b] == 7.0).all()) and bool((lse[a:b] == 7.0).all())
        else:
            assert bool(torch.isnan(out[a:b]).all()) and bool(torch.isnan(lse[a:b]).all())
    assert bool((out[c.n:] == 7.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kw", CASES)
def test_void_rows_are_nan_and_the_thread_is_told(dtype, kw):
    c = Case(dtype, window=0, seed=31, **kw)
    want, want_lse = c.run(V)
    out, lse = buffers(c)
    assert held_up(c, out, lse) == V.OK
    torch.cuda.synchronize()
    all_void(c, out, lse)
    seen = {}

    def other():
        V.init()
        seen["got"] = c.run(V)   # raises if it is told
        torch.cuda.synchronize()
    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert torch.equal(seen["got"][0], want) and torch.equal(seen["got"][1], want_lse)
    out, lse = buffers(c)
    with pytest.raises(V.VoxCudaError, match="timed out"):
        c.run(V, out=out)
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())          # not enqueued
    got, got_lse = c.run(V)                  # once
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


def test_a_replayed_graph_says_it_in_its_rows():
    c = Case("bf16", window=0, seed=32, **CASES[0])
    out, lse = buffers(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert held_up(c, out, lse, torch.cuda.current_stream().cuda_stream) == V.OK
    for _ in range(2):
        out.fill_(7.0), lse.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        all_void(c, out, lse)
    with pytest.raises(V.VoxCudaError, match="timed out"):
        c.run(V)
    c.run(V)
    torch.cuda.synchronize()
