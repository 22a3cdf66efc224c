"""Attention over a paged cache in e4m3 in each of its forms, by name: tiles of 8
rows with one, two and three CTAs on an SM, of 16, of 128 and of 256, whole and in
shares, with and without masks inside a tile."""
import pytest
import torch

import voxcuda as V
from paged_ref import NAN8, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


# form (packed rows of a CTA, CTAs on an SM), in shares; heads, kv, dim, page; streams, rows, position
FORMS = [
    ((8, 2), False, 8, 2, 128, 16, 1, 1, 100), ((8, 2), True, 8, 2, 128, 64, 8, 8, 690), ((8, 2), False, 12, 12, 64, 16, 60, 1, 280),
    ((8, 2), True, 16, 4, 64, 32, 12, 8, 700), ((8, 1), True, 8, 2, 128, 32, 1, 6, 2990), ((8, 1), True, 8, 2, 64, 128, 3, 1, 4000),
    ((8, 3), False, 16, 16, 128, 16, 24, 1, 990), ((8, 3), False, 12, 12, 128, 16, 30, 1, 880), ((16, 2), True, 16, 4, 128, 32, 16, 4, 2900),
    ((128, 2), False, 8, 2, 128, 16, 1, 40, 250), ((128, 2), True, 2, 2, 64, 64, 1, 300, 900), ((128, 2), False, 8, 4, 128, 128, 4, 300, 10),
    ((256, 1), True, 8, 2, 128, 32, 1, 300, 2600), ((256, 1), False, 8, 4, 128, 64, 12, 300, 15), ((256, 1), True, 8, 8, 64, 32, 3, 200, 480)]


@pytest.mark.parametrize("form,shared,heads,kv,dim,page,streams,rows,pos", FORMS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_forms(form, shared, heads, kv, dim, page, streams, rows, pos, dtype):
    c = Case(dtype, heads, kv, dim, page, [max(0, pos - 7 * s) for s in range(streams)], [rows] * streams, seed=rows + pos)
    plan = V.attention_paged_plan(c.cache(V), c.rows(V), dtype, heads, 0, 0)
    assert plan[:2] == form and (plan[2] > 1) == shared, plan
    out, lse = c.run(V)
    torch.cuda.synchronize()
    c.check(out, lse, some=range(0, streams, max(1, streams // 4)))


@pytest.mark.parametrize("heads,kv,dim,page,streams,rows,pos", [
    (8, 2, 128, 16, 3, 2, 1500), (8, 2, 64, 32, 1, 4, 1500), (16, 4, 128, 16, 16, 4, 2900), (4, 4, 64, 16, 2, 700, 200),
    (8, 2, 128, 32, 2, 60, 300), (4, 2, 128, 16, 4, 700, 900), (8, 8, 64, 32, 8, 256, 100)])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (130, 4), (700, 70), (64, 129), (333, 1)])
def test_windows_in_forms(heads, kv, dim, page, streams, rows, pos, window, n_sink):
    """Rings of blocks between the sinks and windows that begin anywhere, tiles that leave blocks out."""
    c = Case("bf16", heads, kv, dim, page, [pos + 40 * s for s in range(streams)], [rows] * streams, window=window, n_sink=n_sink,
             seed=window)
    out, lse = c.run(V)
    torch.cuda.synchronize()
    c.check(out, lse, some=[0, streams - 1])


@pytest.mark.parametrize("heads,kv,dim,rows", [(4, 4, 64, 500), (8, 2, 128, 200), (4, 2, 128, 30), (4, 4, 64, 6)])
@pytest.mark.parametrize("step", [3.0, -3.0])
def test_scores_that_rise_and_fall_along_the_keys(heads, kv, dim, rows, step):
    """The maximum moves in block after block, or never again: keys whose first dim climbs, q that looks at it alone."""
    c = Case("bf16", heads, kv, dim, 16, [1200], [rows], seed=rows)
    c.q[:] = 0
    c.q[:, :, 0] = 1.0
    c.dq = c.q.cuda()
    for j in range(1200 + rows):
        g, at = c.table[0][j // 16], j % 16
        v = (j if step > 0 else 1200 + rows - j) / (1200 + rows) * 400
        c.pool.code[0][0, g, :, at, 0] = int(torch.tensor([v]).to(torch.float8_e4m3fn).view(torch.uint8))
    c.pool.scale[0].fill_(2.0 ** -1)
    c.pool.upload()
    out, lse = c.run(V, scale=abs(step) / 4)
    torch.cuda.synchronize()
    c.check(out, lse, scale=abs(step) / 4)


@pytest.mark.parametrize("heads,kv,dim,rows,pos", [(8, 2, 128, 1, 900), (8, 2, 128, 40, 900), (8, 2, 128, 200, 900), (4, 4, 64, 600, 900)])
def test_a_nan_outside_every_window(heads, kv, dim, rows, pos):
    """NaN behind the rows, before their windows, in pages that nobody follows and in their scales: `Case` puts it there;
    here it also stands in the first block that a window cuts, seen by some rows only."""
    c = Case("bf16", heads, kv, dim, 16, [pos], [rows], window=333, n_sink=3, seed=9)
    at = pos - 333 + max(1, rows // 2)
    c.pool.code[1][0, c.table[0][at // 16], 0, at % 16, 7] = NAN8
    c.pool.upload()
    out, lse = c.run(V)
    torch.cuda.synchronize()
    hit = torch.isnan(out).cpu()
    want = torch.zeros_like(hit)
    for i, r in enumerate(c.keys[0]):
        want[i, :heads // kv, 7] = at in r
    assert torch.equal(hit, want) and not bool(torch.isnan(lse).any())


@pytest.mark.parametrize("streams", [2, 31, 32, 33, 40])
def test_every_stream_once(streams):
    """Streams of many lengths, equal ones and ones that sit out among them, in the order of their reach or, beyond 32, in turn."""
    pos = [(s * 37) % 5 * 40 if s % 7 != 3 else -1 for s in range(streams)]
    counts = [(s * 13) % 50 + 1 if s % 5 else 0 for s in range(streams)]
    counts[-1] = 50
    c = Case("bf16", 4, 1, 64, 16, pos, counts, seed=streams, tail=1)
    assert V.attention_paged_plan(c.cache(V), c.rows(V), "bf16", 4, 0, 0)[0] > 0
    out, lse = c.run(V)
    torch.cuda.synchronize()
    c.check(out, lse)
