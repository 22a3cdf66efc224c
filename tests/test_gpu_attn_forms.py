"""Every form that the row attention's launch chooses among - tiles of 32, 128
and 256 packed rows on the tensor cores, of 4, 8 and 64 in fp32, alone or with
others on an SM, with and without key shares - each named by the case, so that
a retuned launch cannot drop one unseen: whole rows against 64 bits, scores that
rise along the keys (each raise moves the running maximum and rescales what is
summed already) or fall, and non-finite values."""
import math

import pytest
import torch

import voxcuda as V
from rows_big import Big

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def streams(n, cap, rows):
    """Positions and counts of n streams: past the ring's end, close to it,
    short; the largest count first, and counts that end tiles early."""
    pos = [(3 * cap, cap - rows, cap + cap // 3, cap // 2)[s % 4] + s for s in range(n)]
    counts = [max(1, (rows, rows // 2, rows, rows - rows // 7)[s % 4]) for s in range(n)]
    return pos, counts


# (heads, KV heads, dim, ring, streams, rows, tree), the form: packed rows of a CTA, CTAs on an SM, shares; step of the heights
TENSOR = [
    ((8, 2, 128, 5200, 8, 1, None), (32, 2, 6), 64), ((8, 2, 64, 5200, 8, 1, None), (32, 2, 6), 64),
    ((32, 32, 64, 600, 16, 8, 3), (32, 2, 1), 64),
    ((32, 8, 128, 1600, 8, 30, None), (128, 2, 4), 64), ((32, 8, 128, 600, 8, 61, 3), (128, 2, 1), 64),
    ((32, 8, 128, 4100, 4, 400, None), (128, 2, 1), 256),   # (200 two-tile CTAs would be two whole waves)
    ((8, 2, 64, 1600, 8, 256, None), (128, 3, 3), 64), ((32, 32, 64, 1600, 8, 61, 4), (128, 3, 1), 128),
    ((32, 8, 128, 5200, 2, 520, None), (256, 1, 1), 320), ((32, 8, 128, 5200, 2, 256, 5), (256, 1, 2), 128),
    ((32, 8, 128, 1600, 16, 61, 3), (256, 1, 1), 128), ((8, 2, 128, 1600, 16, 256, None), (256, 1, 1), 128)]
CORES = [
    ((8, 2, 128, 5200, 24, 1, None), (4, 1, 2), 512), ((32, 32, 64, 600, 16, 2, None), (4, 4, 1), 64),
    ((8, 2, 128, 5200, 1, 30, 4), (8, 1, 4), 512), ((32, 32, 64, 1600, 16, 8, None), (8, 4, 1), 128),
    ((8, 2, 128, 1600, 8, 61, None), (64, 1, 2), 128), ((8, 2, 64, 1600, 8, 61, 3), (64, 1, 2), 128),
    ((32, 32, 64, 600, 16, 61, 3), (64, 2, 1), 64), ((8, 2, 64, 1600, 16, 128, None), (64, 2, 1), 128)]
FORMS = [(d, *f) for f in TENSOR for d in ("bf16", "fp16")] + [("fp32", *f) for f in CORES]


def make(dtype, size, step, **kw):
    heads, kv, dim, cap, n, rows, tree = size
    pos, counts = streams(n, cap, rows)
    return Big(dtype, heads, kv, dim, cap, kw.pop("n_sink", 4), pos, counts, tree=tree, seed=cap + rows, step=step, **kw)


@pytest.mark.parametrize("dtype,shape,form,step", FORMS)
@pytest.mark.parametrize("window", [0, 1])
def test_whole_rows(dtype, shape, form, step, window):
    # (a window of almost the ring keeps the form and masks rows of a tile differently)
    c = make(dtype, shape, step, window=window and shape[3] - 10)
    assert c.form(V) == form
    c.check(*c.run(V))


@pytest.mark.parametrize("dtype,shape,form,step", FORMS)
@pytest.mark.parametrize("order", ["rise", "fall"])
def test_scores_that_rise_and_fall(dtype, shape, form, step, order):
    c = make(dtype, shape, step, shape=order)
    assert c.form(V) == form
    out, lse = c.run(V)
    c.check(out, lse)
    again = c.run(V)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype,shape,form,step", FORMS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_value_stays_with_its_rows(dtype, shape, form, step, bad):
    c = make(dtype, shape, step)
    assert c.form(V) == form
    want, want_lse = c.run(V)
    p, n = c.positions[0], c.counts[0]
    j = p + n // 2              # a row's own key: the earlier rows do not see it, in a tree not all later ones
    from rows_ref import slot
    c.v[0, slot(j, c.cap, c.n_sink), :, 5:9] = bad
    out, lse = c.run(V)
    see = c.see[0][:, (c.key_pos[0] == j).nonzero().item()]
    assert bool(see.any()) and (n == 1 or not bool(see.all()))
    hit = torch.zeros(c.n, dtype=torch.bool, device="cuda")
    hit[:n] = see
    assert torch.equal(lse, want_lse) and torch.equal(out[~hit], want[~hit])
    assert not bool(torch.isfinite(out[hit][..., 5:9]).any())
    # (beside them, the other columns: as before)
    assert torch.equal(out[hit][..., :5], want[hit][..., :5]) and torch.equal(out[hit][..., 9:], want[hit][..., 9:])
