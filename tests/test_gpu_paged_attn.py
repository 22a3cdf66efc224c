"""Attention over a paged cache in e4m3 against its definition in 64 bits."""
import math

import pytest
import torch

import voxcuda as V
from paged_ref import NAN8, Case

pytestmark = pytest.mark.gpu

HEADS = [(32, 8, 128), (32, 32, 64), (28, 4, 128), (16, 2, 64), (6, 6, 128), (10, 1, 64), (64, 1, 128)]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def check(case, **kw):
    out, lse = case.run(V, **kw)
    torch.cuda.synchronize()
    case.check(out, lse, **{k: v for k, v in kw.items() if k == "scale"})
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_one_token(dtype, heads, kv, dim, page):
    """Lengths around tiles and pages; a stream that sits out, one without rows, rows behind the last stream."""
    check(Case(dtype, heads, kv, dim, page, [0, 1, 15, -1, 16, 130, 257, 63], [1, 1, 1, 1, 1, 1, 1, 0], tail=2, seed=page))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("counts", [[2, 1, 3], [9, 4, 16], [37, 40, 1], [130, 0, 65]])
def test_chunks(dtype, heads, kv, dim, counts):
    """Causal rows: from the start, inside a page, over several pages."""
    check(Case(dtype, heads, kv, dim, 32, [0, 45, 200], counts, seed=counts[0], tail=1))


@pytest.mark.parametrize("heads,kv,dim", HEADS[:4])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (16, 0), (50, 4), (64, 1), (1, 7), (90, 33), (1000, 4), (130, 200)])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [7, 70, 3, 20], [150, 1, 129, 64]])
def test_windows_and_sinks(heads, kv, dim, window, n_sink, counts):
    check(Case("bf16", heads, kv, dim, 16, [0, 31, 300, 110], counts, window=window, n_sink=n_sink, seed=window))


@pytest.mark.parametrize("layout", ["heads", "slots", "pages_last"])
@pytest.mark.parametrize("counts", [[1, 1], [66, 17]])
def test_layers_and_strides(layout, counts):
    check(Case("fp16", 8, 2, 64, 16, [70, 129], counts, layers=3, layer=2, layout=layout, seed=5))
    check(Case("bf16", 8, 2, 128, 64, [70, 129], counts, layers=3, layer=1, layout=layout, seed=6))


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 3, 140]])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (40, 3)])
def test_pages_that_are_not_there(counts, window, n_sink):
    """Their keys are left out; a row that has no other sees nothing."""
    lost = [(0, 0), (0, 2), (1, 0), (1, 1), (1, 2), (1, 3), (2, 4)]
    check(Case("bf16", 8, 2, 128, 16, [40, 20, 90], counts, window=window, n_sink=n_sink, lost=lost, seed=8))


@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [5, 3, 1, 9, 2], [100, 80, 33, 1, 64]])
def test_long(counts):
    """Contexts that several CTAs share."""
    check(Case("bf16", 8, 2, 128, 64, [3000, 1111, 4097, 64, 2047], counts, seed=9))
    check(Case("fp16", 4, 4, 64, 16, [3000, 1111, 4097, 64, 2047], counts, seed=10, window=900, n_sink=5))


def test_row_start_left_out():
    """One row for each stream."""
    c = Case("bf16", 8, 2, 128, 16, [40, 20, 90], [1, 1, 1], seed=11)
    out, lse = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    V.attention_paged_dev(c.cache(V), 0, V.Rows(c.dpos.data_ptr(), None, None, 3, 1), c.dq.data_ptr(), "bf16", 8, 0, 0, 0.0,
                          out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    c.check(out, lse)


@pytest.mark.parametrize("scale", [0.25, 1e-4, -0.3])
@pytest.mark.parametrize("counts", [[1, 1], [70, 9]])
def test_scales(scale, counts):
    check(Case("bf16", 8, 2, 128, 32, [100, 333], counts, seed=12), scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("counts", [[1, 1], [6, 2], [70, 9]])
def test_sharp_and_flat_scores(dtype, counts):
    """One key far above the others, and rows of zeros."""
    c = Case(dtype, 8, 2, 128, 32, [700, 333], counts, seed=13, scale_q=30.0)
    check(c)
    c = Case(dtype, 8, 2, 128, 32, [700, 333], counts, seed=14, scale_q=0.0)
    check(c)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("counts", [[1, 1], [12, 2], [70, 9]])
def test_scales_far_apart(dtype, counts):
    """Pages under scales from 2^-24 to 2^4: small numbers beside large ones keep their place."""
    check(Case(dtype, 4, 2, 64, 16, [700, 333], counts, seed=15, exps=(-24, 5), scale_q=0.02))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("amount", [2.0 ** -20, 2.0 ** 12])   # (2^14 would leave fp16)
def test_small_and_large_queries(dtype, amount):
    check(Case(dtype, 4, 2, 64, 16, [300, 33], [3, 70], seed=16, scale_q=amount), scale=0.125 / amount)


@pytest.mark.parametrize("counts", [[1], [5], [80], [200]])
def test_many_small_weights(counts):
    """One key takes nearly all the weight and has V = 0: what comes out is the sum of many keys of 2^-19 each."""
    c = Case("bf16", 4, 1, 64, 16, [6000], counts, seed=17, scale_q=0.0)
    c.q[:, :, 0] = 1.0
    c.dq = c.q.cuda()
    code, scale = c.pool.code, c.pool.scale
    code[0].zero_()
    code[1].fill_(0x38)                       # 1.0
    scale[0].fill_(1.0), scale[1].fill_(1.0)
    first = c.table[0][0]
    code[0][0, first, 0, 0, 0] = 0x55         # 13: a score of 13 (19 times ln 2, near enough)
    code[1][0, first, 0, 0] = 0
    c.pool.upload()
    check(c, scale=1.0)


@pytest.mark.parametrize("rows", [3, 20, 150])
def test_a_nan_is_seen_by_those_who_see_it(rows):
    """A V that is NaN in one dim of one position: rows before it keep their numbers; K: the whole row."""
    for which in (0, 1):
        c = Case("bf16", 4, 2, 64, 16, [50], [rows], seed=18)
        at = 50 + rows // 2
        g = c.table[0][at // 16]
        clean = [x.clone() for x in c.pool.code]
        c.pool.code[which][0, g, 1, at % 16, 5] = NAN8
        c.pool.upload()
        out, lse = c.run(V)
        torch.cuda.synchronize()
        hit = torch.isnan(out).cpu()
        want = torch.zeros_like(hit)
        if which:
            want[rows // 2:, 2:, 5] = True
        else:
            want[rows // 2:, 2:] = True
            assert torch.equal(torch.isnan(lse).cpu(), want.any(-1))
        assert torch.equal(hit, want), which
        c.pool.code = clean
        c.pool.upload()
        good, lse2 = c.run(V)
        torch.cuda.synchronize()
        assert bool(((good == out) | torch.isnan(out)).all())
        c.check(good, lse2)


def test_scores_of_minus_infinity():
    """q of -inf: no weight at all gives zeros and lse -inf."""
    c = Case("bf16", 4, 2, 64, 16, [50, 9], [3, 70], seed=19)
    c.pool.code[0].fill_(0x38)
    c.dq.fill_(0.0)
    c.dq[:, :, 0] = -math.inf
    c.pool.scale[0].fill_(1.0)
    c.pool.upload()
    out, lse = c.run(V)
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("counts", [[1, 1], [66, 17], [300, 2]])
def test_out_may_be_q(counts):
    c = Case("bf16", 8, 2, 128, 16, [700, 129], counts, seed=20)
    want, lse = c.run(V)
    q = c.dq.clone()
    c.dq = q
    out, lse2 = c.run(V, out=q)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, lse2)


@pytest.mark.parametrize("counts", [[1, 1, 1], [20, 3, 6], [200, 20, 90]])
def test_no_lse_and_repeats(counts):
    """Without lse; the same bits every time."""
    c = Case("bf16", 32, 8, 128, 32, [1500, 700, 129], counts, seed=21)
    want, _ = c.run(V)
    for _ in range(3):
        out = torch.full_like(c.dq, 7.0)
        V.attention_paged_dev(c.cache(V), 0, c.rows(V), c.dq.data_ptr(), "bf16", 32, 0, 0, 0.0, out.data_ptr(), None, V.STREAM_LEGACY)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_rows_beyond_the_table_are_left_out():
    """A stream whose table ends: rows that fit are computed, later ones stay as they were."""
    c = Case("bf16", 4, 2, 64, 16, [40], [30], seed=22)
    want, lse0 = c.run(V)
    short = c.dtable[:, :4].contiguous()      # 64 positions: 24 rows
    out, lse = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    V.attention_paged_dev(c.pool.cache(V, short), 0, c.rows(V), c.dq.data_ptr(), "bf16", 4, 0, 0, 0.0, out.data_ptr(), lse.data_ptr(),
                          V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(out[:24], want[:24]) and torch.equal(lse[:24], lse0[:24])
    assert bool((out[24:] == 7.0).all()) and bool((lse[24:] == 7.0).all())


def test_streams_share_pages():
    """A common beginning: the same pages in two tables, and twice in one."""
    c = Case("bf16", 8, 2, 128, 16, [100, 100, 40], [1, 1, 1], seed=23)
    c.table[1][:6] = c.table[0][:6]
    c.table[2][1] = c.table[2][0]
    c.dtable = torch.tensor(c.table, dtype=torch.int32).cuda()
    check(c)


def test_two_streams_at_once_and_a_graph():
    """Calls on two CUDA streams; a captured call replayed over other positions and tables."""
    a, b = Case("bf16", 32, 8, 128, 16, [900, 50], [20, 3], seed=24), Case("fp16", 16, 2, 64, 64, [800, 1], [1, 1], seed=25)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = [c.run(V, stream=s.cuda_stream) for _ in range(5) for c, s in ((a, s1), (b, s2))]
    torch.cuda.synchronize()
    for n, (out, lse) in enumerate(got):
        (a, b)[n % 2].check(out, lse)
    c = Case("bf16", 32, 8, 128, 16, [300, 10], [3, 2], seed=26)
    d = Case("bf16", 32, 8, 128, 16, [200, 250], [2, 3], seed=27)
    cache, rows = c.cache(V), c.rows(V)
    out, lse = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        V.attention_paged_dev(cache, 0, rows, c.dq.data_ptr(), "bf16", 32, 0, 0, 0.0, out.data_ptr(), lse.data_ptr(),
                              torch.cuda.current_stream().cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    c.check(out, lse)
    # the second case's streams in the first one's buffers: its pages behind the first one's
    grown = min(c.pool.pages, d.pool.pages)
    assert d.pool.pages >= grown and d.dq.shape == c.dq.shape
    keep = [t.clone() for t in (c.dpos, c.dstart)]
    c.dpos.copy_(d.dpos - 150)
    c.dstart.copy_(d.dstart)
    e = Case("bf16", 32, 8, 128, 16, [300, 10], [3, 2], seed=26)
    g.replay()
    eager, lse_e = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    V.attention_paged_dev(cache, 0, rows, c.dq.data_ptr(), "bf16", 32, 0, 0, 0.0, eager.data_ptr(), lse_e.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    same = (out == eager) | (torch.isnan(out) & torch.isnan(eager))
    assert bool(same.all()) and not bool((out == e.run(V)[0]).all())
    del keep
