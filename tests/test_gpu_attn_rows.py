"""Window and tree attention over a cache slab against the definition in 64
bits.  Every slot that no row sees holds NaN, so a key too many shows at once;
the tolerances are derived in rows_ref.Case.check."""
import itertools
import math

import pytest

import voxcuda as V
from conftest import ROOT  # noqa: F401  (the import paths)
from rows_ref import Case

pytestmark = pytest.mark.gpu

HEADS = [(32, 8, 128), (4, 4, 64), (14, 2, 128), (10, 1, 64)]
TYPES_HEADS = list(itertools.product(["fp32", "bf16", "fp16"], HEADS))


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def go(c, **kw):
    import torch
    out, lse = c.run(V, **kw)
    torch.cuda.synchronize()
    c.check(out, lse, scale=kw.get("scale", 0.0), rounded_p=c.dtype != "fp32")


@pytest.mark.parametrize("dtype,heads", TYPES_HEADS)
def test_one_token_each(dtype, heads):
    # first token, a short stream, a wrapped ring, a stream that sits out
    go(Case(dtype, *heads, cap=70, n_sink=3, positions=[0, 5, 200, -1, 66], counts=[1] * 5, window=50, seed=1))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (1, 0), (1, 2), (33, 0), (64, 4), (1000, 5)])
def test_windows_and_sinks(dtype, window, n_sink):
    go(Case(dtype, 8, 2, 64, cap=130, n_sink=n_sink, positions=[0, 1, 64, 127, 128, 129, 5000], counts=[1] * 7, window=window,
            seed=2))


@pytest.mark.parametrize("dtype,heads", TYPES_HEADS)
def test_chunks_of_ragged_streams(dtype, heads):
    # rows from the very start, an empty stream, a wrap inside the chunk, rows behind the last stream
    go(Case(dtype, *heads, cap=150, n_sink=4, positions=[0, 40, 140, 9], counts=[37, 0, 33, 1], window=45, seed=3, tail=2))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,pos,cap,window,n_sink", [
    (150, 0, 200, 0, 0), (129, 300, 260, 128, 1), (65, 64, 129, 64, 0), (64, 63, 500, 17, 9), (200, 7, 200, 0, 0)])
def test_long_chunks(dtype, rows, pos, cap, window, n_sink):
    go(Case(dtype, 2, 2, 64, cap=cap, n_sink=n_sink, positions=[pos], counts=[rows], window=window, seed=4))


@pytest.mark.parametrize("dtype,heads", TYPES_HEADS)
def test_trees(dtype, heads):
    go(Case(dtype, *heads, cap=90, n_sink=2, positions=[0, 30, 300, 88], counts=[13, 8, 21, 2], window=0, seed=5, tree=4))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (3, 0), (3, 2), (40, 5)])
def test_trees_with_windows(dtype, window, n_sink):
    # deep, narrow trees: the window cuts ancestors too, unless they are sinks
    go(Case(dtype, 4, 2, 64, cap=70, n_sink=n_sink, positions=[0, 1, 100], counts=[24, 9, 30], window=window, seed=6, tree=2))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_the_largest_tree(dtype):
    go(Case(dtype, 2, 1, 64, cap=300, n_sink=0, positions=[70], counts=[256], window=0, seed=7, tree=9))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_a_chain_is_a_chunk(dtype):
    # the window's lower edge starts a tree's key tiles elsewhere, so both are
    # held to the definition, not to each other's last bit
    import torch
    c = Case(dtype, 8, 2, 128, cap=400, n_sink=1, positions=[333, 20], counts=[40, 70], window=100, seed=8)
    go(c)
    c.dparent = torch.cat([torch.arange(n) - 1 for n in c.counts]).to(torch.int32).cuda()
    go(c)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["heads", "streams_last"])
def test_strides_and_layers(dtype, layout):
    go(Case(dtype, 8, 4, 64, cap=40, n_sink=2, positions=[35, 90], counts=[5, 9], window=20, seed=9, layers=3, layer=2,
            layout=layout))
    go(Case(dtype, 8, 4, 128, cap=40, n_sink=2, positions=[35, 90], counts=[1, 1], window=20, seed=9, layers=3, layer=1,
            layout=layout))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("scale", [0.25, -0.1, 3.0])
def test_scales(dtype, scale):
    # 3.0: one key takes nearly all the weight
    go(Case(dtype, 4, 1, 64, cap=64, n_sink=0, positions=[50, 63], counts=[2, 7], window=0, seed=10), scale=scale)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tree", [None, 3])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_key_stays_with_its_rows(dtype, tree, bad):
    """A NaN or infinite K and V row reaches the rows that see it, no others."""
    import torch
    c = Case(dtype, 8, 2, 128, cap=200, n_sink=2, positions=[70], counts=[30], window=25, seed=11, tree=tree)
    want, want_lse = c.run(V)
    j = 80                      # a drafted row, or a key of the chunk
    c.dv[0, 0, 80, :, 5:9] = bad
    got, got_lse = c.run(V)
    torch.cuda.synchronize()
    see = torch.tensor([j in keys for keys in c.keys[0]]).cuda()
    assert 0 < int(see.sum()) < len(see)
    assert torch.equal(got[~see], want[~see]) and torch.equal(got_lse, want_lse)
    assert not bool(torch.isfinite(got[see][..., 5:9]).any())
    assert torch.equal(got[see][..., 9:], want[see][..., 9:])
    c.dk[0, 0, 80] = math.nan
    got, got_lse = c.run(V)
    torch.cuda.synchronize()
    assert torch.equal(got[~see], want[~see]) and torch.equal(got_lse[~see], want_lse[~see])
    assert bool(torch.isnan(got[see]).all()) and bool(torch.isnan(got_lse[see]).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 12])
def test_rows_without_weight(dtype, rows):
    """Scores of -inf throughout: zeros, and lse -inf."""
    import torch
    c = Case(dtype, 4, 2, 64, cap=64, n_sink=0, positions=[20], counts=[rows], window=0, seed=12)
    c.dk.fill_(math.inf)
    c.dq.fill_(0.0)
    c.dq[..., 0] = -1.0
    c.dk[..., 1:] = 0.0
    out, lse = c.run(V)
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads", [(8, 2, 128), (8, 8, 64), (7, 1, 64), (20, 1, 128)])
@pytest.mark.parametrize("rows,tree", [(1, None), (9, None), (9, 3), (30, None)])
def test_long_contexts(dtype, heads, rows, tree):
    # few tiles, many keys: every kernel's shares and their merge
    go(Case(dtype, *heads, cap=2500, n_sink=3, positions=[7000], counts=[rows], window=2400, seed=20, tree=tree))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,tree", [(1, None), (20, None), (20, 3), (100, None)])
@pytest.mark.parametrize("n_sink", [0, 100])
def test_the_largest_windows_are_no_limit(dtype, rows, tree, n_sink):
    import torch

    def run(window):
        c = Case(dtype, 8, 4, 64, cap=300, n_sink=n_sink, positions=[3, 700], counts=[rows, rows], window=window, seed=21, tree=tree)
        got = c.run(V)
        torch.cuda.synchronize()
        return got
    want = run(0)
    for window in (300 - n_sink, 2 ** 31 - 1):
        for a, b in zip(run(window), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kinds", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp16")])
def test_two_streams_at_once(kinds):
    """Calls under way on two streams: each as by itself, again and again."""
    import torch
    cases = [Case(d, 8, 2, 128, cap=900, n_sink=0, positions=[800] * 4, counts=[n] * 4, window=0, seed=22 + i)
             for i, (d, n) in enumerate(zip(kinds, (70, 9)))]
    want = [c.run(V) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[(torch.full_like(c.dq, 7.0), torch.full_like(w[1], 7.0)) for _ in range(10)] for c, w in zip(cases, want)]
    torch.cuda.synchronize()
    for turn in range(10):
        for c, st, o in zip(cases, streams, outs):
            V.attention_window_dev(c.cache(V), 0, c.rows(V), c.dq.data_ptr(), c.heads, 0, 0.0, o[turn][0].data_ptr(),
                                   o[turn][1].data_ptr(), st.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        for got in o:
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_the_first_call_may_be_captured():
    """Every operator's first call in a process, inside a capture."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = ["tests", "voxtral.c_b200"]
import voxcuda as V
from rows_ref import Case
V.init()
cases = [Case(d, *h, cap=90, n_sink=1, positions=[40, 60], counts=n, window=0, seed=1, tree=t)
         for d in ("fp32", "bf16") for h in ((8, 2, 64), (8, 2, 128)) for n in ([1, 1], [3, 9], [30, 20], [64, 70]) for t in (None, 3)]
x = torch.randn(3, 5000, device="cuda")
tok, lp = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
outs = [(torch.empty_like(c.dq), torch.empty(c.dq.shape[:2], device="cuda")) for c in cases]
k = torch.randn(2, 3, 20, 2, 64, device="cuda")
kv = V.KvCache(k.data_ptr(), k.clone().data_ptr(), "fp32", 2, 3, 20, 2, 64)
pos, path = torch.full((3,), 5, dtype=torch.int32, device="cuda"), torch.ones(3, 1, dtype=torch.int32, device="cuda")
qkv, q = torch.randn(3, 8, 64, device="cuda"), torch.empty(3, 4, 64, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    V.token_logprobs_dev(x.data_ptr(), "fp32", 3, 5000, 0, tok.data_ptr(), 0, lp.data_ptr(), None, None, None, st)
    V.rope_append_dev(kv, 0, V.Rows(pos.data_ptr(), n_rows=3), qkv.data_ptr(), "fp32", 4, 0, None, None, 0.0, 1e4, q.data_ptr(), st)
    V.kv_commit_dev(kv, pos.data_ptr(), path.data_ptr(), 1, path.data_ptr(), 1, None, st)
    V.kv_fork_dev(kv, [0], [1], pos.data_ptr(), st)
    for c, (o, l) in zip(cases, outs):
        call = V.attention_window_dev if c.dparent is None else V.attention_tree_dev
        call(c.cache(V), 0, c.rows(V), c.dq.data_ptr(), c.heads, 0, 0.0, o.data_ptr(), l.data_ptr(), st)
g.replay()
torch.cuda.synchronize()
for c, (o, l) in zip(cases, outs):
    c.check(o, l, rounded_p=c.dtype != "fp32")
assert abs(float(lp[0]) - float(torch.log_softmax(x[0].double(), 0)[0])) < 1e-4
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_device_arrays_are_clamped():
    """Row ranges beyond the buffers and parents out of order fault nothing:
    ranges are cut, such parents count as none."""
    import torch
    c = Case("fp32", 4, 2, 64, cap=64, n_sink=0, positions=[20, 30], counts=[4, 4], window=0, seed=13, tree=2)
    c.dstart.copy_(torch.tensor([0, 4, 4000], dtype=torch.int32))
    bad = c.dparent.clone()
    bad[1], bad[2], bad[5] = 3, 2, -77
    c.dparent = bad
    out, _ = c.run(V)
    for s, cut in ((0, [-1, -1, -1]), (1, None)):
        fixed = [p if 0 <= p < i else -1 for i, p in enumerate(bad[4 * s:4 * s + 4].tolist())]
        c.parents[s] = fixed
    from rows_ref import visible
    c.keys = [[visible(p, 4, i, 64, 0, 0, c.parents[s]) for i in range(4)] for s, p in enumerate(c.positions)]
    _, lse = c.run(V)
    torch.cuda.synchronize()
    c.check(out, lse)


def test_one_row_each_without_ranges():
    import torch
    c = Case("bf16", 8, 2, 64, cap=64, n_sink=1, positions=[20, 0, 99], counts=[1, 1, 1], window=30, seed=14)
    rows = V.Rows(c.dpos.data_ptr(), n_rows=3, max_rows=1)
    out, lse = torch.empty_like(c.dq), torch.empty(3, 8, device="cuda")
    V.attention_window_dev(c.cache(V), 0, rows, c.dq.data_ptr(), 8, 30, 0.0, out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    c.check(out, lse, rounded_p=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 1], [9, 30]])
def test_out_may_be_q(dtype, counts):
    import torch
    c = Case(dtype, 8, 2, 128, cap=300, n_sink=1, positions=[250, 100], counts=counts, window=0, seed=15)
    want, _ = c.run(V)
    c.run(V, out=c.dq)
    torch.cuda.synchronize()
    assert torch.equal(want, c.dq)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tree", [None, 3])
def test_captured_and_replayed(dtype, tree):
    """A captured call reads positions and trees when it is replayed; two
    graphs and an eager call on other streams do not disturb each other."""
    import torch
    cs = [Case(dtype, 8, 2, 128, cap=500, n_sink=1, positions=[400, 77 + s], counts=[5, 6], window=300, seed=16 + s, tree=tree)
          for s in range(3)]
    want = [c.run(V) for c in cs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cs]
    for c, st in zip(cs[:2], streams):
        out, lse = torch.zeros_like(c.dq), torch.zeros(c.dq.shape[:2], device="cuda")
        g = torch.cuda.CUDAGraph()
        keep = c.dpos.clone()
        c.dpos.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            call = V.attention_tree_dev if tree else V.attention_window_dev
            call(c.cache(V), 0, c.rows(V), c.dq.data_ptr(), 8, 300, 0.0, out.data_ptr(), lse.data_ptr(),
                 torch.cuda.current_stream().cuda_stream)
        c.dpos.copy_(keep)
        graphs.append(g)
        outs.append((out, lse))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        last = cs[2].run(V, stream=streams[2].cuda_stream)
    torch.cuda.synchronize()
    for (a, la), (b, lb) in zip(outs + [last], want):
        assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 20])
def test_offsets_beyond_32_bits(dtype, rows):
    """The second stream's slab starts 2^32 elements into the cache."""
    import torch
    c = Case(dtype, 4, 2, 64, cap=64, n_sink=1, positions=[30, 70], counts=[rows, rows], window=0, seed=17)
    far = (1 << 32) + 1024
    big = torch.empty(2 * 64 * 128 + far, dtype=c.dk.dtype, device="cuda")
    n = 64 * 2 * 64
    cache = c.cache(V)
    for s in range(2):
        big[s * far:s * far + n] = c.dk[0, s].reshape(-1)
        big[s * far + n:s * far + 2 * n] = c.dv[0, s].reshape(-1)
    cache.k, cache.v = big.data_ptr(), big.data_ptr() + n * big.element_size()
    cache.stream_stride = cache.layer_stride = far
    out, lse = torch.full_like(c.dq, 7.0), torch.empty(c.dq.shape[:2], device="cuda")
    V.attention_window_dev(cache, 0, c.rows(V), c.dq.data_ptr(), 4, 0, 0.0, out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    c.check(out, lse, rounded_p=dtype != "fp32")


def test_a_long_stream_repeats_bit_for_bit():
    """Many shares of one row's keys, merged in a fixed order."""
    import torch
    c = Case("fp32", 32, 8, 128, cap=2100, n_sink=4, positions=[100000], counts=[1], window=2048, seed=18)
    a, la = c.run(V)
    for _ in range(10):
        b, lb = c.run(V)
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.equal(la, lb)
    c.check(a, la)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_positions_up_to_the_limit(dtype, rows):
    top = (1 << 30) - rows
    c = Case.__new__(Case)
    import rows_ref
    # the same residues as a short stream's, far out: only the ring's keys are visible
    old = rows_ref.visible
    rows_ref.visible = lambda pos, n, i, cap, sink, window, parent=None: (
        list(range(sink)) + list(range(max(sink, pos + n - (cap - sink), pos + i - window + 1 if window else 0), pos + i + 1)))
    try:
        c.__init__(dtype, 4, 2, 64, cap=90, n_sink=3, positions=[top], counts=[rows], window=45, seed=19)
    finally:
        rows_ref.visible = old
    go(c)
