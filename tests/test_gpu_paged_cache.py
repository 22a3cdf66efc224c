"""Rotary append to a paged cache in e4m3, copies of pages, and the operators
over it as they are used together, against the definitions in 64 bits."""
import math

import pytest
import torch

import voxcuda as V
from paged_ref import NAN8, Case, Pool, from_e4m3, scale_for, tables, to_e4m3
from rows_ref import TORCH, U32, half_step

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-5, 1.0e6


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def ptr(t):
    return None if t is None else t.data_ptr()


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def starts(counts):
    return [sum(counts[:s]) for s in range(len(counts) + 1)]


def rotate(x, p, theta):
    """One head's interleaved pairs turned by p * theta^(-2d / dim), 64 bits."""
    dim = x.shape[-1]
    a = torch.tensor([p * theta ** (-2.0 * d / dim) for d in range(dim // 2)], dtype=torch.float64)
    return torch.stack((x[..., 0::2] * a.cos() - x[..., 1::2] * a.sin(), x[..., 0::2] * a.sin() + x[..., 1::2] * a.cos()), -1).flatten(-2)


class Calls:
    """A pool, its streams' tables, and appends of qkv rows to them."""

    def __init__(self, kv, dim, page, widths, seed=0, layers=1, layer=0, layout="heads", lost=()):
        pages = sum(widths) + 3
        self.pool = Pool(layers, pages, page, kv, dim, seed, layout)
        self.table = tables(widths, pages, seed, spare=0)
        for s, i in lost:
            self.table[s][i] = (-1, pages, 1 << 30)[i % 3]
        self.pool.upload()
        self.dtable, self.layer, self.kv, self.dim, self.page = ints(self.table), layer, kv, dim, page

    def append(self, heads, positions, counts, qkv, q_type, theta=THETA, gq=None, gk=None, most=None, stream=None, q=None):
        """qkv: [rows][heads + 2 kv][dim] on the GPU, rows as far apart as its stride tells."""
        src = {v: k for k, v in TORCH.items()}[qkv.dtype]
        self.hold = (ints(positions), ints(starts(counts)))
        q = torch.full((qkv.shape[0], heads, self.dim), 7.0, dtype=TORCH[q_type], device="cuda") if q is None else q
        r = V.Rows(ptr(self.hold[0]), ptr(self.hold[1]), None, qkv.shape[0], most or max(max(counts), 1))
        V.rope_append_paged_dev(self.pool.cache(V, self.dtable), self.layer, r, ptr(qkv), src, heads, qkv.stride(0), ptr(gq), ptr(gk),
                                EPS, theta, ptr(q), q_type, V.STREAM_LEGACY if stream is None else stream)
        return q


def expect(c, was, which, positions, counts, x, most=None):
    """What the pool's K (0) or V (1) holds after an append of x [rows][kv][dim], 64 bits, to `was`: (codes, scales),
    and for every page and head written by the call the values before they are rounded."""
    code, scale = was[0].clone(), was[1].clone()
    start, plain = starts(counts), {}
    for s, (p, n) in enumerate(zip(positions, counts)):
        n = 0 if p < 0 else max(0, min(n, len(c.table[s]) * c.page - p, most or n))
        for i in range(p // c.page, (p + n - 1) // c.page + 1) if n else []:
            g = c.table[s][i]
            if not 0 <= g < c.pool.pages:
                continue
            a, b = max(p, i * c.page), min(p + n, (i + 1) * c.page)
            for h in range(c.kv):
                rows = x[start[s] + a - p:start[s] + b - p, h]
                fin = rows[torch.isfinite(rows)].abs()
                need = scale_for(float(fin.max()) if fin.numel() else 0.0)
                old, lo = float(scale[c.layer, g, h]), a - i * c.page
                now = need if lo == 0 else max(old, need)
                if lo and now != old:
                    code[c.layer, g, h, :lo] = to_e4m3(from_e4m3(code[c.layer, g, h, :lo].contiguous()) * (old / now))
                code[c.layer, g, h, lo:lo + b - a] = to_e4m3(rows / now)
                scale[c.layer, g, h] = now
                plain[g, h] = (lo, rows / now)
    return code, scale, plain


@pytest.mark.parametrize("src,q_type", [("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (3, 3, 64), (7, 1, 64)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("layout", ["heads", "slots", "pages_last"])
def test_append_rounds_as_defined(src, q_type, heads, kv, dim, page, layout):
    """Without norm and rotation every bit is known: scales, ties to even, earlier slots under a grown scale, slots that
    stay as they were.  Three calls: from the start, then rows of other sizes."""
    c = Calls(kv, dim, page, [4, 4, 2, 3, 1], seed=page, layers=2, layer=1, layout=layout)
    g = torch.Generator().manual_seed(page + dim)
    pos, width = [0, 0, -1, 5, 0], heads + 2 * kv
    for turn, (counts, size) in enumerate([([3, page, 4, 1, 0], 1.0), ([1, 1, 0, page + 3, 1], 300.0), ([2 * page, 5, 1, 2, 9], 0.01)]):
        wide = (torch.randn(sum(counts) + 2, width * dim + 16, generator=g) * size).to(TORCH[src]).cuda()
        qkv = wide[:, :width * dim].unflatten(1, (width, dim))
        was = [c.pool.held(i) for i in (0, 1)]
        q = c.append(heads, pos, counts, qkv, q_type, theta=0.0)
        torch.cuda.synchronize()
        x = qkv.double().cpu()
        for which, rows in ((0, x[:, heads:heads + kv]), (1, x[:, heads + kv:])):
            code, scale, _ = expect(c, was[which], which, pos, counts, rows)
            got, got_scale = c.pool.held(which)
            assert torch.equal(got_scale, scale), (turn, which)
            assert torch.equal(got, code), (turn, which, int((got != code).sum()))
        at = starts(counts)
        for s, p in enumerate(pos):
            want = torch.full_like(q[at[s]:at[s + 1]], 7.0) if p < 0 else qkv[at[s]:at[s + 1], :heads].to(TORCH[q_type])
            assert torch.equal(q[at[s]:at[s + 1]], want)
        assert bool((q[at[-1]:] == 7.0).all())
        pos = [p if p < 0 else p + n for p, n in zip(pos, counts)]


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (3, 1, 64), (7, 7, 128)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [40, 7, 70, 3]])
def test_append_rotates(heads, kv, dim, norm, counts):
    """A pair (a, b) of size r turned by an angle whose cosine and sine are off by 2^-21 (sincospi of a fraction of a turn
    rounded to fp32) is off by 2^-20 r, the norm by (dim + 8) u; then half a step of q's type.  In the cache: a value x =
    K / scale is held within half a step, 2^-4 |x| or 2^-10, and what x is off by.  (A maximum within that of a border could
    take either scale: these inputs have none.)"""
    positions, page, q_type = [0, 61, 900001 % 4096 + 33, 127], 32, "bf16"
    c = Calls(kv, dim, page, [140] * 4, seed=heads, layout="slots")
    g = torch.Generator().manual_seed(heads)
    qkv = torch.randn(sum(counts), heads + 2 * kv, dim, generator=g).cuda()
    gq, gk = (1 + 0.1 * torch.randn(dim, generator=g)).cuda(), (1 + 0.1 * torch.randn(dim, generator=g)).cuda()
    was = c.pool.held(0)
    q = c.append(heads, positions, counts, qkv, q_type, gq=gq if norm else None, gk=gk if norm else None)
    torch.cuda.synchronize()
    x = qkv.double().cpu()
    pre_q, pre_k = x[:, :heads], x[:, heads:heads + kv]
    if norm:
        pre_q = pre_q / (pre_q.square().mean(-1, keepdim=True) + EPS).sqrt() * gq.double().cpu()
        pre_k = pre_k / (pre_k.square().mean(-1, keepdim=True) + EPS).sqrt() * gk.double().cpu()
    at = [p + i for p, n in zip(positions, counts) for i in range(n)]
    want_q = torch.stack([rotate(a, p, THETA) for a, p in zip(pre_q, at)])
    want_k = torch.stack([rotate(a, p, THETA) for a, p in zip(pre_k, at)])

    def off(pre):
        r = pre.unflatten(-1, (dim // 2, 2)).norm(dim=-1).repeat_interleave(2, -1)
        return r * (2.0 ** -20 + ((dim + 8) * U32 if norm else 0.0) + 2 * U32)
    assert bool(((q.double().cpu() - want_q).abs() <= off(pre_q) + half_step(q_type) * want_q.abs()).all())
    _, scale, plain = expect(c, was, 0, positions, counts, want_k)
    got, got_scale = c.pool.held(0)
    assert torch.equal(got_scale, scale)
    k_off, start, rows = off(pre_k), starts(counts), {}
    for s, (p, n) in enumerate(zip(positions, counts)):
        for i in range(n):
            rows.setdefault((c.table[s][(p + i) // page]), []).append(start[s] + i)
    for (page_no, h), (lo, y) in plain.items():
        held = from_e4m3(got[0, page_no, h, lo:lo + len(y)].contiguous())
        e = k_off[rows[page_no], h] / float(scale[0, page_no, h])
        assert bool(((held - y).abs() <= torch.maximum(2.0 ** -4 * y.abs(), torch.tensor(2.0 ** -10)) * (1 + 2.0 ** -10) + e).all())


def test_append_far_position():
    """Angles of positions whose product with a frequency leaves fp32 behind."""
    c = Calls(1, 64, 128, [8192], seed=3)
    qkv = torch.randn(1, 4, 64).cuda()
    p = 128 * 8191 + 77
    q = c.append(2, [p], [1], qkv, "fp16")
    torch.cuda.synchronize()
    x = qkv.double().cpu()
    for h in range(2):
        r = x[0, h].unflatten(-1, (32, 2)).norm(dim=-1).repeat_interleave(2, -1)
        want = rotate(x[0, h], p, THETA)
        assert bool(((q[0, h].double().cpu() - want).abs() <= r * 2.0 ** -19 + 2.0 ** -11 * want.abs()).all())


def test_append_agrees_with_the_slab():
    """The same q, bit for bit, as the append to a slab."""
    qkv, pos, start = torch.randn(9, 12, 128).cuda(), ints([1000]), ints([0, 9])
    k, v = torch.zeros(1, 1, 2000, 2, 128, dtype=torch.bfloat16).cuda(), torch.zeros(1, 1, 2000, 2, 128, dtype=torch.bfloat16).cuda()
    want = torch.empty(9, 8, 128, dtype=torch.bfloat16).cuda()
    g = torch.ones(128).cuda()
    V.rope_append_dev(V.KvCache(ptr(k), ptr(v), "bf16", 1, 1, 2000, 2, 128), 0, V.Rows(ptr(pos), ptr(start), None, 9, 9), ptr(qkv),
                      "fp32", 8, 0, ptr(g), ptr(g), EPS, THETA, ptr(want), V.STREAM_LEGACY)
    c = Calls(2, 128, 64, [20])
    q = c.append(8, [1000], [9], qkv, "bf16", gq=g, gk=g)
    torch.cuda.synchronize()
    # the norm's sum may run in another order: half a step and its 2^-16
    assert bool(((q.double() - want.double()).abs() <= (2 * half_step("bf16") + 2.0 ** -16) * want.double().abs() + 2.0 ** -16).all())


@pytest.mark.parametrize("counts", [[1, 1], [20, 40]])
def test_append_of_what_is_not_finite(counts):
    """NaN and infinities become NaN and leave the scale alone; a page of nothing else gets the least scale."""
    c = Calls(2, 64, 16, [4, 4], seed=4)
    qkv = torch.randn(sum(counts), 8, 64)
    qkv[0, 4, 3], qkv[0, 5, 0], qkv[0, 6, 9], qkv[-1, 7] = math.nan, math.inf, -math.inf, math.nan
    qkv[0, 4, 5], qkv[0, 6, 10] = 3.0e38, 1e-40
    qkv = qkv.cuda()
    was = [c.pool.held(i) for i in (0, 1)]
    c.append(4, [0, 15], counts, qkv, "bf16", theta=0.0)
    torch.cuda.synchronize()
    x = qkv.double().cpu()
    for which, rows in ((0, x[:, 4:6]), (1, x[:, 6:])):
        code, scale, _ = expect(c, was[which], which, [0, 15], counts, rows)
        got, got_scale = c.pool.held(which)
        assert torch.equal(got_scale, scale)
        nan = (code & 127) == NAN8
        assert torch.equal((got & 127) == NAN8, nan) and torch.equal(got[~nan], code[~nan])


def test_append_zeros_and_tiny():
    c = Calls(1, 64, 16, [2], seed=5)
    for value in (0.0, 1e-37, 1e-44):
        qkv = torch.full((3, 3, 64), value).cuda()
        c.append(1, [0], [3], qkv, "fp16", theta=0.0)
        torch.cuda.synchronize()
        got, scale = c.pool.held(0)
        assert float(scale[0, c.table[0][0], 0]) == scale_for(float(qkv[0, 0, 0]))
        assert torch.equal(got[0, c.table[0][0], 0, :3], to_e4m3(qkv[:, 1].double().cpu() / scale_for(float(qkv[0, 0, 0]))))


@pytest.mark.parametrize("counts", [[1, 1, 1], [50, 20, 70]])
def test_append_drops_what_has_no_page(counts):
    """Pages that are not there, rows past the table (q too), and a larger max_rows than any stream has."""
    lost = [(0, 1), (0, 2), (1, 0), (2, 4)]
    c = Calls(2, 128, 16, [5, 5, 5], seed=6, lost=lost)
    pos = [16, 7, 62]
    qkv = torch.randn(sum(counts), 8, 128).cuda()
    was = [c.pool.held(i) for i in (0, 1)]
    q = c.append(4, pos, counts, qkv, "bf16", theta=0.0, most=80 if counts[0] > 1 else None)
    torch.cuda.synchronize()
    x = qkv.double().cpu()
    for which, rows in ((0, x[:, 4:6]), (1, x[:, 6:])):
        code, scale, _ = expect(c, was[which], which, pos, counts, rows)
        got, got_scale = c.pool.held(which)
        assert torch.equal(got_scale, scale) and torch.equal(got, code)
    at = starts(counts)
    for s, (p, n) in enumerate(zip(pos, counts)):
        n0 = min(n, 80 - p)
        assert torch.equal(q[at[s]:at[s] + n0], qkv[at[s]:at[s] + n0, :4].bfloat16()) and bool((q[at[s] + n0:at[s + 1]] == 7.0).all())


def test_no_more_rows_than_declared():
    c = Calls(2, 64, 16, [5], seed=7)
    qkv = torch.randn(40, 6, 64).cuda()
    was = c.pool.held(0)
    q = c.append(2, [3], [40], qkv, "bf16", theta=0.0, most=20)
    torch.cuda.synchronize()
    code, scale, _ = expect(c, was, 0, [3], [40], qkv.double().cpu()[:, 2:4], most=20)
    got, got_scale = c.pool.held(0)
    assert torch.equal(got, code) and torch.equal(got_scale, scale)
    assert torch.equal(q[:20], qkv[:20, :2].bfloat16()) and bool((q[20:] == 7.0).all())


def test_a_page_of_its_own_again():
    """A page that another stream filled: slot 0 among the new rows starts its scale anew."""
    c = Calls(1, 64, 16, [1], seed=8)
    big, small = torch.full((16, 3, 64), 1e6).cuda(), torch.full((2, 3, 64), 1e-3).cuda()
    c.append(1, [0], [16], big, "bf16", theta=0.0)
    c.append(1, [0], [2], small, "bf16", theta=0.0)
    torch.cuda.synchronize()
    got, scale = c.pool.held(1)
    assert float(scale[0, c.table[0][0], 0]) == scale_for(float(small[0, 0, 0]))


@pytest.mark.parametrize("layout", ["heads", "slots", "pages_last"])
@pytest.mark.parametrize("kv,dim,page", [(3, 64, 16), (8, 128, 64), (1, 128, 128)])
def test_copy_pages(layout, kv, dim, page):
    """Every layer, scales too; pairs with a page that is none are left out."""
    p = Pool(3, 40, page, kv, dim, seed=9, layout=layout).upload()
    before = [p.held(i) for i in (0, 1)]
    src, dst = [0, 39, 7, -1, 3, 40, 1 << 30], [20, 21, 22, 23, 41, 24, 25]
    cache, a, b = p.cache(V, torch.zeros(1, 1, dtype=torch.int32).cuda()), ints(src), ints(dst)
    V.kv_copy_pages_dev(cache, ptr(a), ptr(b), len(src), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    for which in (0, 1):
        code, scale = (t.clone() for t in before[which])
        for s, d in list(zip(src, dst))[:3]:
            code[:, d], scale[:, d] = code[:, s].clone(), scale[:, s].clone()
        got, got_scale = p.held(which)
        assert torch.equal(got, code) and torch.equal(got_scale, scale)


def test_copy_needs_no_table():
    p = Pool(1, 4, 16, 1, 64, seed=10).upload()
    c = V.PagedCache(ptr(p.dk), ptr(p.dv), ptr(p.dks), ptr(p.dvs), None, 0, 1, 4, 16, 0, 1, 64)
    a, b = ints([1]), ints([2])
    V.kv_copy_pages_dev(c, ptr(a), ptr(b), 1, V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(p.dk[0, 2], p.dk[0, 1]) and torch.equal(p.dvs[0, 2], p.dvs[0, 1])


@pytest.mark.parametrize("dtype,heads,kv,dim,page", [("bf16", 8, 2, 128, 16), ("fp16", 6, 6, 64, 64), ("bf16", 32, 8, 128, 32)])
def test_streams_served(dtype, heads, kv, dim, page):
    """Prompts of three streams, a fork of one, steps of all: append and attention in a graph that is replayed, each
    output held against the definition over what the cache holds then."""
    counts, layers = [37, 5, 90], 2
    width, most = heads + 2 * kv, 128 // page + 2
    c = Calls(kv, dim, page, [most] * 4, seed=11, layers=layers)
    g = torch.Generator().manual_seed(12)

    def check(positions, counts, q, out, lse, layer):
        case = Case.__new__(Case)
        case.__dict__.update(dtype=dtype, heads=heads, kv=kv, dim=dim, page=page, positions=positions, counts=counts, window=0, n_sink=0,
                             layer=layer, n=sum(counts), q=q.cpu(), table=c.table, start=starts(counts),
                             keys=[[] if p < 0 else [list(range(p + i + 1)) for i in range(n)] for p, n in zip(positions, counts)])
        case.pool = Pool.__new__(Pool)
        held = [c.pool.held(i) for i in (0, 1)]
        case.pool.code, case.pool.scale = [h[0] for h in held], [h[1] for h in held]
        case.check(out, lse)

    positions = [0, 0, 0, -1]
    for layer in range(layers):
        c.layer = layer
        qkv = torch.randn(sum(counts), width, dim, generator=g).cuda()
        q = c.append(heads, positions, counts + [0], qkv, dtype)
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
        r = V.Rows(ptr(c.hold[0]), ptr(c.hold[1]), None, q.shape[0], max(counts))
        V.attention_paged_dev(c.pool.cache(V, c.dtable), layer, r, ptr(q), dtype, heads, 0, 0, 0.0, ptr(out), ptr(lse), V.STREAM_LEGACY)
        torch.cuda.synchronize()
        check(positions, counts + [0], q, out, lse, layer)
    # the fourth stream goes on from the first: full pages shared, the last one copied
    full = counts[0] // page
    c.table[3][:full] = c.table[0][:full]
    c.dtable.copy_(ints(c.table))
    a, b = ints([c.table[0][full]]), ints([c.table[3][full]])
    V.kv_copy_pages_dev(c.pool.cache(V, c.dtable), ptr(a), ptr(b), 1, V.STREAM_LEGACY)
    lengths = counts + [counts[0]]
    pos = ints(lengths)
    qkv = torch.zeros(layers, 4, width, dim).cuda()
    q = torch.empty(layers, 4, heads, dim, dtype=TORCH[dtype]).cuda()
    out, lse = torch.empty_like(q), torch.empty(layers, 4, heads).cuda()
    cache, rows = c.pool.cache(V, c.dtable), V.Rows(ptr(pos), None, None, 4, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        for layer in range(layers):
            V.rope_append_paged_dev(cache, layer, rows, ptr(qkv[layer]), "fp32", heads, 0, None, None, EPS, THETA, ptr(q[layer]), dtype, st)
            V.attention_paged_dev(cache, layer, rows, ptr(q[layer]), dtype, heads, 0, 0, 0.0, ptr(out[layer]), ptr(lse[layer]), st)
    for step in range(5):
        qkv.copy_(torch.randn(qkv.shape, generator=g) * (1 + step))
        graph.replay()
        torch.cuda.synchronize()
        for layer in range(layers):
            check(lengths, [1] * 4, q[layer], out[layer], lse[layer], layer)
        lengths = [n + 1 for n in lengths]
        pos.copy_(ints(lengths))
