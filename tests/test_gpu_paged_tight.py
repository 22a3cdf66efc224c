"""The operators over a paged cache to their last bits: keys and queries on the side
of a rounding that the definition gives, the log of the sum where scores are small,
the kernel of many rows with its streams in order."""
import pytest
import torch

import voxcuda as V
from paged_ref import Case, from_e4m3, to_e4m3
from rows_ref import TORCH, U32
from test_gpu_paged_cache import THETA, Calls, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def turned(x, at, dim):
    """x [rows][heads][dim] turned by the rows' angles, 64 bits, and what the kernel may be off by: cosine and sine by 2^-23.7
    (the kernel's word) and 2^-30 of a far angle, each product and their sum by a rounding."""
    a = at.double()[:, None] * THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    c, s = a.cos()[:, None], a.sin()[:, None]
    p, q = x[..., 0::2], x[..., 1::2]
    e = (2.0 ** -23.7 + 2.0 ** -30) * (p.abs() + q.abs())
    one, two = p * c - q * s, p * s + q * c
    off = torch.stack((e + U32 * ((p * c).abs() + (q * s).abs() + one.abs()), e + U32 * ((p * s).abs() + (q * c).abs() + two.abs())), -1)
    return torch.stack((one, two), -1).flatten(-2), off.flatten(-2)


def check_rounded(c, heads, positions, counts, q_type, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(sum(counts), heads + 2 * c.kv, c.dim, generator=g).cuda()
    q = c.append(heads, positions, counts, qkv, q_type)
    torch.cuda.synchronize()
    x, at = qkv.double().cpu(), torch.tensor([p + i for p, n in zip(positions, counts) for i in range(n)])
    want, off = turned(x[:, :heads], at, c.dim)
    got, typ = q.cpu(), TORCH[q_type]
    assert bool((got >= (want - off).to(typ)).all()) and bool((got <= (want + off).to(typ)).all())
    want, off = turned(x[:, heads:heads + c.kv], at, c.dim)
    code, scale = c.pool.held(0)
    start, near = starts(counts), 0
    for s, (p, n) in enumerate(zip(positions, counts)):
        for i in range(p // c.page, (p + n - 1) // c.page + 1):
            a, b = max(p, i * c.page), min(p + n, (i + 1) * c.page)
            page, rows = c.table[s][i], slice(start[s] + a - p, start[s] + b - p)
            held = from_e4m3(code[0, page, :, a - i * c.page:b - i * c.page].contiguous())                 # kv, rows, dim
            by = scale[0, page][:, None, None]
            low, high = (from_e4m3(to_e4m3(y / by)) for y in ((want - off)[rows].transpose(0, 1), (want + off)[rows].transpose(0, 1)))
            assert bool((held >= low).all()) and bool((held <= high).all()), (s, i)
            near += int((low != high).sum())
    return near, want.numel()


@pytest.mark.parametrize("q_type", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (16, 16, 64)])
def test_keys_land_on_the_definitions_side(q_type, heads, kv, dim):
    """Rotated heads: the e4m3 number, and q's, is that of the 64-bit value but where a border lies within what the value is off
    by, which is so for few.  With a sine that is 2^-21 off several of these keys would take the other neighbour."""
    c = Calls(kv, dim, 64, [5, 8, 48, 66], seed=1)
    near, of = check_rounded(c, heads, [0, 7, 2600, 3999], [300, 301, 299, 200], q_type, seed=2)
    assert near < of * 2.0 ** -14


def test_far_keys_too():
    """Positions next to 2^20: the angle's fraction is fp64's."""
    c = Calls(1, 64, 128, [8192], seed=3)
    check_rounded(c, 2, [128 * 8190 + 5], [250], "fp16", seed=4)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim,rows", [(8, 2, 128, 1), (8, 2, 128, 9), (8, 2, 128, 50), (8, 4, 64, 50), (8, 8, 128, 150), (8, 2, 64, 100)])
def test_lse_of_small_scores(dtype, heads, kv, dim, rows):
    """Scores of 2^-3 and less: with S as in the check of outputs, the lse is off by (dim + 10) u S of the scores and 2^-22 of ex2;
    by the sums, in which a weight goes through 24 + N / 8 additions at most of fp32 (lanes, groups, steps; shares beside one
    another); and by the log's and the base's roundings, (4 |lse| + 16) u."""
    c = Case(dtype, heads, kv, dim, 16, [11, 40, 3], [rows] * 3, seed=rows, scale_q=0.02)
    _, lse = c.run(V)
    torch.cuda.synchronize()
    lse = lse.double().cpu()
    for s, seen in enumerate(c.keys):
        n = len(seen[-1])
        for h in range(heads):
            k, _ = c.values(s, list(range(n)), h // (heads // kv))
            q = c.q[c.start[s]:c.start[s + 1], h].double()
            mask = torch.arange(n)[None] <= c.positions[s] + torch.arange(rows)[:, None]
            z = torch.logsumexp(((q @ k.T) / dim ** 0.5).masked_fill(~mask, -torch.inf), -1)
            big = ((q.abs() @ k.abs().T) / dim ** 0.5).amax(-1)
            tol = ((dim + 10) * big + 24 + mask.sum(-1) / 8 + 4 * z.abs() + 16) * U32 + 2.0 ** -22
            off = (lse[c.start[s]:c.start[s + 1], h] - z).abs()
            assert bool((off <= tol).all()), (s, h, float((off / tol).max()))


@pytest.mark.parametrize("heads,kv,dim,rows,exp", [(8, 2, 128, 1, -7), (8, 2, 64, 9, 3), (16, 16, 128, 9, -2), (8, 2, 128, 60, -7), (8, 2, 128, 60, 7),
                                                   (8, 8, 64, 150, -3)])
def test_a_weight_of_one_rounds_to_itself(heads, kv, dim, rows, exp):
    """The row that sees one key gives its V: the largest weight loses nothing to fp16, 2^-20 is left for ex2, the sum and
    their quotient.  Another page's V is 2^exp times as large as the first one's."""
    c = Case("fp16", heads, kv, dim, 16, [0], [rows], seed=rows)
    for i, g in enumerate(c.table[0]):
        if 0 <= g < c.pool.pages:
            c.pool.scale[1][0, g] = 2.0 ** (-7 + (exp if i else 0))
    c.pool.upload()
    out, _ = c.run(V)
    torch.cuda.synchronize()
    for h in range(heads):
        v = c.values(0, [0], h // (heads // kv))[1][0]
        low, high = ((v - 2.0 ** -20 * v.abs()).half(), (v + 2.0 ** -20 * v.abs()).half())
        got = out[0, h].cpu()
        assert bool((got >= low).all()) and bool((got <= high).all()), h


@pytest.mark.parametrize("streams", [2, 31, 32, 33, 40])
def test_streams_in_order_of_the_many_rows_kernel(streams):
    """Streams of many lengths, in the order of their reach or, beyond 32, in turn: the kernel that orders them is the one called."""
    pos = [(s * 53) % 7 * 30 if s % 6 != 4 else -1 for s in range(streams)]
    counts = [(s * 29) % 70 + 1 if s % 4 != 3 else 0 for s in range(streams)]
    counts[0] = 70
    c = Case("fp16", 4, 1, 64, 16, pos, counts, seed=streams, tail=1)
    assert V.attention_paged_plan(c.cache(V), c.rows(V), "fp16", 4, 0, 0)[0] >= 128
    out, lse = c.run(V)
    torch.cuda.synchronize()
    c.check(out, lse)
