"""Token log probabilities, entropy and top alternatives against 64 bits."""
import math

import pytest
import torch

import voxcuda as V
from rows_ref import TORCH, U32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def ptr(t):
    return None if t is None else t.data_ptr()


def run(x, tokens, n_top, dtype, stream=V.STREAM_LEGACY):
    """x: a 2-D view with unit inner stride."""
    n, vocab = x.shape
    lp, ent = torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    ids = torch.full((n, max(n_top, 1)), 7, dtype=torch.int32, device="cuda")
    top = torch.full((n, max(n_top, 1)), 7.0, device="cuda")
    V.token_logprobs_dev(x.data_ptr(), dtype, n, vocab, x.stride(0) if n > 1 else 0, ptr(tokens), n_top, ptr(lp), ptr(ent),
                         ptr(ids) if n_top else None, ptr(top) if n_top else None, stream)
    torch.cuda.synchronize()
    return lp.cpu(), ent.cpu(), ids.cpu()[:, :n_top], top.cpu()[:, :n_top]


def check(x, tokens, n_top, dtype, got):
    """A logit's distance from the maximum is exact to half a step; e^d to 2
    ulp of ex2 and d's own 2 u, at most 2^-22 + 2 u |d| relative; the sums of
    n terms in up to ~600 sequential adds per thread, 24 folds: 640 u
    relative.  So ln Z is off by at most e = 2^-22 + 640 u + (weighted) 2 u |d|
    plus a step of its size, and the entropy, a sum of e^d |d| / Z, by the
    same relative error of its terms."""
    lp, ent, ids, top = got
    x = x.double().cpu()
    p = torch.log_softmax(x, -1)
    w = p.exp()
    m = x.amax(-1, keepdim=True)
    d = torch.where(w > 0, (x - m).abs(), 0.0)
    mean_d = (w * d).sum(-1)
    e = 2.0 ** -22 + 640 * U32 + 2 * U32 * mean_d
    tok = tokens.long().cpu()
    want = p.gather(1, tok[:, None]).squeeze(1)
    size = (x.gather(1, tok[:, None]) - m).abs().squeeze(1)
    tol = e + 2 * U32 * (size + want.abs() + 1)
    fine = torch.isfinite(want)
    assert bool(((lp - want).abs()[fine] <= tol[fine]).all()), float(((lp - want).abs() / tol)[fine].max())
    assert torch.equal(lp[~fine].double(), want[~fine])
    want = -torch.where(w > 0, w * p, 0.0).sum(-1)
    tol = e + (2.0 ** -22 + 640 * U32) * mean_d + 2 * U32 * (w * d * d).sum(-1) + 4 * U32 * (want + mean_d)
    assert bool(((ent - want).abs() <= tol).all()), float(((ent - want).abs() / tol).max())
    if n_top:
        order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :n_top]
        assert torch.equal(ids.long(), order)
        want = p.gather(1, order)
        tol = (e[:, None] + 2 * U32 * ((x.gather(1, order) - m).abs() + want.abs() + 1))
        ok = torch.isfinite(want)
        assert bool(((top - want).abs()[ok] <= tol[ok]).all()) and torch.equal(top[~ok].double(), want[~ok])


def rows(n, vocab, dtype, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(n, vocab, generator=g, device="cuda") * scale).to(TORCH[dtype])
    return x, torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,vocab,n_top", [
    (1, 131072, 5), (1, 131072, 32), (3, 131072, 1), (200, 4099, 20), (1, 1, 1), (2, 7, 7), (5, 33, 32), (1, 1025, 0),
    (300, 1000, 32), (1, 300007, 32), (40, 65537, 3), (149, 8191, 12)])
def test_rows(dtype, n, vocab, n_top):
    x, tok = rows(n, vocab, dtype, seed=vocab + n_top)
    check(x, tok, n_top, dtype, run(x, tok, n_top, dtype))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shift", [1, 3, 5])
def test_unaligned_rows(dtype, shift):
    x, tok = rows(4, 5003, dtype, seed=shift)
    wide = torch.full((4, 5003 + 2 * shift), 50.0, dtype=TORCH[dtype], device="cuda")   # neighbours would win
    wide[:, shift:shift + 5003] = x
    check(x, tok, 8, dtype, run(wide[:, shift:shift + 5003], tok, 8, dtype))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ties_go_to_the_lowest_id(dtype):
    for x in (torch.zeros(2, 131072), torch.arange(131072).remainder(3).float()[None].repeat(2, 1),
              -torch.arange(20000).remainder(50).float()[None].repeat(160, 1),
              torch.tensor([0.0, -0.0] * 5000)[None].repeat(2, 1)):
        x = x.to(TORCH[dtype]).cuda()
        tok = torch.full((x.shape[0],), 4, dtype=torch.int32, device="cuda")
        check(x, tok, 32, dtype, run(x, tok, 32, dtype))


@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("n", [1, 160])
def test_sorted_rows(order, n):
    x = (torch.linspace(-20, 20, 50021) * order)[None].repeat(n, 1).cuda()
    tok = torch.full((n,), 25000, dtype=torch.int32, device="cuda")
    check(x, tok, 32, "fp32", run(x, tok, 32, "fp32"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_masked_and_lowest_logits(dtype):
    x, tok = rows(4, 40000, dtype, seed=3)
    x[0, 100:] = -math.inf                      # a hundred left
    x[1, 5:] = -math.inf                        # fewer than asked for
    x[2, 1::2] = torch.finfo(x.dtype).min       # the type's lowest value
    x[3] = torch.finfo(x.dtype).min             # nothing else: uniform
    check(x, tok, 20, dtype, run(x, tok, 20, dtype))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n", [4, 300])
def test_the_largest_logits(dtype, n):
    x, tok = rows(n, 5003, dtype, seed=5)
    most = torch.finfo(x.dtype).max
    x[0, 77] = most                             # distances of 3e38
    x[1, ::3] = most
    x[2] = most / 2
    x[3, 1::2] = torch.finfo(x.dtype).min
    x[3, ::2] = most
    tok[3] = 5002
    check(x, tok, 5, dtype, run(x, tok, 5, dtype))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rows_without_a_distribution(dtype):
    x, tok = rows(6, 9000, dtype, seed=4)
    good = x[5:].clone()
    x[0] = -math.inf
    x[1, 4000] = math.nan
    x[2, 8999] = math.inf
    x[3] = math.nan
    tok[4] = 9000
    x[4, 3:] = math.nan
    lp, ent, ids, top = run(x, tok, 5, dtype)
    assert bool(torch.isnan(lp[:5]).all()) and bool(torch.isnan(ent[:4]).all())
    assert bool(torch.isnan(top[:5]).all())
    assert ids[0].tolist() == [0, 1, 2, 3, 4] and ids[3].tolist() == [-1] * 5
    assert sorted(ids[4, :3].tolist()) == [0, 1, 2] and ids[4, 3:].tolist() == [-1, -1]
    assert ids[2, 0] == 8999 and 4000 not in ids[1].tolist()
    check(good, tok[5:], 5, dtype, (lp[5:], ent[5:], ids[5:], top[5:]))


def test_a_token_outside_gives_nan_only_for_itself():
    x, tok = rows(3, 500, "fp32", seed=5)
    tok[1], tok[2] = -1, 500
    lp, ent, _, _ = run(x, tok, 0, "fp32")
    assert bool(torch.isfinite(lp[0])) and bool(torch.isnan(lp[1:]).all()) and bool(torch.isfinite(ent).all())


def test_confident_rows_keep_their_digits():
    """ln Z = log1p(rest): a log probability and an entropy near 0 are right
    to their own size, not to that of 1."""
    x = torch.full((3, 2000), -30.0, device="cuda")
    x[:, 7] = 0.0
    x[1, 8], x[2, 9] = -12.0, -5.0
    tok = torch.full((3,), 7, dtype=torch.int32, device="cuda")
    lp, ent, _, _ = run(x, tok, 0, "fp32")
    d = x.double().cpu()
    d[:, 7] = -math.inf
    rest = d.exp().sum(-1)   # apart from the 1 of the maximum: 64 bits added to 1 keep only 2^-53
    lz = torch.log1p(rest)
    p = lz[:, None].neg().expand(3, 8)
    want = lz + (d.exp() * -d.clamp(min=-1e9)).sum(-1) / (1 + rest)
    # terms are right to 2^-22 + 2 u |d|, |d| <= 30, their sums to 20 u: 2^-17 in all
    assert bool(((lp - p[:, 7]).abs() <= 2.0 ** -17 * p[:, 7].abs()).all())
    assert bool(((ent - want).abs() <= 2.0 ** -17 * want).all())


def test_every_part_on_its_own_and_a_replayed_graph():
    x, tok = rows(9, 70001, "fp32", seed=6)
    lp, ent, ids, top = run(x, tok, 6, "fp32")
    a, b = torch.empty(9, device="cuda"), torch.empty(9, device="cuda")
    i = torch.empty(9, 6, dtype=torch.int32, device="cuda")
    V.token_logprobs_dev(x.data_ptr(), "fp32", 9, 70001, 0, ptr(tok), 0, ptr(a), None, None, None, V.STREAM_LEGACY)
    V.token_logprobs_dev(x.data_ptr(), "fp32", 9, 70001, 0, None, 0, None, ptr(b), None, None, V.STREAM_LEGACY)
    V.token_logprobs_dev(x.data_ptr(), "fp32", 9, 70001, 0, None, 6, None, None, ptr(i), None, V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(a.cpu(), lp) and torch.equal(b.cpu(), ent) and torch.equal(i.cpu(), ids)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        V.token_logprobs_dev(x.data_ptr(), "fp32", 9, 70001, 0, ptr(tok), 0, ptr(a), ptr(b), None, None,
                             torch.cuda.current_stream().cuda_stream)
    y, _ = rows(9, 70001, "fp32", seed=7)
    x.copy_(y)
    g.replay()
    torch.cuda.synchronize()
    lp, ent, _, _ = run(y, tok, 0, "fp32")
    assert torch.equal(a.cpu(), lp) and torch.equal(b.cpu(), ent)


def test_offsets_beyond_32_bits():
    ld = (1 << 31) + 8
    big = torch.empty(ld + 5000, dtype=torch.bfloat16, device="cuda")
    x, tok = rows(2, 5000, "bf16", seed=8)
    big[:5000], big[ld:] = x[0], x[1]
    out = [torch.empty(2, device="cuda") for _ in range(2)]
    V.token_logprobs_dev(big.data_ptr(), "bf16", 2, 5000, ld, ptr(tok), 0, ptr(out[0]), ptr(out[1]), None, None, V.STREAM_LEGACY)
    torch.cuda.synchronize()
    lp, ent, _, _ = run(x, tok, 0, "bf16")
    assert torch.equal(out[0].cpu(), lp) and torch.equal(out[1].cpu(), ent)
