"""Rotary append, commit and fork over a cache slab, and the row operators in
a round as they are used together, against the definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

import voxcuda as V
from rows_ref import TORCH, U32, attention, depths, half_step, slot, visible

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


def slab(dtype, layers, streams, cap, kv, dim, seed=0, layout="slots"):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, streams, cap, kv, dim)
    k, v = torch.randn(shape, generator=g).to(TORCH[dtype]).cuda(), torch.randn(shape, generator=g).to(TORCH[dtype]).cuda()
    if layout == "heads":   # the same view, each head's slots together
        k = k.transpose(2, 3).contiguous().transpose(2, 3)
        v = v.transpose(2, 3).contiguous().transpose(2, 3)
    return k, v


def cache_of(k, v, dtype, n_sink):
    st = k.stride()
    return V.KvCache(k.data_ptr(), v.data_ptr(), dtype, k.shape[0], k.shape[1], k.shape[2], k.shape[3], k.shape[4], n_sink,
                     st[0], st[1], st[2], st[3])


def rotate(x, p, theta):
    """One head's interleaved pairs turned by p * theta^(-2d / dim), 64 bits."""
    dim = x.shape[-1]
    a = torch.tensor([p * theta ** (-2.0 * d / dim) for d in range(dim // 2)], dtype=torch.float64)
    return torch.stack((x[..., 0::2] * a.cos() - x[..., 1::2] * a.sin(), x[..., 0::2] * a.sin() + x[..., 1::2] * a.cos()),
                       -1).flatten(-2)


@pytest.mark.parametrize("src,dtype", [("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (3, 1, 64), (7, 7, 128)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_rope_append(src, dtype, heads, kv, dim, norm, tree):
    """A pair (a, b) of size r turned by an angle whose cosine and sine are off
    by 2^-21 (sincospi of a fraction of a turn rounded to fp32) is off by
    2^-20 r, the norm by (dim + 8) u, then half a step of the type."""
    layers, cap, n_sink, layer = 2, 40, 3, 1
    positions, counts, tail = [0, 30, -1, 900001, 35], [7, 0, 4, 9, 1], 2
    n = sum(counts)
    g = torch.Generator().manual_seed(heads)
    k, v = slab(dtype, layers, len(positions), cap, kv, dim, seed=1, layout="heads" if heads == 7 else "slots")
    k0, v0 = k.clone(), v.clone()
    width = heads + 2 * kv
    wide = torch.randn(n + tail, width * dim + 16, generator=g).to(TORCH[src]).cuda()
    qkv = wide[:, :width * dim].unflatten(1, (width, dim))
    gq, gk = (1 + 0.1 * torch.randn(dim, generator=g)).cuda(), (1 + 0.1 * torch.randn(dim, generator=g)).cuda()
    par, flat = None, None
    if tree:
        flat = [[max(i - 1 - i % 3, -1) for i in range(c)] for c in counts]
        par = ints([p for row in flat for p in row] + [-1] * tail)
    start = [sum(counts[:s]) for s in range(len(counts) + 1)]
    dpos, dstart = ints(positions), ints(start)
    q = torch.full((n + tail, heads, dim), 7.0, dtype=TORCH[dtype], device="cuda")
    V.rope_append_dev(cache_of(k, v, dtype, n_sink), layer, V.Rows(ptr(dpos), ptr(dstart), ptr(par), n + tail, max(counts)),
                      wide.data_ptr(), src, heads, wide.stride(0), ptr(gq) if norm else None, ptr(gk) if norm else None, EPS,
                      THETA, q.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    u = half_step(dtype)
    touched = torch.zeros(len(positions), cap, dtype=torch.bool)
    for s, (p, c) in enumerate(zip(positions, counts)):
        if p < 0:
            assert bool((q[start[s]:start[s + 1]] == 7.0).all())
            continue
        dep = depths(flat[s]) if tree else list(range(c))
        for i in range(c):
            x = qkv[start[s] + i].double().cpu()
            want_q, want_k, want_v = x[:heads], x[heads:heads + kv], x[heads + kv:]
            if norm:
                want_q = want_q / (want_q.square().mean(-1, keepdim=True) + EPS).sqrt() * gq.double().cpu()
                want_k = want_k / (want_k.square().mean(-1, keepdim=True) + EPS).sqrt() * gk.double().cpu()
            at = slot(p + i, cap, n_sink)
            touched[s, at] = True
            for got, pre in ((q[start[s] + i], want_q), (k[layer, s, at], want_k)):
                r = pre.unflatten(-1, (dim // 2, 2)).norm(dim=-1).repeat_interleave(2, -1)
                want = rotate(pre, p + dep[i], THETA)
                tol = r * (2.0 ** -20 + ((dim + 8) * U32 if norm else 0.0)) + u * want.abs() * (dtype != "fp32") + 2 * U32 * r
                assert bool(((got.double().cpu() - want).abs() <= tol).all()), (s, i)
            assert torch.equal(v[layer, s, at].cpu(), want_v.to(TORCH[dtype]))
    for new, old in ((k, k0), (v, v0)):
        assert torch.equal(new[0], old[0])
        assert torch.equal(new[layer][~touched.cuda()], old[layer][~touched.cuda()])
    assert bool((q[n:] == 7.0).all())


def test_rope_append_without_rotation_is_a_copy():
    k, v = slab("fp32", 1, 1, 8, 2, 64)
    qkv = torch.randn(3, 8, 64).cuda()
    q = torch.empty(3, 4, 64, device="cuda")
    pos, start = ints([6]), ints([0, 3])
    V.rope_append_dev(cache_of(k, v, "fp32", 0), 0, V.Rows(ptr(pos), ptr(start), None, 3, 3), qkv.data_ptr(), "fp32", 4, 0, None,
                      None, EPS, 0.0, q.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(q, qkv[:, :4]) and torch.equal(k[0, 0, [6, 7, 0]], qkv[:, 4:6])
    assert torch.equal(v[0, 0, [6, 7, 0]], qkv[:, 6:])


def test_rope_matches_the_stand_alone_rotation():
    """The same angles as vox_cuda_rope_dev, to fp32's rounding of a near position's."""
    x = torch.randn(1, 10, 128).cuda()
    k, v = slab("fp32", 1, 1, 4, 1, 128)
    q, pos = torch.empty(1, 8, 128, device="cuda"), ints([3])
    V.rope_append_dev(cache_of(k, v, "fp32", 0), 0, V.Rows(ptr(pos), n_rows=1), x.data_ptr(), "fp32", 8, 0, None, None, 0.0,
                      THETA, q.data_ptr(), V.STREAM_LEGACY)
    y = x[0, :8].contiguous()
    torch.cuda.synchronize()
    V.check(V.lib().vox_cuda_rope_dev(y.data_ptr(), 8, 128, 3, None, V.STREAM_LEGACY), "rope_dev")
    # an angle of at most 3 rad computed in fp32 is off by a few 2^-23 of it
    assert float((q[0] - y).abs().max()) <= 8 * 3 * 2.0 ** -23 * float(x.abs().max())


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["slots", "heads"])
def test_commit(dtype, layout):
    layers, cap, n_sink, ld = 3, 60, 2, 12
    positions = [0, 50, -1, 1000, 7, 3, 9]
    # identity, in order and dense (sources are other rows' targets), sits out, with gaps, cut at a repeat, none, cut at a large index
    paths = [[0, 1, 2], list(range(1, 13)), [5], [0, 4, 9, 30, 31, 32], [2, 3, 3, 9], [], [1, 57, 58]]
    kept = [3, 12, 0, 6, 2, 0, 2]
    k, v = slab(dtype, layers, len(positions), cap, 4, 64, seed=2, layout=layout)
    want_k, want_v = k.clone(), v.clone()
    for s, p in enumerate(positions):
        for n in range(kept[s]):
            a, b = slot(p + paths[s][n], cap, n_sink), slot(p + n, cap, n_sink)
            want_k[:, s, b], want_v[:, s, b] = k[:, s, a], v[:, s, a]
    dpos, took, new = ints(positions), ints([len(x) for x in paths]), ints([99] * 7)
    path = ints([x + [0] * (ld - len(x)) for x in paths])
    V.kv_commit_dev(cache_of(k, v, dtype, n_sink), ptr(dpos), ptr(path), ld, ptr(took), 12, ptr(new), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert new.tolist() == [p + n for p, n in zip(positions, kept)]


def test_commit_takes_no_more_than_declared():
    k, v = slab("fp32", 1, 2, 30, 1, 64, seed=3)
    k0 = k.clone()
    dpos, took, new, path = ints([4, 5]), ints([100, -3]), ints([0, 0]), ints([[3, 4, 5, 6], [1, 2, 3, 4]])
    V.kv_commit_dev(cache_of(k, v, "fp32", 0), ptr(dpos), ptr(path), 4, ptr(took), 2, ptr(new), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert new.tolist() == [6, 5]
    k0[0, 0, 4], k0[0, 0, 5] = k0[0, 0, 7].clone(), k0[0, 0, 8].clone()
    assert torch.equal(k, k0)


def test_commit_of_a_whole_tree_straddles_sinks_and_wrap():
    k, v = slab("bf16", 1, 2, 300, 1, 64, seed=4)
    want = k.clone()
    idx = [i for i in range(256) if i % 2 or i > 200]
    for s, p in enumerate([2, 290]):
        for n, a in enumerate(idx):
            want[0, s, slot(p + n, 300, 5)] = k[0, s, slot(p + a, 300, 5)]
    dpos, took, path = ints([2, 290]), ints([len(idx)] * 2), ints([idx + [0] * (256 - len(idx))] * 2)
    V.kv_commit_dev(cache_of(k, v, "bf16", 5), ptr(dpos), ptr(path), 256, ptr(took), 256, None, V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(k, want)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("layout", ["slots", "heads"])
@pytest.mark.parametrize("dim,kv", [(64, 3), (128, 8)])
def test_fork(dtype, layout, dim, kv):
    cap, positions = 33, [0, 5, 33, 5000, -1, 1, 1, 1, 1, 1, 1, 1]
    k, v = slab(dtype, 3, 12, cap, kv, dim, seed=5, layout=layout)
    want_k, want_v = k.clone(), v.clone()
    src, dst = [0, 1, 2, 3, 4, 3], [6, 7, 8, 9, 10, 11]
    for a, b in zip(src, dst):
        n = max(0, min(positions[a], cap))
        want_k[:, b, :n], want_v[:, b, :n] = k[:, a, :n], v[:, a, :n]
    dpos = ints(positions)
    V.kv_fork_dev(cache_of(k, v, dtype, 2), src, dst, ptr(dpos), V.STREAM_LEGACY)
    V.kv_fork_dev(cache_of(k, v, dtype, 2), [], [], ptr(dpos), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_a_round_of_drafting(seed=6):
    """Two rounds of: append a tree, attend it, score the drafts, commit a
    path, fork; then a plain token.  All captured in one graph and replayed,
    against the definitions on the host's copy of what the cache must hold."""
    dtype, heads, kv, dim, cap, n_sink, window, streams, n, vocab = "bf16", 8, 2, 64, 48, 2, 30, 3, 9, 501
    t = TORCH[dtype]
    g = torch.Generator().manual_seed(seed)
    k, v = slab(dtype, 1, streams, cap, kv, dim, seed=7)
    cache = cache_of(k, v, dtype, n_sink)
    pos, new, start = ints([20, 46, 11]), ints([0] * streams), ints([0, n, 2 * n, 3 * n])
    qkv = torch.randn(streams * n, heads + 2 * kv, dim, generator=g).cuda()
    parent = [-1, 0, 0, 1, 1, 2, 3, -1, 7]
    par = ints(parent * streams)
    path, took = ints([[0, 1, 4, 0]] * streams), ints([3, 2, 0])
    head = torch.randn(vocab, heads * dim, generator=g).to(t).cuda()
    q, out = torch.empty(streams * n, heads, dim, dtype=t, device="cuda"), torch.empty(streams * n, heads, dim, dtype=t, device="cuda")
    logits = torch.empty(streams * n, vocab, device="cuda")
    tok, lp, ent = ints([5] * (streams * n)), torch.empty(streams * n, device="cuda"), torch.empty(streams * n, device="cuda")
    ids, top = torch.empty(streams * n, 3, dtype=torch.int32, device="cuda"), torch.empty(streams * n, 3, device="cuda")
    rows = V.Rows(ptr(pos), ptr(start), ptr(par), streams * n, n)

    def one_round():
        st = torch.cuda.current_stream().cuda_stream or V.STREAM_LEGACY
        V.rope_append_dev(cache, 0, rows, qkv.data_ptr(), "fp32", heads, 0, None, None, EPS, THETA, q.data_ptr(), st)
        V.attention_tree_dev(cache, 0, rows, q.data_ptr(), heads, window, 0.0, out.data_ptr(), None, st)
        torch.matmul(out.flatten(1).float(), head.float().T, out=logits)
        V.token_logprobs_dev(logits.data_ptr(), "fp32", streams * n, vocab, 0, ptr(tok), 3, ptr(lp), ptr(ent), ptr(ids), ptr(top), st)
        V.kv_commit_dev(cache, ptr(pos), ptr(path), 4, ptr(took), 3, ptr(new), st)
        pos.copy_(new)

    held_k, held_v, held_pos = k.clone(), v.clone(), pos.clone()
    s0 = torch.cuda.Stream()
    s0.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s0):
        one_round()   # the library product's own set-up, before the capture
    torch.cuda.synchronize()
    k.copy_(held_k), v.copy_(held_v), pos.copy_(held_pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s0):
        one_round()
    k.copy_(held_k), v.copy_(held_v), pos.copy_(held_pos)

    mk, mv, mpos = k[0].double().cpu(), v[0].double().cpu(), pos.tolist()
    dep = depths(parent)
    u = half_step(dtype)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        x = qkv.double().cpu()
        for s in range(streams):
            for i in range(n):
                at = slot(mpos[s] + i, cap, n_sink)
                mk[s, at] = rotate(x[s * n + i, heads:heads + kv], mpos[s] + dep[i], THETA).to(t).double()
                mv[s, at] = x[s * n + i, heads + kv:].to(t).double()
            for i in range(n):
                keys = [slot(j, cap, n_sink) for j in visible(mpos[s], n, i, cap, n_sink, window, parent)]
                for h in range(heads):
                    qq = rotate(x[s * n + i, h], mpos[s] + dep[i], THETA).to(t).double()
                    o, _, big = attention(qq, mk[s, keys, h // 4], mv[s, keys, h // 4], keys, 1 / math.sqrt(dim))
                    # q and k may each be rounded to the neighbour of the definition's: a step, 2 u, of a score's terms
                    d = 4 * u * big
                    tol = (2 * d + u) * float(mv[s, keys, h // 4].abs().max()) + u * o.abs()
                    assert bool(((out[s * n + i, h].double().cpu() - o).abs() <= tol).all())
            for m in range(took.tolist()[s]):
                a, b = slot(mpos[s] + [0, 1, 4][m], cap, n_sink), slot(mpos[s] + m, cap, n_sink)
                mk[s, b], mv[s, b] = mk[s, a].clone(), mv[s, a].clone()
            mpos[s] += took.tolist()[s]
        p = torch.log_softmax(logits.double().cpu(), -1)
        # x - m exact to half a step, ln Z to a few steps of its size
        assert float((lp.double().cpu() - p[:, 5]).abs().max()) <= 8 * U32 * (float(p.abs().max()) + 1)
        assert torch.equal(ids.cpu().long(), torch.topk(logits, 3).indices.cpu())
        assert pos.tolist() == mpos
        # (the appended rows may round differently by a step)
        assert bool(((k[0].double().cpu() - mk).abs() <= 2 * u * mk.abs() + 1e-6).all()) and torch.equal(v[0].double().cpu(), mv)


def test_on_a_decoder_state():
    """The decoder's own ring as a slab: window attention of a step's query
    agrees with the library's decode attention, and the state's confidences
    with its logits."""
    import bind as B
    w = B.DecoderWeights(seed=11, n_layers=2, distinct=2, vocab=8192, norm_noise=0.1)
    dec = V.Decoder(w.tok_emb, w.norm, [tuple(w.layer_w[i]) + tuple(w.layer_n[i]) for i in range(2)], ada_scale=w.ada_scale,
                    vocab=w.vocab)
    st = dec.state(kv_cap=64)
    with pytest.raises(V.VoxCudaError, match="no decode step"):
        st.token_logprobs(0)
    st.prefill(B.normal_f32((40, B.DEC_DIM), 12))
    for i in range(20):
        tok, logits = st.step(B.normal_f32(B.DEC_DIM, 13 + i))
    p = logits.astype(np.float64)
    p = p - p.max() - np.log(np.exp(p - p.max()).sum())
    lp, ent, ids, top = st.token_logprobs(77, 4)
    tol = 8 * U32 * (np.abs(p).max() + 1)
    assert abs(lp - p[77]) <= tol and abs(ent + (np.exp(p) * p).sum()) <= tol
    assert ids[0] == tok and ids.tolist() == np.argsort(-logits, kind="stable")[:4].tolist()
    assert np.abs(top - p[ids]).max() <= tol
    assert st.token_logprobs(0)[2].size == 0
    c = st.kv_cache()
    assert (c.n_layers, c.n_streams, c.cap, c.n_kv_heads, c.head_dim, c.n_sink) == (2, 1, 64, 8, 128, 0)
    k, v = st.read_kv(1, 0, 60)
    q = torch.randn(1, 32, 128).cuda()
    out, pos = torch.empty_like(q), ints([st.position - 1])
    V.attention_window_dev(c, 1, V.Rows(ptr(pos), n_rows=1), q.data_ptr(), 32, 0, 0.0, out.data_ptr(), None, V.STREAM_LEGACY)
    dk, dv, ref = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.empty_like(q)
    V.attention_decode_dev(q.data_ptr(), dk.data_ptr(), dv.data_ptr(), 60, 59, ref.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    # each is off by at most (128 + 8) u S of a weight; S from the values
    kk, big = dk.view(60, 8, 128).abs().double(), 0.0
    for h in range(32):
        big = max(big, float((kk[:, h // 4] @ q[0, h].abs().double()).max()) / math.sqrt(128))
    tol = 4 * ((136 * U32) * big + 2.0 ** -22) * float(dv.abs().max())
    assert float((out - ref).abs().max()) <= tol
    st.free()
    dec.free()
