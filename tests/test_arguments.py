"""The row operators and the token log probabilities refuse what they cannot
do before they touch a device.  CPU only: the addresses are never read."""
import ctypes as C

import pytest

import voxcuda as V

A = 1 << 20   # an aligned address


def cache(**kw):
    d = dict(k=A, v=2 * A, dtype="fp32", n_layers=2, n_streams=3, cap=64, n_kv_heads=2, head_dim=64, n_sink=4)
    d.update(kw)
    return V.KvCache(**d)


def rows(**kw):
    d = dict(pos=A, row_start=A, parent=None, n_rows=6, max_rows=4)
    d.update(kw)
    return V.Rows(**d)


def attend(c=None, r=None, layer=0, q=A, heads=8, window=0, scale=0.0, out=A, tree=False):
    f = V.lib().vox_cuda_attention_tree_dev if tree else V.lib().vox_cuda_attention_window_dev
    return f(c or cache(), layer, r or rows(), q, heads, window, scale, out, None, None)


def append(c=None, r=None, qkv=A, type=0, heads=8, stride=0, eps=1e-5, theta=1e6, q_out=64 * A, gq=None):
    return V.lib().vox_cuda_rope_append_dev(c or cache(), 0, r or rows(), qkv, type, heads, stride, gq, None, eps, theta, q_out,
                                            None)


def commit(c=None, pos=A, path=2 * A, stride=4, took=3 * A, most=4, new=4 * A):
    return V.lib().vox_cuda_kv_commit_dev(c or cache(), pos, path, stride, took, most, new, None)


def fork(src, dst, c=None, n=None, pos=A):
    a, b = (C.c_int * max(1, len(src)))(*src), (C.c_int * max(1, len(dst)))(*dst)
    return V.lib().vox_cuda_kv_fork_dev(c or cache(), a, b, len(src) if n is None else n, pos, None)


def score(logits=A, type=0, n=2, vocab=100, stride=0, tokens=A, top=3, lp=A, ent=A, ids=A, tlp=A):
    return V.lib().vox_cuda_token_logprobs_dev(logits, type, n, vocab, stride, tokens, top, lp, ent, ids, tlp, None)


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(k=A + 4), dict(n_layers=0), dict(n_streams=0), dict(n_streams=70000), dict(cap=0),
    dict(n_kv_heads=0), dict(head_dim=96), dict(head_dim=256), dict(n_sink=-1), dict(n_sink=64), dict(slot_stride=129),
    dict(head_stride=32), dict(stream_stride=-1024), dict(layer_stride=1 << 60)])
def test_caches(bad):
    c = cache(**bad)
    for call in (lambda: attend(c), lambda: append(c), lambda: commit(c), lambda: fork([0], [1], c)):
        assert call() == V.ERR_ARG, bad
        assert V.last_error()


def test_unknown_types():
    c = cache()
    c.dtype = 3
    assert attend(c) == V.ERR_ARG
    assert append(type=1) == V.ERR_ARG          # bf16 rows for an fp32 cache
    assert append(cache(dtype="bf16"), type=2) == V.ERR_ARG
    assert score(type=7) == V.ERR_ARG
    with pytest.raises(KeyError):
        V.KvCache(A, A, "fp8")


@pytest.mark.parametrize("bad", [
    dict(pos=None), dict(n_rows=-1), dict(max_rows=0), dict(max_rows=7), dict(row_start=None),
    dict(row_start=None, n_rows=3, max_rows=2)])
def test_row_counts(bad):
    assert attend(r=rows(**bad)) == V.ERR_ARG and append(r=rows(**bad)) == V.ERR_ARG


def test_what_a_ring_or_a_tree_cannot_hold():
    assert attend(r=rows(n_rows=100, max_rows=61)) == V.ERR_CAPACITY
    assert append(r=rows(n_rows=100, max_rows=61)) == V.ERR_CAPACITY
    assert "cannot hold" in V.last_error()
    big = cache(cap=1000)
    assert attend(big, rows(n_rows=300, max_rows=257, parent=A), tree=True) == V.ERR_ARG
    assert append(big, rows(n_rows=300, max_rows=257, parent=A)) == V.ERR_ARG
    assert attend(tree=True) == V.ERR_ARG                # a tree without parents
    assert attend(r=rows(parent=A)) == V.ERR_ARG         # a window with parents


@pytest.mark.parametrize("bad", [
    dict(layer=2), dict(layer=-1), dict(q=None), dict(q=A + 8), dict(out=None), dict(out=A + 8), dict(heads=0), dict(heads=7),
    dict(heads=130), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38)])
def test_attention_arguments(bad):
    assert attend(**bad) == V.ERR_ARG
    assert attend(r=rows(parent=A), tree=True, **bad) == V.ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(qkv=None), dict(qkv=A + 4), dict(q_out=None), dict(q_out=A + 4), dict(stride=12 * 64 - 4), dict(stride=12 * 64 + 2),
    dict(eps=-1.0), dict(eps=float("nan")), dict(theta=-1.0), dict(theta=float("inf")), dict(q_out=A + 64), dict(gq=A + 4),
    dict(heads=9)])
def test_append_arguments(bad):
    assert append(**bad) == V.ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(pos=None), dict(path=None), dict(took=None), dict(most=0), dict(most=257, stride=300), dict(stride=3), dict(new=A),
    dict(new=A + 8), dict(new=2 * A + 44), dict(new=3 * A)])
def test_commit_arguments(bad):
    assert commit(**bad) == V.ERR_ARG


def test_fork_arguments():
    assert fork([0], [0]) == V.ERR_ARG              # onto itself
    assert fork([0, 1], [2, 2]) == V.ERR_ARG        # written twice
    assert fork([0, 1], [1, 2]) == V.ERR_ARG        # read and written
    assert fork([0], [3]) == V.ERR_ARG and fork([-1], [1]) == V.ERR_ARG
    assert fork([0], [1], pos=None) == V.ERR_ARG and fork([], [], n=65) == V.ERR_ARG and fork([], [], n=-1) == V.ERR_ARG
    with pytest.raises(ValueError):
        V.kv_fork_dev(cache(), [0], [1, 2], A)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(logits=A + 2), dict(n=-1), dict(vocab=0), dict(stride=99), dict(top=33), dict(top=-1),
    dict(vocab=2, stride=2), dict(ids=None), dict(top=0), dict(tokens=None), dict(lp=None),
    dict(tokens=None, lp=None, ent=None, top=0, tlp=None, ids=None)])
def test_logprob_arguments(bad):
    assert score(**bad) == V.ERR_ARG


def test_nothing_to_do_is_no_error():
    empty = rows(n_rows=0, max_rows=0)
    assert attend(r=empty, q=None, out=None) == V.OK and append(r=empty, qkv=None, q_out=None) == V.OK
    assert fork([], []) == V.OK and score(n=0) == V.OK


def test_decoder_state_entries():
    f, i = (C.c_float * 4)(), (C.c_int * 4)()
    assert V.lib().vox_cuda_decoder_token_logprobs(None, 0, 0, f, f, i, f) == V.ERR_ARG
    assert V.lib().vox_cuda_dec_state_kv_cache(None, V.KvCache()) == V.ERR_ARG
