"""The operators over a paged cache refuse what they cannot do before they
touch a device.  CPU only: the addresses are never read."""
import pytest

import voxcuda as V

A = 1 << 24   # an aligned address


def pool(**kw):
    d = dict(k=A, v=2 * A, k_scale=3 * A, v_scale=4 * A, table=5 * A, table_stride=4, n_layers=2, n_pages=20, page_size=16, n_streams=3,
             n_kv_heads=2, head_dim=64)
    d.update(kw)
    return V.PagedCache(**d)


def rows(**kw):
    d = dict(pos=A, row_start=A, parent=None, n_rows=6, max_rows=4)
    d.update(kw)
    return V.Rows(**d)


def attend(c=None, r=None, layer=0, q=A, type=1, heads=8, window=0, sinks=0, scale=0.0, out=8 * A, lse=None):
    return V.lib().vox_cuda_attention_paged_dev(c or pool(), layer, r or rows(), q, type, heads, window, sinks, scale, out, lse, None)


def append(c=None, r=None, layer=0, qkv=A, type=0, heads=8, stride=0, gq=None, eps=1e-5, theta=1e6, q_out=64 * A, q_type=1):
    return V.lib().vox_cuda_rope_append_paged_dev(c or pool(), layer, r or rows(), qkv, type, heads, stride, gq, None, eps, theta,
                                                  q_out, q_type, None)


def copy(c=None, src=A, dst=2 * A, n=3):
    return V.lib().vox_cuda_kv_copy_pages_dev(c or pool(), src, dst, n, None)


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=A + 8), dict(v=A + 4), dict(k_scale=A + 2),
    dict(v_scale=A + 1), dict(n_layers=0), dict(n_layers=40000), dict(n_pages=0), dict(page_size=0), dict(page_size=48),
    dict(page_size=256), dict(page_size=-16), dict(n_kv_heads=0), dict(n_kv_heads=5000), dict(head_dim=96), dict(head_dim=256),
    dict(slot_stride=65), dict(slot_stride=48), dict(head_stride=72), dict(page_stride=-1024), dict(layer_stride=1 << 60)])
def test_pools(bad):
    c = pool(**bad)
    for call in (attend, append, copy):
        assert call(c) == V.ERR_ARG and V.last_error(), bad


@pytest.mark.parametrize("bad", [dict(table=None), dict(table_stride=0), dict(table_stride=(1 << 26) + 1), dict(n_streams=0),
                                 dict(n_streams=70000)])
def test_tables(bad):
    c = pool(**bad)
    assert attend(c) == V.ERR_ARG and append(c) == V.ERR_ARG and V.last_error()


@pytest.mark.parametrize("bad,code", [
    (dict(pos=None), V.ERR_ARG), (dict(parent=A), V.ERR_ARG), (dict(n_rows=-1), V.ERR_ARG), (dict(max_rows=0), V.ERR_ARG),
    (dict(max_rows=7), V.ERR_ARG), (dict(row_start=None), V.ERR_ARG), (dict(n_rows=100, max_rows=65), V.ERR_CAPACITY)])
def test_rows(bad, code):
    r = rows(**bad)
    assert attend(r=r) == code and append(r=r) == code and V.last_error()


def test_none():
    assert attend(r=rows(n_rows=0, max_rows=0), q=None, out=None) == V.OK
    assert append(r=rows(n_rows=0, max_rows=0), qkv=None, q_out=None) == V.OK
    assert copy(n=0, src=None, dst=None) == V.OK
    f = V.lib().vox_cuda_attention_paged_dev
    assert f(None, 0, rows(), A, 1, 8, 0, 0, 0.0, 8 * A, None, None) == V.ERR_ARG
    assert f(pool(), 0, None, A, 1, 8, 0, 0, 0.0, 8 * A, None, None) == V.ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(layer=-1), dict(layer=2), dict(heads=0), dict(heads=7), dict(heads=2 * 65), dict(type=0), dict(type=3), dict(window=-1),
    dict(sinks=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(q=None), dict(out=None), dict(q=A + 8),
    dict(out=A + 2), dict(lse=A + 2), dict(out=A + 16), dict(lse=A), dict(lse=8 * A + 4)])
def test_attention(bad):
    assert attend(**bad) == V.ERR_ARG and V.last_error(), bad


@pytest.mark.parametrize("bad", [
    dict(layer=2), dict(heads=3), dict(q_type=0), dict(q_type=5), dict(type=2), dict(type=-1), dict(stride=700), dict(stride=769),
    dict(stride=1 << 41), dict(eps=-1.0), dict(eps=float("nan")), dict(theta=-1.0), dict(theta=float("inf")), dict(qkv=None),
    dict(qkv=A + 4), dict(q_out=None), dict(q_out=A + 16), dict(gq=A + 4)])
def test_append(bad):
    assert append(**bad) == V.ERR_ARG and V.last_error(), bad


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=21), dict(src=None), dict(dst=None)])
def test_copies(bad):
    assert copy(**bad) == V.ERR_ARG and V.last_error(), bad


def test_a_form_is_asked_for_rows():
    plan = (V.C.c_int * 3)()
    f = V.lib().vox_cuda_selftest_attention_paged_plan
    assert f(pool(), rows(), 1, 8, 0, 0, None) == V.ERR_ARG and f(pool(), None, 1, 8, 0, 0, plan) == V.ERR_ARG
    assert f(None, rows(), 1, 8, 0, 0, plan) == V.ERR_ARG and f(pool(), rows(n_rows=0, max_rows=0), 1, 8, 0, 0, plan) == V.ERR_ARG
    assert f(pool(), rows(), 0, 8, 0, 0, plan) == V.ERR_ARG and f(pool(), rows(), 1, 7, 0, 0, plan) == V.ERR_ARG
    assert f(pool(), rows(), 1, 8, -1, 0, plan) == V.ERR_ARG and f(pool(), rows(), 1, 8, 0, -1, plan) == V.ERR_ARG
