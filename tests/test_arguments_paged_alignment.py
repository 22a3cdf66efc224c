"""Arrays of whole numbers that are not aligned as such - a table, pages to copy,
positions, row ranges, parents - are refused, not read.  CPU only: the addresses are
never read."""
import pytest

import voxcuda as V
from test_arguments_paged import A, append, attend, copy, pool, rows


def slab_rows(**kw):
    d = dict(pos=A, row_start=A, parent=None, n_rows=6, max_rows=4)
    d.update(kw)
    return V.Rows(**d)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_tables(off):
    c = pool(table=5 * A + off)
    assert attend(c) == V.ERR_ARG and append(c) == V.ERR_ARG and "aligned" in V.last_error()
    plan = (V.C.c_int * 3)()
    assert V.lib().vox_cuda_selftest_attention_paged_plan(c, rows(), 1, 8, 0, 0, plan) == V.ERR_ARG
    assert copy(pool(table=5 * A + off), n=0, src=None, dst=None) == V.OK   # which asks for no table


@pytest.mark.parametrize("off", [1, 2, 3])
def test_copies(off):
    assert copy(src=A + off) == V.ERR_ARG and "aligned" in V.last_error()
    assert copy(dst=2 * A + off) == V.ERR_ARG and "aligned" in V.last_error()


@pytest.mark.parametrize("bad", [dict(pos=A + 2), dict(row_start=A + 1), dict(row_start=A + 2)])
def test_rows(bad):
    assert attend(r=rows(**bad)) == V.ERR_ARG and append(r=rows(**bad)) == V.ERR_ARG and "aligned" in V.last_error()


@pytest.mark.parametrize("bad", [dict(pos=A + 2), dict(row_start=A + 1), dict(parent=A + 2)])
def test_rows_of_a_slab(bad):
    """The slab's operators check their rows by the same rules."""
    c = V.KvCache(A, 2 * A, dtype="bf16", n_layers=1, n_streams=3, cap=64, n_kv_heads=2, head_dim=64)
    tree = dict(parent=3 * A) | bad
    f = V.lib().vox_cuda_attention_tree_dev
    assert f(c, 0, slab_rows(**tree), 4 * A, 8, 0, 0.0, 5 * A, None, None) == V.ERR_ARG and "aligned" in V.last_error()
