"""More of what the row operators refuse before they touch a device.  CPU only."""
import pytest

import voxcuda as V
from test_arguments import A, cache, rows


@pytest.mark.parametrize("kw,wait", [(dict(), 5), (dict(dtype="bf16"), 0), (dict(dtype="bf16"), 10001), (dict(dtype="bf16", head_dim=96), 5)])
def test_the_wait_that_never_ends_has_a_limit(kw, wait):
    f = V.lib().vox_cuda_selftest_attention_timeout
    assert f(cache(**kw), 0, rows(), A, 8, A, None, wait, None) == V.ERR_ARG and V.last_error()


def test_a_form_is_asked_for_rows():
    plan = (V.C.c_int * 3)()
    f = V.lib().vox_cuda_selftest_attention_plan
    assert f(cache(), rows(), 8, 0, None) == V.ERR_ARG and f(None, rows(), 8, 0, plan) == V.ERR_ARG
    assert f(cache(), rows(n_rows=0, max_rows=0), 8, 0, plan) == V.ERR_ARG and f(cache(), None, 8, 0, plan) == V.ERR_ARG
    assert f(cache(), rows(), 7, 0, plan) == V.ERR_ARG and f(cache(), rows(), 8, -1, plan) == V.ERR_ARG


@pytest.mark.parametrize("tree", [False, True])
def test_attention_buffers_that_overlap(tree):
    f = V.lib().vox_cuda_attention_tree_dev if tree else V.lib().vox_cuda_attention_window_dev
    r = rows(parent=A) if tree else rows()
    size = 6 * 8 * 64 * 4                       # bytes of q: 6 rows of 8 heads of 64, fp32

    def call(q, out, lse=None):
        return f(cache(), 0, r, q, 8, 0, 0.0, out, lse, None)
    for q, out, lse in ((A, A + 16, None), (A + size - 16, A, None), (A, A + size, A), (A, A + size, A + 2 * size - 4),
                        (A, A, A + size - 4), (A, A + size, A - 6 * 8 * 4 + 4)):
        assert call(q, out, lse) == V.ERR_ARG and "apart" in V.last_error()
