"""More of what the row operators refuse before they touch a device.  CPU only."""
import pytest

import voxcuda as V
from test_arguments import A, cache, rows


@pytest.mark.parametrize("kw,wait", [(dict(), 5), (dict(dtype="bf16"), 0), (dict(dtype="bf16"), 10001), (dict(dtype="bf16", head_dim=96), 5)])
def test_the_wait_that_never_ends_has_a_limit(kw, wait):
    f = V.lib().vox_cuda_selftest_attention_timeout
    assert f(cache(**kw), 0, rows(), A, 8, A, None, wait, None) == V.ERR_ARG and V.last_error()
