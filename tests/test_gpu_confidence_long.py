"""Long rows in the kernel of many rows, where a slot of batch maxima serves
several batches."""
import pytest
import torch

import voxcuda as V
from test_gpu_confidence import check, rows, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n_top", [1, 32])
def test_many_long_rows(dtype, n_top):
    x, tok = rows(160, 150001, dtype, seed=41)
    span = 2048 * (1 if dtype == "fp32" else 2)     # logits of a batch of the CTA's 128 threads
    x[3, 7::16 * span], x[4, 5::32 * span] = 30.0, 31.0   # the best in batches that share a slot
    x[5, -40:] = 25.0
    x[6, : 40 * span : span] = 20.0
    check(x, tok, n_top, dtype, run(x, tok, n_top, dtype))
