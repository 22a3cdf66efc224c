"""Many keys with small weights beside a large one: what each adds is below the
steps of a 16-bit weight, what they add together is not."""
import math

import pytest
import torch

import voxcuda as V
from rows_ref import TORCH, U32, half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("weight", [-22.0, -25.125, -28.0])
@pytest.mark.parametrize("rows,heads,dim,keys,large", [
    (1, 4, 64, 1 << 20, 1 << 17), (1, 4, 128, 1 << 19, 1 << 17),      # a token
    (600, 64, 64, 1 << 18, 1 << 18), (300, 64, 128, 1 << 18, 1 << 18),   # many rows: a tile's keys in one or few shares
    (9, 8, 64, 1 << 20, 1 << 17), (9, 8, 128, 1 << 19, 1 << 17)])
def test_keys_with_small_weights_count(dtype, weight, rows, heads, dim, keys, large):
    """Every `large`-th key has the score 0, the others `weight` (log2).  A
    weight is off by half a step of its type or, fp16, by 2^-32 of the row's
    largest.  A score is one product, so its weight is off by 4 u |s| and the
    2^-22 of ex2 or 2^-18 of the polynomial (rows_ref.Case.check).  The tensor
    cores bring each product to the exponent of the sum that it joins and may
    cut what lies below the sum's last place: 2 u of the sum for each key.  So
    a sum that holds the large keys' values (columns 0, 1) is good to 2 u N of
    its size only, one in which theirs are 0 (columns 2, 3) to 2 u N of the
    small keys'.  l adds the sums of 64 weights."""
    t = TORCH[dtype]
    k, v = torch.zeros(1, 1, keys, 1, dim, device="cuda"), torch.zeros(1, 1, keys, 1, dim, device="cuda")
    k[..., 0] = 1.0
    k[0, 0, ::large, 0, 0] = 0.0
    v[...] = -1.0
    v[0, 0, ::large] = 1.0
    v[..., 1] = torch.linspace(-1, 1, keys, device="cuda")[:, None]
    v[..., 2], v[..., 3] = 1.0, torch.linspace(0.25, 1, keys, device="cuda")[:, None]
    v[0, 0, ::large, 0, 2:4] = 0.0
    q = torch.zeros(rows, heads, dim, device="cuda")
    q[..., 0] = weight
    k, v, q = k.to(t), v.to(t), q.to(t)
    out, lse = torch.empty_like(q), torch.empty(rows, heads, device="cuda")
    pos, start = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([keys - rows], [0, rows]))
    V.attention_window_dev(V.KvCache(k.data_ptr(), v.data_ptr(), dtype, 1, 1, keys, 1, dim, 0), 0,
                           V.Rows(pos.data_ptr(), start.data_ptr(), None, rows, rows), q.data_ptr(), heads, 0, math.log(2.0),
                           out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    u = half_step(dtype)
    s = k[0, 0, :, 0, 0].double() * float(q[0, 0, 0])
    w = torch.exp2(s)
    z = torch.cumsum(w, 0)
    at = torch.arange(keys - rows, keys, device="cuda")
    lz = z[at].log()
    d = 4 * U32 * abs(weight) + 2.0 ** -22 + 2.0 ** -18
    steps_l = keys // 64 + 128
    for col in (0, 1, 2, 3):
        x = v[0, 0, :, 0, col].double()
        want, size = torch.cumsum(w * x, 0)[at] / z[at], torch.cumsum(w * x.abs(), 0)[at] / z[at]
        tol = (2 * d + u + (2 * keys + steps_l) * U32) * size + keys * 2.0 ** -32 * (dtype == "fp16") + u * want.abs()
        err = (out[..., col].double() - want[:, None]).abs()
        assert bool((err <= tol[:, None]).all()), (col, float((err / tol[:, None]).max()))
    assert bool(((lse.double() - lz[:, None]).abs() <= d + steps_l * U32 + 4 * U32 * lz[:, None].abs()).all())
