"""Strides of 0 beside given ones, in a paged cache whose heads lie inside its slots."""
import pytest
import torch

import voxcuda as V
from paged_ref import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[1, 1], [40, 17]])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages_of_slots_of_heads(counts, dim):
    """[layer][page][slot][head][dim]: with the strides of slots and heads given, pages and layers follow by themselves."""
    V.init()
    c = Case("bf16", 8, 2, dim, 16, [70, 29], counts, layers=2, layer=1, seed=5)
    pool = c.pool
    k, v = (code.permute(0, 1, 3, 2, 4).contiguous().cuda() for code in pool.code)
    cache = V.PagedCache(k.data_ptr(), v.data_ptr(), pool.dks.data_ptr(), pool.dvs.data_ptr(), c.dtable.data_ptr(), c.dtable.shape[1],
                         2, pool.pages, 16, 2, 2, dim, slot_stride=2 * dim, head_stride=dim)
    out, lse = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    V.attention_paged_dev(cache, 1, c.rows(V), c.dq.data_ptr(), "bf16", 8, 0, 0, 0.0, out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    c.check(out, lse)
