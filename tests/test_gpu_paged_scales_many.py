"""Attention of many rows over a paged cache whose pages' V stand far apart: a row's
result goes by the scales that it sees alone."""
import pytest
import torch

import paged_scales as S
import voxcuda as V
from paged_ref import NAN8, Case

pytestmark = pytest.mark.gpu

# form; heads, kv, dim, page; rows of the streams looked at; positions of others, whose tables make the plan
FORMS = [
    ((128, 2), 8, 2, 128, 16, [60], []), ((128, 2), 8, 2, 64, 16, [60], []), ((128, 2), 12, 12, 64, 16, [128], [1590]),
    ((128, 2), 16, 4, 128, 64, [90], []), ((256, 1), 8, 2, 128, 16, [60], [1590]), ((256, 1), 8, 2, 128, 32, [200] * 12, []),
    ((256, 1), 8, 2, 64, 16, [60], [1590]), ((256, 1), 12, 12, 64, 64, [200] * 12, [])]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


@pytest.mark.parametrize("form,heads,kv,dim,page,counts,far", FORMS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_small_first_page(dtype, form, heads, kv, dim, page, counts, far):
    S.small_first_page(dtype, form, heads, kv, dim, page, counts, far)


@pytest.mark.parametrize("form,heads,kv,dim,page,counts,far", FORMS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_page_left_behind(dtype, form, heads, kv, dim, page, counts, far):
    S.large_page_left_behind(dtype, None, heads, kv, dim, page, counts, far)   # (a window makes other plans)


@pytest.mark.parametrize("form,heads,kv,dim,page,counts,far", FORMS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_zeros_take_the_weight(dtype, form, heads, kv, dim, page, counts, far):
    S.zeros_take_the_weight(dtype, form, heads, kv, dim, page, counts, far)


@pytest.mark.parametrize("form,heads,kv,dim,page,counts,far", FORMS)
def test_any_scales(form, heads, kv, dim, page, counts, far):
    S.any_scales(form, heads, kv, dim, page, counts, far)


@pytest.mark.parametrize("form,heads,kv,dim,page,counts,far", FORMS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_others_pages_change_nothing(dtype, form, heads, kv, dim, page, counts, far):
    S.others_pages_change_nothing(dtype, form, heads, kv, dim, page, counts, far, same_to=5)   # (2^14 times the rows' own)


@pytest.mark.parametrize("form,heads,kv,dim,page,counts,far", FORMS[:7])
def test_nan_and_lost_pages(form, heads, kv, dim, page, counts, far):
    """A NaN that only some rows see, and pages that are not there, among V scales far apart."""
    c = Case("bf16", heads, kv, dim, page, [page + 3] * len(counts) + far, counts + [1] * len(far), seed=8, lost=[(0, 2)])
    S.spread(c, lambda s, i: (-60, 90, 0, -3)[i % 4])
    want, want_lse = S.run(c, form)
    S.check(c, want, want_lse, some=[0])
    at = page + 13
    c.pool.code[1][0, c.table[0][1], 0, at % page, 5] = NAN8
    c.pool.upload()
    out, lse = S.run(c, form)
    hit = torch.isnan(out).cpu()
    seen = torch.zeros_like(hit)
    seen[at - page - 3:counts[0], :heads // kv, 5] = True
    assert torch.equal(hit, seen) and bool(((out == want) | torch.isnan(out)).all()) and torch.equal(lse, want_lse)
