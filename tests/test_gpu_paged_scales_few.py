"""Attention of a few rows over a paged cache whose pages' V stand far apart: a row's
result goes by the scales that it sees alone."""
import pytest

import paged_scales as S
import voxcuda as V

pytestmark = pytest.mark.gpu

# form; heads, kv, dim, page; rows of the streams looked at; positions of others, whose tables make the plan
FORMS = [
    ((8, 2), 8, 2, 128, 16, [24], []), ((8, 2), 8, 2, 128, 16, [24], [310]), ((8, 2), 8, 2, 64, 16, [24], []),
    ((8, 2), 12, 12, 64, 32, [50], []), ((8, 1), 8, 2, 128, 16, [30], [1590, 1580, 1570]), ((8, 1), 4, 4, 128, 16, [24], [3190]),
    ((8, 1), 12, 12, 64, 16, [20], [1590, 1590, 1590]), ((8, 3), 16, 16, 128, 16, [20], [1590]), ((16, 2), 16, 4, 128, 16, [24], [1590])]


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
    S.others_pages_change_nothing(dtype, form, heads, kv, dim, page, counts, far)
