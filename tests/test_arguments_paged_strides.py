"""Strides of a paged cache that would put one element on another are refused.  CPU
only: the addresses are never read."""
import pytest

import voxcuda as V
from test_arguments_paged import append, attend, copy, pool

# 2 layers, 20 pages of 16 positions, 2 KV heads of 64
@pytest.mark.parametrize("bad", [
    dict(head_stride=64), dict(page_stride=64), dict(page_stride=1024), dict(page_stride=2032), dict(layer_stride=2048),
    dict(slot_stride=128, head_stride=64, page_stride=1024), dict(slot_stride=64, head_stride=512), dict(layer_stride=20 * 2048 - 16),
    dict(slot_stride=64, head_stride=1024, page_stride=2048, layer_stride=1024)])
def test_overlaps(bad):
    c = pool(**bad)
    for call in (attend, append, copy):
        assert call(c) == V.ERR_ARG and "apart" in V.last_error(), bad


@pytest.mark.parametrize("good", [
    dict(), dict(slot_stride=80), dict(slot_stride=128, head_stride=64), dict(slot_stride=128, head_stride=64, page_stride=2048),
    dict(page_stride=4096, layer_stride=2048),                       # layers inside pages
    dict(page_stride=64, slot_stride=20 * 64, head_stride=16 * 20 * 64, layer_stride=2 * 16 * 20 * 64),
    dict(n_pages=1, page_stride=64), dict(n_layers=1, layer_stride=64), dict(n_kv_heads=1, head_stride=64, slot_stride=64)])
def test_layouts(good):
    """Any order of the axes is a layout: nothing is asked of a device for an empty call."""
    assert copy(pool(**good), n=0, src=None, dst=None) == V.OK, V.last_error()
