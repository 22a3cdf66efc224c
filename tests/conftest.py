"""Shared test setup: the `gpu` marker, import paths and golden-file access."""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for sub in ("oracle", os.path.join("tests", "golden"), "voxtral.c_b200"):
    p = os.path.join(ROOT, sub)
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


def reference_sources():
    """Whether the reference's tree is on this machine (the condition under
    which __graft_entry__.build() builds its host; an empty folder is none)."""
    return os.path.isfile(os.path.join(os.environ.get("VOX_REFERENCE_DIR", "/root/reference"), "voxtral.c"))


def pytest_collection_modifyitems(items):
    """What needs the reference's sources, or its host built from them, is
    skipped where there are none."""
    if reference_sources():
        return
    host = os.path.exists(os.path.join(ROOT, "integration", "_build", "libvoxhost_cuda.so"))
    skip = pytest.mark.skip(reason="the reference's sources are not on this machine")
    for item in items:
        name = os.path.basename(str(item.fspath))
        if item.name in ("test_hooks_land_once_each", "test_a_moved_anchor_stops_the_build") or (name == "test_gpu_host_cuda.py" and not host):
            item.add_marker(skip)


def load_golden(name):
    return np.load(os.path.join(ROOT, "tests", "golden", name + ".npz"))


def unpack(g, prefix):
    """(indices, values, full-norm, size) of a packed golden output."""
    return g[prefix + "_idx"], g[prefix + "_val"], float(g[prefix + "_norm"]), int(g[prefix + "_size"])


@pytest.fixture(scope="session")
def golden():
    return load_golden
