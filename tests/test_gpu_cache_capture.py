"""Append, commit and fork whose first call in a process is inside a capture:
what they wrote is what eager calls write on copies."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import sys, torch
sys.path[:0] = ["tests", "voxtral.c_b200"]
import voxcuda as V
V.init()
dev = "cuda"
kinds = [(src, dt, dim) for src, dt in (("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp16")) for dim in (64, 128)]
T = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)
sets = []
for src, dt, dim in kinds:
    k, v = torch.randn(2, 3, 20, 2, dim, device=dev).to(T[dt]), torch.randn(2, 3, 20, 2, dim, device=dev).to(T[dt])
    qkv = torch.randn(3, 8, dim, device=dev).to(T[src])
    sets.append((src, dt, dim, qkv, [(k, v, torch.zeros(3, 4, dim, device=dev, dtype=T[dt])),
                                     (k.clone(), v.clone(), torch.zeros(3, 4, dim, device=dev, dtype=T[dt]))]))
pos = torch.tensor([5, 30, 0], dtype=torch.int32, device=dev)
path, took = torch.tensor([[1, 3], [0, 2], [4, 5]], dtype=torch.int32, device=dev), torch.tensor([2, 2, 1], dtype=torch.int32, device=dev)
new = [torch.zeros(3, dtype=torch.int32, device=dev) for _ in range(2)]
torch.cuda.synchronize()

def go(which, st):
    for src, dt, dim, qkv, copies in sets:
        k, v, q = copies[which]
        kv = V.KvCache(k.data_ptr(), v.data_ptr(), dt, 2, 3, 20, 2, dim, 1)
        V.rope_append_dev(kv, 1, V.Rows(pos.data_ptr(), n_rows=3), qkv.data_ptr(), src, 4, 0, None, None, 0.0, 1e4, q.data_ptr(), st)
        V.kv_commit_dev(kv, pos.data_ptr(), path.data_ptr(), 2, took.data_ptr(), 2, new[which].data_ptr(), st)
        V.kv_fork_dev(kv, [1], [2], pos.data_ptr(), st)

g = torch.cuda.CUDAGraph()
before = [(k.clone(), v.clone()) for *_, ((k, v, q), _) in sets]
with torch.cuda.graph(g):
    go(0, torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()
assert all(torch.equal(k, a) and torch.equal(v, b) for (*_, ((k, v, q), _)), (a, b) in zip(sets, before))   # nothing ran yet
g.replay()
torch.cuda.synchronize()
go(1, V.STREAM_LEGACY)
torch.cuda.synchronize()
for *_, (a, b) in sets:
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and bool((a[2] != 0).any())
assert not any(torch.equal(k, a) for (*_, ((k, v, q), _)), (a, b) in zip(sets, before))
assert new[0].tolist() == new[1].tolist() == [7, 32, 1]
print("captured")
"""


def test_first_calls_inside_a_capture_write_what_eager_ones_do():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
