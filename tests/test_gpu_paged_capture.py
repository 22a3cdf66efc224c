"""Paged append, attention and copies whose first call in a process is inside a
capture write what eager calls write; pools beyond 4 GB; several host
threads at once."""
import subprocess
import sys
import threading

import pytest
import torch

import voxcuda as V
from conftest import ROOT
from paged_ref import Case, from_e4m3

pytestmark = pytest.mark.gpu

CODE = """
import sys, torch
sys.path[:0] = ["tests", "voxtral.c_b200"]
import voxcuda as V
V.init()
dev = "cuda"
T = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)
sets = []
for src, qt in (("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")):
    for dim in (64, 128):
        for rows in (1, 5, 40, 70):          # few rows and many
            pool = [torch.zeros(2, 30, 2, 16, dim, dtype=torch.uint8, device=dev) for _ in range(2)]
            scale = [torch.ones(2, 30, 2, device=dev) for _ in range(2)]
            qkv = torch.randn(2 * rows, 8, dim, device=dev).to(T[src])
            q = torch.zeros(2 * rows, 4, dim, device=dev, dtype=T[qt])
            one = (*pool, *scale, q, torch.zeros_like(q), torch.zeros(2 * rows, 4, device=dev))
            start = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=dev)
            sets.append((src, qt, dim, rows, qkv, start, [one, tuple(t.clone() for t in one)]))
table = torch.tensor([list(range(0, 12)), list(range(12, 24))], dtype=torch.int32, device=dev)
pos, a, b = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([5, 30], [0, 13], [25, 29]))
torch.cuda.synchronize()

def go(which, st):
    for src, qt, dim, rows, qkv, start, copies in sets:
        k, v, ks, vs, q, out, lse = copies[which]
        c = V.PagedCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(), 12, 2, 30, 16, 2, 2, dim)
        r = V.Rows(pos.data_ptr(), start.data_ptr(), None, 2 * rows, rows)
        V.rope_append_paged_dev(c, 1, r, qkv.data_ptr(), src, 4, 0, None, None, 0.0, 1e4, q.data_ptr(), qt, st)
        V.attention_paged_dev(c, 1, r, q.data_ptr(), qt, 4, 0, 0, 0.0, out.data_ptr(), lse.data_ptr(), st)
        V.kv_copy_pages_dev(c, a.data_ptr(), b.data_ptr(), 2, st)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    go(0, torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()
assert not any(bool((x[0][5] != 0).any()) for *_, x in sets)   # nothing ran yet
g.replay()
torch.cuda.synchronize()
go(1, V.STREAM_LEGACY)
torch.cuda.synchronize()
for *_, (x, y) in sets:
    assert all(torch.equal(s, t) for s, t in zip(x, y)) and bool((x[5] != 0).any())
print("captured")
"""


@pytest.fixture(scope="module", autouse=True)
def cuda():
    V.init()
    yield


def test_first_calls_inside_a_capture_write_what_eager_ones_do():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_pools_beyond_four_gigabytes(rows):
    """Pages whose offsets pass 32 bits."""
    c = Case("bf16", 8, 2, 128, 64, [150], [rows], seed=3)
    want, want_lse = c.run(V)
    pages = 300000                            # 64 KB of K each: 4.9 GB a tensor, and as much of V
    big = [torch.empty(1, pages, 2, 64, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(1, pages, 2, device="cuda") for _ in range(2)]
    there = [p for p in c.table[0] if 0 <= p < c.pool.pages]
    moved = {p: pages - 1 - 1000 * i for i, p in enumerate(there)}
    for t, s, code, scale in zip(big, scales, (c.pool.dk, c.pool.dv), (c.pool.dks, c.pool.dvs)):
        for p, m in moved.items():
            t[0, m], s[0, m] = code[0, p], scale[0, p]
    table = torch.tensor([[moved.get(p, -1) for p in c.table[0]]], dtype=torch.int32).cuda()
    cache = V.PagedCache(big[0].data_ptr(), big[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), table.data_ptr(),
                         table.shape[1], 1, pages, 64, 1, 2, 128)
    out, lse = torch.full_like(c.dq, 7.0), torch.full(c.dq.shape[:2], 7.0, device="cuda")
    V.attention_paged_dev(cache, 0, c.rows(V), c.dq.data_ptr(), "bf16", 8, 0, 0, 0.0, out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    # an append to the same pages, and a copy of the last one
    qkv, q = torch.randn(rows, 12, 128).cuda(), torch.empty_like(c.dq)
    V.rope_append_paged_dev(cache, 0, c.rows(V), qkv.data_ptr(), "fp32", 8, 0, None, None, 0.0, 0.0, q.data_ptr(), "bf16", V.STREAM_LEGACY)
    last = moved[c.table[0][(150 + rows - 1) // 64]]
    a, b = (torch.tensor([x], dtype=torch.int32).cuda() for x in (last, pages // 2 + 7))
    V.kv_copy_pages_dev(cache, a.data_ptr(), b.data_ptr(), 1, V.STREAM_LEGACY)
    torch.cuda.synchronize()
    at = 150 + rows - 1
    held = from_e4m3(big[1][0, last, :, at % 64].cpu()) * scales[1][0, last].cpu().double()[:, None]
    assert bool(((held - qkv[-1, 10:].double().cpu()).abs() <= 2.0 ** -4 * qkv[-1, 10:].double().cpu().abs() + 2.0 ** -10).all())
    assert torch.equal(big[0][0, pages // 2 + 7], big[0][0, last]) and torch.equal(scales[1][0, pages // 2 + 7], scales[1][0, last])


def test_threads_at_once():
    """Calls from several host threads, each on its own stream."""
    cases = [Case("bf16", 8, 2, 128, 16, [300 + 50 * i], [(1, 6, 40, 200)[i]], seed=40 + i) for i in range(4)]
    got = {}

    def work(i):
        V.init()
        s = torch.cuda.Stream()
        got[i] = [cases[i].run(V, stream=s.cuda_stream) for _ in range(10)]
        s.synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        for out, lse in got[i]:
            assert torch.equal(out, got[i][0][0])
        c.check(*got[i][0])
