"""The row operators' definitions in 64 bits, one row and one position at a
time, and the caches and rows that their tests use."""
import math

import torch

TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U32 = 2.0 ** -24


def half_step(dtype):
    """Half a step of the type, relative to the value."""
    return torch.finfo(TORCH[dtype]).eps / 2


def slot(j, cap, n_sink):
    return j if j < n_sink else n_sink + (j - n_sink) % (cap - n_sink)


def depths(parent):
    d = []
    for p in parent:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def ancestors(parent, i):
    out = set()
    while i >= 0:
        out.add(i)
        i = parent[i]
    return out


def visible(pos, n, i, cap, n_sink, window, parent=None):
    """The stored positions that row i of a stream's n rows sees."""
    last = pos + n - 1
    held = lambda j: j < n_sink or j > last - (cap - n_sink)   # noqa: E731
    if parent is None:
        p, lowest = pos + i, (pos + i - window + 1 if window else 0)
        return [j for j in range(p + 1) if held(j) and (j < n_sink or j >= lowest)]
    dep = depths(parent)
    p = pos + dep[i]
    lowest = p - window + 1 if window else 0
    seen = [j for j in range(pos) if held(j) and (j < n_sink or j >= lowest)]
    return seen + [pos + a for a in sorted(ancestors(parent, i)) if pos + dep[a] >= lowest or pos + dep[a] < n_sink]


def attention(q, k, v, keys, scale):
    """One row and head in 64 bits: (output, lse, largest sum |q||k| scale)."""
    if not keys:
        return torch.zeros(v.shape[-1], dtype=torch.float64), -math.inf, 0.0
    s = (k @ q) * scale
    lse = torch.logsumexp(s, 0)
    return (s - lse).exp() @ v, float(lse), float((k.abs() @ q.abs()).max()) * abs(scale)


class Case:
    """A cache slab with several streams' rows in it, on the GPU, and the same
    values in 64 bits on the host.  Slots that no row sees hold NaN."""

    def __init__(self, dtype, heads, kv_heads, dim, cap, n_sink, positions, counts, window, seed=0, tree=None, layers=1,
                 layer=0, layout="slots", tail=0, scale_q=2.0):
        self.__dict__.update(dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, cap=cap, n_sink=n_sink, window=window,
                             positions=positions, counts=counts, layers=layers, layer=layer)
        g = torch.Generator().manual_seed(seed)
        t = TORCH[dtype]
        streams = len(positions)
        self.n = sum(counts)
        self.q = (torch.randn(self.n + tail, heads, dim, generator=g) * scale_q).to(t)
        shape = (layers, streams, cap, kv_heads, dim)
        k, v = torch.randn(shape, generator=g).to(t), torch.randn(shape, generator=g).to(t)
        self.parents = None
        if tree:
            self.parents = []
            for n in counts:
                far = torch.randint(1, tree + 1, (n,), generator=g).tolist()
                self.parents.append([max(i - f, -1) for i, f in zip(range(n), far)])
        seen = torch.zeros(streams, cap, dtype=torch.bool)
        self.keys = []
        for s, (p, n) in enumerate(zip(positions, counts)):
            rows = [] if p < 0 else [visible(p, n, i, cap, n_sink, window, self.parents and self.parents[s]) for i in range(n)]
            self.keys.append(rows)
            for r in rows:
                for j in r:
                    seen[s, slot(j, cap, n_sink)] = True
        hide = ~seen[None, :, :, None, None].expand(shape)
        self.k, self.v = k.masked_fill(hide, math.nan), v.masked_fill(hide, math.nan)
        order = {"slots": (0, 1, 2, 3, 4), "heads": (0, 1, 3, 2, 4), "streams_last": (2, 0, 3, 1, 4)}[layout]
        self.dk = self.k.permute(order).contiguous().cuda()
        self.dv = self.v.permute(order).contiguous().cuda()
        back = [order.index(d) for d in range(5)]
        self.strides = [self.dk.stride(d) for d in back]   # layer, stream, slot, head, dim
        start = [sum(counts[:s]) for s in range(streams + 1)]
        self.start = start
        self.dpos = torch.tensor(positions, dtype=torch.int32).cuda()
        self.dstart = torch.tensor(start, dtype=torch.int32).cuda()
        self.dparent = None
        if tree:
            flat = [p for row in self.parents for p in row] + [-1] * tail
            self.dparent = torch.tensor(flat, dtype=torch.int32).cuda()
        self.dq = self.q.cuda()

    def cache(self, V):
        st = self.strides
        return V.KvCache(self.dk.data_ptr(), self.dv.data_ptr(), self.dtype, self.layers, len(self.positions), self.cap,
                         self.kv_heads, self.dim, self.n_sink, st[0], st[1], st[2], st[3])

    def rows(self, V):
        return V.Rows(self.dpos.data_ptr(), self.dstart.data_ptr(), None if self.dparent is None else self.dparent.data_ptr(),
                      n_rows=self.dq.shape[0], max_rows=max(self.counts))

    def run(self, V, stream=None, scale=0.0, out=None):
        out = torch.full_like(self.dq, 7.0) if out is None else out
        lse = torch.full(self.dq.shape[:2], 7.0, device="cuda")
        call = V.attention_window_dev if self.dparent is None else V.attention_tree_dev
        call(self.cache(V), self.layer, self.rows(V), self.dq.data_ptr(), self.heads, self.window, scale, out.data_ptr(),
             lse.data_ptr(), V.STREAM_LEGACY if stream is None else stream)
        return out, lse

    def check(self, out, lse, scale=0.0, rounded_p=False):
        """Compares with the definition.  With u = 2^-24 and S the largest sum
        of |q||k| * scale of a row, a score is off by at most (dim + 4) u S
        (its products and sums, the scaled q), its exponential by as much, the
        2 ulp of ex2 and, where weights are rounded to 16 bits, the 2.7e-6 <
        2^-18 of a polynomial of degree 4 for 2^x.  So a weight is off by
        d = (dim + 8) u S + 2^-22 (+ 2^-18) relative; an output by 2 d max|v|
        (numerator and denominator), the sums' N u max|v|, half a step of a
        16-bit weight, and half a step of its own type."""
        out, lse = out.double().cpu(), lse.double().cpu()
        scale = scale or 1.0 / math.sqrt(self.dim)
        group = self.heads // self.kv_heads
        u = half_step(self.dtype)
        for s, rows in enumerate(self.keys):
            for i, keys in enumerate(rows):
                at = [slot(j, self.cap, self.n_sink) for j in keys]
                row = self.start[s] + i
                for h in range(self.heads):
                    k = self.k[self.layer, s, at, h // group].double()
                    v = self.v[self.layer, s, at, h // group].double()
                    o, z, big = attention(self.q[row, h].double(), k, v, keys, scale)
                    d = (self.dim + 8) * U32 * big + 2.0 ** -22 + (2.0 ** -18 if rounded_p else 0.0)
                    most = float(v.abs().max()) if keys else 0.0
                    tol = (2 * d + len(keys) * U32 + (u if rounded_p else 0.0)) * most + u * o.abs() + 1e-30
                    err = (out[row, h] - o).abs()
                    assert bool((err <= tol).all()), (s, i, h, float((err / tol).max()), self.positions[s])
                    tol_z = d + len(keys) * U32 + 4 * U32 * abs(z)
                    assert abs(float(lse[row, h]) - z) <= tol_z, (s, i, h, float(lse[row, h]), z)
        gone = [s for s, p in enumerate(self.positions) if p < 0]
        for s in gone:   # a stream that sits out
            assert bool((out[self.start[s]:self.start[s + 1]] == 7.0).all()), s
        assert bool((out[self.n:] == 7.0).all()) and bool((lse[self.n:] == 7.0).all())
