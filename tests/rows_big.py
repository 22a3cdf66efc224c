"""Cases of the row attention with many rows and keys: the definition in 64
bits on the GPU, all keys of a stream at once."""
import math

import torch

from rows_ref import TORCH, U32, depths, half_step, slot


class Big:
    """One layer of a cache with several streams' rows.  Slots that no row sees
    hold NaN.  shape: 'random', or scores in log2 units that 'rise' or 'fall'
    along the keys: every 16th key is large for a quarter of the rows (by
    packed row), each `step` keys by 9, 5, 12 or 3 more than before."""

    def __init__(self, dtype, heads, kv_heads, dim, cap, n_sink, positions, counts, window=0, tree=None, seed=0, shape="random",
                 step=64):
        self.__dict__.update(dtype=dtype, heads=heads, kv=kv_heads, dim=dim, cap=cap, n_sink=n_sink, window=window,
                             positions=positions, counts=counts, shape=shape)
        t, dev, streams = TORCH[dtype], "cuda", len(positions)
        g = torch.Generator(device=dev).manual_seed(seed)
        rng = torch.Generator().manual_seed(seed)
        self.n = sum(counts)
        self.start = [sum(counts[:s]) for s in range(streams + 1)]
        self.parents = None
        if tree:
            self.parents = [[max(i - f, -1) for i, f in enumerate(torch.randint(1, tree + 1, (n,), generator=rng).tolist())]
                            for n in counts]
        q = torch.randn(self.n, heads, dim, generator=g, device=dev)
        k = torch.randn(streams, cap, kv_heads, dim, generator=g, device=dev)
        v = torch.randn(streams, cap, kv_heads, dim, generator=g, device=dev)
        self.scale = 0.0
        if shape == "random":
            q *= 2
        else:
            self.scale = math.log(2.0)   # a score in log2 units is q.k
            q, k = 0.1 * q, 0.3 * k
            kind = (torch.arange(self.n * heads, device=dev) % 4).view(self.n, heads, 1)
            q[..., :4] = (torch.arange(4, device=dev) == kind).float()
        self.key_pos, self.see = [], []
        hide = torch.ones(streams, cap, dtype=torch.bool)
        for s, (p, n) in enumerate(zip(positions, counts)):
            end, ring = p + n, cap - n_sink
            j = torch.tensor([] if p < 0 or n == 0 else list(range(min(end, n_sink))) + list(range(max(n_sink, end - ring), end)), dtype=torch.long)
            self.key_pos.append(j)
            i = torch.arange(n)
            if tree:
                dep = torch.tensor(depths(self.parents[s]), dtype=torch.long)
                line = torch.zeros(n, n, dtype=torch.bool)
                for a in range(n):
                    line[a, a] = True
                    if self.parents[s][a] >= 0:
                        line[a] |= line[self.parents[s][a]]
                node = (j - p).clamp(min=0)
                logical = torch.where(j >= p, p + dep[node], j)
                here = p + dep
                see = torch.where((j >= p)[None], line[:, node], torch.ones(1, dtype=torch.bool))
            else:
                logical, here = j, p + i
                see = j[None] <= here[:, None]
            if window:
                see &= (logical[None] > here[:, None] - window) | (logical < n_sink)[None]
            self.see.append(see.cuda())
            at = torch.tensor([slot(x, cap, n_sink) for x in j.tolist()], dtype=torch.long)
            if len(j):
                hide[s, at[see.any(0)]] = False
            if shape != "random" and len(j):
                order = torch.arange(len(j)) if shape == "rise" else torch.arange(len(j) - 1, -1, -1)
                heights = torch.cumsum(torch.tensor([9.0, 5.0, 12.0, 3.0]).repeat(len(j) // step // 4 + 1), 0)
                large = (order % 16 == 5).nonzero().squeeze(1)
                k[s, at[large].cuda(), :, :4] = 0.0
                k[s, at[large].cuda(), :, (order[large] // 16 % 4).cuda()] = heights[order[large] // step].cuda()[:, None]
        hide = hide.cuda()[:, :, None, None]
        self.k, self.v, self.q = k.masked_fill(hide, math.nan).to(t), v.masked_fill(hide, math.nan).to(t), q.to(t)
        self.dpos = torch.tensor(positions, dtype=torch.int32, device=dev)
        self.dstart = torch.tensor(self.start, dtype=torch.int32, device=dev)
        self.dparent = None if not tree else torch.tensor([x for row in self.parents for x in row], dtype=torch.int32, device=dev)

    def args(self, V):
        return (V.KvCache(self.k.data_ptr(), self.v.data_ptr(), self.dtype, 1, len(self.positions), self.cap, self.kv, self.dim,
                          self.n_sink),
                V.Rows(self.dpos.data_ptr(), self.dstart.data_ptr(), None if self.dparent is None else self.dparent.data_ptr(),
                       self.n, max(self.counts)))

    def form(self, V):
        cache, rows = self.args(V)
        return V.attention_plan(cache, rows, self.heads, self.window)

    def run(self, V):
        cache, rows = self.args(V)
        out, lse = torch.full_like(self.q, 7.0), torch.full((self.n, self.heads), 7.0, device="cuda")
        call = V.attention_window_dev if self.dparent is None else V.attention_tree_dev
        call(cache, 0, rows, self.q.data_ptr(), self.heads, self.window, self.scale, out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY)
        torch.cuda.synchronize()
        return out, lse

    def check(self, out, lse, skip=()):
        """rows_ref.Case.check's bounds, all rows of a stream at once, but for
        two: fp16 weights may be off by 2^-32 of the row's largest, and an
        addition on the tensor cores, which may cut, by 2 u.  Columns in `skip`
        are left out."""
        scale = self.scale or 1.0 / math.sqrt(self.dim)
        u, group, rounded = half_step(self.dtype), self.heads // self.kv, self.dtype != "fp32"
        keep = [d for d in range(self.dim) if d not in skip]
        for s, (p, n) in enumerate(zip(self.positions, self.counts)):
            a, b = self.start[s], self.start[s] + n
            if n == 0:
                continue
            if p < 0:
                assert bool((out[a:b] == 7.0).all()) and bool((lse[a:b] == 7.0).all())
                continue
            at = torch.tensor([slot(x, self.cap, self.n_sink) for x in self.key_pos[s].tolist()], device="cuda")
            see = self.see[s]
            some = see.any(0)
            number = see.sum(1).double()[:, None]
            for h in range(self.heads):
                k, v = self.k[s, at, h // group].double(), self.v[s, at, h // group].double()
                k, v = torch.where(some[:, None], k, 0.0), torch.where(some[:, None], v, 0.0)[:, keep]
                q = self.q[a:b, h].double()
                z = (q @ k.T * scale).masked_fill(~see, -math.inf)
                big = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(~see, 0.0).amax(1, keepdim=True)
                lz = torch.logsumexp(z, 1, keepdim=True)
                want = (z - lz).exp() @ v
                most = v.abs().max()
                d = (self.dim + 8) * U32 * big + 2.0 ** -22 + (2.0 ** -18 if rounded else 0.0)
                tol = (2 * d + (2 if rounded else 1) * number * U32 + (u if rounded else 0.0)
                       + (number * 2.0 ** -32 if self.dtype == "fp16" else 0.0)) * most + u * want.abs() + 1e-30
                err = (out[a:b, h].double()[:, keep] - want).abs()
                assert bool((err <= tol).all()), (s, h, float((err / tol).nan_to_num(nan=1e9).max()))
                err = (lse[a:b, h, None].double() - lz).abs()
                assert bool((err <= d + number * U32 + 4 * U32 * lz.abs()).all()), (s, h, "lse", float(err.max()))
