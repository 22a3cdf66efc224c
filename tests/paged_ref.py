"""The operators over a paged cache in e4m3 by their definitions in 64 bits,
and the caches that their tests use."""
import math

import torch

from rows_ref import TORCH, U32, half_step

E4M3 = torch.float8_e4m3fn
NAN8 = 0x7F           # e4m3's NaN
LEAST_EXP = -100      # of a scale
# the finite numbers of 0 and up, in order: number i has the code i
NUMBERS = torch.arange(NAN8, dtype=torch.uint8).view(E4M3).double()


def to_e4m3(x):
    """Codes of the nearest numbers, ties to the even code; NaN for what is not finite."""
    a = x.double().abs()
    hi = torch.searchsorted(NUMBERS, a.contiguous()).clamp(1, len(NUMBERS) - 1)
    down, up = a - NUMBERS[hi - 1], NUMBERS[hi] - a
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    code = torch.where(torch.isfinite(x), code, NAN8)
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def from_e4m3(code):
    return code.view(E4M3).double()


def scale_for(a):
    """2^e, e the smallest whole number >= LEAST_EXP with a <= 448 * 2^e."""
    e = LEAST_EXP
    if a > 0:
        m, x = math.frexp(a / 448.0)          # exact enough: a has 24 bits, and 448 * 2^e 3
        e = max(e, x if a > 448.0 * 2.0 ** (x - 1) else x - 1)
    return 2.0 ** e


def visible(p, window, n_sink, there):
    """The positions that the row at position p sees."""
    return [j for j in range(p + 1) if there(j) and (j < n_sink or not window or j > p - window)]


class Pool:
    """Pages of K and V on the GPU: random numbers under random scales, other
    slots, pages and scales NaN once `hide` is called with what is seen."""

    def __init__(self, layers, pages, page, kv, dim, seed=0, layout="heads", exps=(-8, -5)):
        g = torch.Generator().manual_seed(seed)
        self.shape = (layers, pages, kv, page, dim)
        self.layers, self.pages, self.page, self.kv, self.dim, self.layout = layers, pages, page, kv, dim, layout
        self.code = [to_e4m3((torch.randn(self.shape, generator=g) * 100).clamp(-448, 448)) for _ in range(2)]
        self.scale = [torch.exp2(torch.randint(*exps, self.shape[:3], generator=g).double()) for _ in range(2)]

    def hide(self, seen):
        """seen: truth values [pages][page]; what nobody sees becomes NaN, in every layer."""
        for code, scale in zip(self.code, self.scale):
            code.masked_fill_(~seen[None, :, None, :, None], NAN8)
            scale.masked_fill_(~seen.any(-1)[None, :, None], math.nan)

    def upload(self):
        order = {"heads": (0, 1, 2, 3, 4), "slots": (0, 1, 3, 2, 4), "pages_last": (2, 0, 3, 1, 4)}[self.layout]
        back = [order.index(d) for d in range(5)]
        dev = []
        for code in self.code:
            wide = code.permute(order).contiguous()
            if self.layout == "slots":        # and a gap behind every head
                wide = torch.cat((wide, torch.full_like(wide[..., :16], NAN8)), -1)
            dev.append(wide.cuda())
        self.dk, self.dv = dev
        self.strides = [self.dk.stride(d) for d in back]   # layer, page, head, slot
        self.back = back
        self.dks, self.dvs = (s.float().cuda() for s in self.scale)
        return self

    def held(self, which):
        """(codes, scales) of K (0) or V (1) as the GPU has them now."""
        d = (self.dk, self.dv)[which].cpu()[..., :self.dim].permute(self.back).contiguous()
        return d, (self.dks, self.dvs)[which].cpu().double()

    def cache(self, V, table):
        st = self.strides
        self.table = table
        return V.PagedCache(self.dk.data_ptr(), self.dv.data_ptr(), self.dks.data_ptr(), self.dvs.data_ptr(), table.data_ptr(),
                            table.shape[1], self.layers, self.pages, self.page, table.shape[0], self.kv, self.dim, st[0], st[1],
                            st[2], st[3])


def tables(counts, pages, seed=0, spare=1, filler=-1):
    """Pages for streams of so many positions, in any order; `filler` behind them."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    width = max(counts) + spare
    out = []
    for n in counts:
        out.append([order.pop() for _ in range(n)] + [filler] * (width - n))
    return out


class Case:
    """Streams' rows over a pool; slots, pages, scales and table entries that no row sees are NaN or nonsense."""

    def __init__(self, dtype, heads, kv, dim, page, positions, counts, window=0, n_sink=0, seed=0, layers=1, layer=0, layout="heads",
                 tail=0, scale_q=2.0, lost=(), exps=(-8, -5)):
        self.__dict__.update(dtype=dtype, heads=heads, kv=kv, dim=dim, page=page, positions=positions, counts=counts, window=window,
                             n_sink=n_sink, layer=layer)
        g = torch.Generator().manual_seed(seed)
        self.n = sum(counts)
        self.q = (torch.randn(self.n + tail, heads, dim, generator=g) * scale_q).to(TORCH[dtype])
        need = [-(-(max(p, 0) + n) // page) for p, n in zip(positions, counts)]
        pages = sum(need) + 3
        self.table = tables(need, pages, seed, filler=1 << 30)
        for s, i in lost:                                    # pages that are not there
            self.table[s][i] = -1 if i % 2 else pages + 7
        self.pool = Pool(layers, pages, page, kv, dim, seed, layout, exps)
        seen = torch.zeros(pages, page, dtype=torch.bool)
        self.keys = []
        for s, (p, n) in enumerate(zip(positions, counts)):
            there = lambda j: 0 <= self.table[s][j // page] < pages   # noqa: E731
            rows = [] if p < 0 else [visible(p + i, window, n_sink, there) for i in range(n)]
            self.keys.append(rows)
            for r in rows:
                for j in r:
                    seen[self.table[s][j // page], j % page] = True
            if p >= 0:      # entries that nobody follows
                used = {j // page for r in rows for j in r}
                self.table[s] = [t if i in used or (s, i) in lost else (1 << 30) - i for i, t in enumerate(self.table[s])]
        self.pool.hide(seen)
        self.pool.upload()
        self.start = [sum(counts[:s]) for s in range(len(counts) + 1)]
        self.dtable = torch.tensor(self.table, dtype=torch.int32).cuda()
        self.dpos = torch.tensor(positions, dtype=torch.int32).cuda()
        self.dstart = torch.tensor(self.start, dtype=torch.int32).cuda()
        self.dq = self.q.cuda()

    def cache(self, V):
        return self.pool.cache(V, self.dtable)

    def rows(self, V):
        return V.Rows(self.dpos.data_ptr(), self.dstart.data_ptr(), None, n_rows=self.dq.shape[0], max_rows=max(self.counts))

    def run(self, V, stream=None, scale=0.0, out=None):
        out = torch.full_like(self.dq, 7.0) if out is None else out
        lse = torch.full(self.dq.shape[:2], 7.0, device="cuda")
        V.attention_paged_dev(self.cache(V), self.layer, self.rows(V), self.dq.data_ptr(), self.dtype, self.heads, self.window,
                              self.n_sink, scale, out.data_ptr(), lse.data_ptr(), V.STREAM_LEGACY if stream is None else stream)
        return out, lse

    def values(self, s, keys, head):
        """K and V of a stream's positions, one head, in 64 bits."""
        g = torch.tensor([self.table[s][j // self.page] for j in keys], dtype=torch.long)
        at = torch.tensor([j % self.page for j in keys], dtype=torch.long)
        return [from_e4m3(c[self.layer, g, head, at]) * sc[self.layer, g, head][:, None] for c, sc in zip(self.pool.code, self.pool.scale)]

    def check(self, out, lse, scale=0.0, some=None):
        """Compares with the definition.  K, V and q are exact in the products.
        With u = 2^-24 and S the largest sum of |q||k| * scale of a row, a score
        is off by at most (dim + 6) u S (products and sums, the two scales), its
        exponential by as much, the 2 ulp of ex2 and the 2.7e-6 < 2^-18 of a
        polynomial for 2^x.  So a weight is off by d = (dim + 10) u S + 2^-22 +
        2^-18 relative, and by its rounding to fp16, half a step of it (2^-11), or
        2^-32 of the row's largest where that is more; an output by (2 d + 2^-11 +
        N (u + 2^-32)) max|v| (numerator, denominator, sums, a V scaled to fp16's
        range), and half a step of its own type."""
        out, lse = out.double().cpu(), lse.double().cpu()
        scale = scale or 1.0 / math.sqrt(self.dim)
        group, u = self.heads // self.kv, half_step(self.dtype)
        for s, rows in enumerate(self.keys):
            last = sorted(set(j for r in rows for j in r))
            place = {j: n for n, j in enumerate(last)}
            if some is not None and s not in some:
                continue
            mask = torch.zeros(len(rows), max(1, len(last)), dtype=torch.bool)
            for i, r in enumerate(rows):
                mask[i, [place[j] for j in r]] = True
            for h in range(self.heads):
                at = slice(self.start[s], self.start[s] + len(rows))
                if not last:
                    assert bool((out[at, h] == 0).all()) and bool((lse[at, h] == -math.inf).all()), (s, h)
                    continue
                k, v = self.values(s, last, h // group)
                q = self.q[at, h].double()
                a = ((q @ k.T) * scale).masked_fill(~mask, -math.inf)
                z = torch.logsumexp(a, -1)
                none = ~mask.any(-1)
                w = torch.where(none[:, None], 0.0, (a - z[:, None]).exp())
                o = w @ v
                big = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(~mask, 0).amax(-1)
                d = (self.dim + 10) * U32 * big + 2.0 ** -22 + 2.0 ** -18
                most = (v.abs()[None] * mask[:, :, None]).amax((1, 2)) if len(rows) * v.numel() < 1e8 else v.abs().max().expand(len(rows))
                n = mask.sum(-1)
                tol = ((2 * d + 2.0 ** -11 + n * (U32 + 2.0 ** -32)) * most)[:, None] + u * o.abs() + 2.0 ** -25
                err = (out[at, h] - o).abs()
                assert bool((err <= tol).all()), (s, h, float((err / tol).max()), self.positions[s], int((err / tol).amax(-1).argmax()))
                tol_z = d + n * U32 + 4 * U32 * z.abs()
                same = torch.where(none, lse[at, h] == -math.inf, (lse[at, h] - z).abs() <= tol_z)
                assert bool(same.all()), (s, h, lse[at, h][~same], z[~same])
        for s, p in enumerate(self.positions):   # a stream that sits out
            if p < 0:
                assert bool((out[self.start[s]:self.start[s + 1]] == 7.0).all()), s
        assert bool((out[self.n:] == 7.0).all()) and bool((lse[self.n:] == 7.0).all())
