"""V's scales far apart, for the tests of the attention over a paged cache: what a
row may be off by, told from the keys that it sees and from nothing else."""
import math

import torch

import voxcuda as V
from paged_ref import Case
from rows_ref import U32, half_step

LEAST = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25}   # half the least step of the type


def spread(c, exp):
    """V's scales become 2^exp(stream, index of the page in its stream); what nobody sees stays NaN."""
    for s, pages in enumerate(c.table):
        for i, g in enumerate(pages):
            if 0 <= g < c.pool.pages and not bool(torch.isnan(c.pool.scale[1][c.layer, g]).any()):
                c.pool.scale[1][c.layer, g] = 2.0 ** exp(s, i)
    c.pool.upload()
    return c


def heavy(c, keys, stream=0, most=None):
    """q looks at the first dim alone, whose K is `most` at the positions `keys` and 0 elsewhere: scores, with scale 1."""
    c.q[:] = 0
    c.q[:, :, 0] = 1.0
    c.dq = c.q.cuda()
    c.pool.scale[0][torch.isfinite(c.pool.scale[0])] = 1.0
    last = max([j for r in c.keys[stream] for j in r])
    for j in range(last + 1):
        g, at = c.table[stream][j // c.page], j % c.page
        if 0 <= g < c.pool.pages and bool((c.pool.code[0][c.layer, g, :, at] & 0x7f != 0x7f).all()):
            c.pool.code[0][c.layer, g, :, at] = 0
            if j in keys:
                c.pool.code[0][c.layer, g, :, at, 0] = int(torch.tensor([float(most)]).to(torch.float8_e4m3fn).view(torch.uint8))
    c.pool.upload()
    return c


def check(c, out, lse, scale=0.0, some=None):
    """Compares with the definition, row by row.  With u = 2^-24 and S the largest sum of |q||k| * scale over the row's keys,
    a score is off by at most (dim + 6) u S, its exponential by as much and the 2 ulp of ex2: a weight w, or its product w s
    with V's scale, is off by d = (dim + 10) u S + 2^-22 relative.  The product is rounded to fp16, by half a step of it
    (2^-11), or by 2^-32 of the row's largest product where that is more.  N sums of fp32, each off by 2 u at most of what has
    come together (the tensor cores cut off).  So an output is off by (2 d + 2^-11 + 3 N u) sum(w |v|) + 2^-32 max(w s) sum(|v| / s)
    and half a step of its own type; the lse by d + N u + (4 |lse| + 16) u.
    The kernel of many rows, where V's scales are near one another, rounds the weights and has s in V, exactly: a weight is then
    off by 2^-32 of the row's largest weight (a half step of fp16 is 2^-25 at least, and the largest P is 2^7 at least), an output
    by 2^-32 max(w) sum(|v|) in the place of the term with s, which may be more or less: the larger one is taken."""
    out, lse = out.double().cpu(), lse.double().cpu()
    scale, group, u = scale or 1.0 / math.sqrt(c.dim), c.heads // c.kv, half_step(c.dtype)
    for s, rows in enumerate(c.keys):
        last = sorted(set(j for r in rows for j in r))
        if not last or (some is not None and s not in some):
            continue
        place = {j: n for n, j in enumerate(last)}
        mask = torch.zeros(len(rows), len(last), dtype=torch.bool)
        for i, r in enumerate(rows):
            mask[i, [place[j] for j in r]] = True
        pages = torch.tensor([c.table[s][j // c.page] for j in last])
        at = slice(c.start[s], c.start[s] + len(rows))
        for h in range(c.heads):
            k, v = c.values(s, last, h // group)
            vs = c.pool.scale[1][c.layer, pages, h // group]
            q = c.q[at, h].double()
            a = ((q @ k.T) * scale).masked_fill(~mask, -math.inf)
            z = torch.logsumexp(a, -1)
            w = (a - z[:, None]).exp()
            o, mean, n = w @ v, w @ v.abs(), mask.sum(-1)
            big = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(~mask, 0).amax(-1)
            d = (c.dim + 10) * U32 * big + 2.0 ** -22
            lost = (w * vs).amax(-1)[:, None] * (mask.double() @ (v.abs() / vs[:, None]))
            if c.many:
                lost = torch.maximum(lost, w.amax(-1)[:, None] * (mask.double() @ v.abs()))
            tol = (2 * d + 2.0 ** -11 + 3 * n * U32)[:, None] * mean + 2.0 ** -32 * lost + u * o.abs() + LEAST[c.dtype]
            err = (out[at, h] - o).abs()
            assert bool((err <= tol).all()), (s, h, float((err / tol).max()), int((err / tol).amax(-1).argmax()))
            off = (lse[at, h] - z).abs()
            assert bool((off <= d + n * U32 + (4 * z.abs() + 16) * U32).all()), (s, h, float(off.max()))


def run(c, form=None, **kw):
    """form: packed rows of a CTA and CTAs on an SM that the call has to take."""
    plan = V.attention_paged_plan(c.cache(V), c.rows(V), c.dtype, c.heads, c.window, c.n_sink)
    assert plan[:2] == (form or plan[:2]), plan
    c.many = plan[0] >= 128
    out, lse = c.run(V, **kw)
    torch.cuda.synchronize()
    return out, lse


# Each takes a form, its shape (heads, kv, dim, page, counts of rows) and the positions before
# which other streams' tables reach, which make the plan.  bf16 holds what fp16 does not, so its
# spread is wider.
def small_first_page(dtype, form, heads, kv, dim, page, counts, far):
    """The first page's V is small, the next ones', which later rows of the same tile see, large."""
    for low, high in (((-23, 7),) if dtype == "fp16" else ((-20, 20), (-100, 3), (-60, 110))):
        c = spread(Case(dtype, heads, kv, dim, page, [3] * len(counts) + far, counts + [1] * len(far), seed=3, scale_q=0.3),
                   lambda s, i: low if i == 0 else high)
        check(c, *run(c, form), some=range(len(counts)))


def large_page_left_behind(dtype, form, heads, kv, dim, page, counts, far):
    """The pages that the first rows' windows still hold are large, those that all see small."""
    for low, high in (((-23, 7),) if dtype == "fp16" else ((-20, 20), (-100, 3), (-60, 110))):
        window, first = 3 * page, [5 * page - 4] * len(counts)   # the fourth row's window begins past page 1
        c = spread(Case(dtype, heads, kv, dim, page, first + far, counts + [1] * len(far), window=window, seed=4, scale_q=0.3),
                   lambda s, i: high if i <= 1 else low)
        check(c, *run(c, form), some=range(len(counts)))


def zeros_take_the_weight(dtype, form, heads, kv, dim, page, counts, far):
    """A page whose V is 0, under the scale 2^-100 that it gets, takes nearly all the weight of rows that see large V too; and
    the other way round."""
    for keys in (range(page), range(page, 2 * page)):
        for high in ((7,) if dtype == "fp16" else (7, 110)):
            c = Case(dtype, heads, kv, dim, page, [page + 2] * len(counts) + far, counts + [1] * len(far), seed=5, scale_q=0.0)
            heavy(c, keys, most=6.0)
            c.pool.code[1][c.layer, c.table[0][0]] = 0
            spread(c, lambda s, i: -100 if i == 0 else high)
            check(c, *run(c, form, scale=1.0), scale=1.0, some=[0])


def any_scales(form, heads, kv, dim, page, counts, far):
    """Every page its own scale, from 2^-100 to 2^110."""
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        e = torch.randint(-100, 111, (8, 4096), generator=g).tolist()
        c = spread(Case("bf16", heads, kv, dim, page, [37] * len(counts) + far, counts + [1] * len(far), seed=6 + seed, scale_q=3.0),
                   lambda s, i: e[s % 8][i])
        check(c, *run(c, form))


def others_pages_change_nothing(dtype, form, heads, kv, dim, page, counts, far, same_to=110):
    """Rows give the same bits whatever stands in pages, and in their scales (up to 2^same_to), that they do not see."""
    c = Case(dtype, heads, kv, dim, page, [3] * len(counts) + far, counts + [1] * len(far), seed=7)
    spread(c, lambda s, i: -9)
    out, lse = run(c, form)
    assert min(counts) > page
    for high in (5, 7, 110) if dtype == "bf16" else (5, 7):
        for s in range(len(counts)):
            for i in range(1, len(c.table[s])):
                g = c.table[s][i]
                if 0 <= g < c.pool.pages:
                    c.pool.code[1][0, g] = c.pool.code[1][0, g].flip(-1)
        spread(c, lambda s, i: -9 if i == 0 or s >= len(counts) else high)
        out2, lse2 = run(c, form)
        for s in range(len(counts)):
            a, b = c.start[s], c.start[s] + page - 3
            assert high > same_to or torch.equal(out[a:b], out2[a:b]) and torch.equal(lse[a:b], lse2[a:b]), (high, s)
        check(c, out2, lse2, some=range(len(counts)))
