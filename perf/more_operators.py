"""The operators over a paged cache held in 8 bits, measured: rotary append,
attention of tokens, drafts, chunks and whole prompts, copies of pages.

The cache holds K and V as e4m3 in pages of 16 to 128 positions; a stream's
pages are listed in its row of a table, and every (page, KV head) has a scale
for K and one for V, a power of two.  A number of the cache is its e4m3 value
times its scale; `run` returns both as they are held (float8 and fp32).

`run` computes an operator either through the library's entry points
(`own = True`) or in its plain form: elementary torch operations in 32 bits
(64 for rotation angles and for the scales, where a maximum may stand next to a
border), rounded once at the end.  `exact` computes the same outputs in 64 bits
from the definitions, stream by stream.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0       # of e4m3
LEAST_EXP = -100      # of a scale
EPS = 1e-5
THETA = 1.0e6


def _lib():
    """The library's ctypes binding, initialised on the current device."""
    path = os.path.join(os.getcwd(), "voxtral.c_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import voxcuda
    voxcuda.init(torch.cuda.current_device())
    return voxcuda


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    heads = {"heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # one decode step of eight streams of the decoder: fp32 q|k|v rows behind a GEMV
        {"name": "append-step", "op": "append", "dtype": "bf16", "src": "fp32", "streams": 8, "rows": 1, "less": 0, **heads,
         "page": 64, "pos": 740, "gap": 101, "norm": False},
        # prompt chunks of several streams far into their recordings, normalised heads, fp32 GEMM outputs
        {"name": "append-chunk", "op": "append", "dtype": "bf16", "src": "fp32", "streams": 4, "rows": 1021, "less": 100, **heads,
         "page": 64, "pos": 15000, "gap": 3333, "norm": True},
        # an encoder chunk: 32 heads of 64, all with keys of their own
        {"name": "append-encoder", "op": "append", "dtype": "fp16", "src": "fp16", "streams": 1, "rows": 1500, "less": 0,
         "heads": 32, "kv_heads": 32, "dim": 64, "page": 128, "pos": 3001, "gap": 0, "norm": False},
        # one token of one stream: the decoder's full window
        {"name": "token-one", "op": "attention", "dtype": "bf16", "streams": 1, "rows": 1, "less": 0, **heads, "page": 64,
         "pos": 8191, "gap": 0, "window": 0, "sinks": 0},
        # one token each of many streams, a sliding window and sinks, small pages
        {"name": "token-batch", "op": "attention", "dtype": "fp16", "streams": 24, "rows": 1, "less": 0, **heads, "page": 16,
         "pos": 6000, "gap": 251, "window": 4096, "sinks": 4},
        # a full server: 64 streams, up to twenty minutes of tokens (80 ms each)
        {"name": "token-many", "op": "attention", "dtype": "bf16", "streams": 64, "rows": 1, "less": 0, **heads, "page": 64,
         "pos": 16000, "gap": 171, "window": 0, "sinks": 0},
        # six drafted tokens of eight streams, checked at once
        {"name": "draft", "op": "attention", "dtype": "bf16", "streams": 8, "rows": 6, "less": 0, **heads, "page": 32,
         "pos": 3000, "gap": 300, "window": 0, "sinks": 0},
        # an encoder chunk: 32 heads of 64, window 750, every row its own window
        {"name": "chunk-encoder", "op": "attention", "dtype": "fp16", "streams": 1, "rows": 1500, "less": 0, "heads": 32,
         "kv_heads": 32, "dim": 64, "page": 128, "pos": 3001, "gap": 0, "window": 750, "sinks": 4},
        # whole prompts of four streams, causal
        {"name": "prompt", "op": "attention", "dtype": "bf16", "streams": 4, "rows": 1021, "less": 100, **heads, "page": 64,
         "pos": 0, "gap": 0, "window": 0, "sinks": 0},
        # prompt chunks of two streams over long caches
        {"name": "chunk", "op": "attention", "dtype": "bf16", "streams": 2, "rows": 1024, "less": 27, **heads, "page": 64,
         "pos": 14011, "gap": 7000, "window": 0, "sinks": 0},
        # eight streams forked for a second hypothesis: the page that each was filling, all 26 layers
        {"name": "copy-fork", "op": "copy", "dtype": "bf16", **heads, "page": 64, "layers": 26, "pages": 160, "copies": 8},
        # streams moved whole to other pages, all 26 layers
        {"name": "copy-streams", "op": "copy", "dtype": "bf16", **heads, "page": 64, "layers": 26, "pages": 640, "copies": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """(multiply-adds of an attention, scores that the plain form holds, values of K that it holds)"""
    keys = max(p + n for p, n in zip(_positions(c), _counts(c)))
    return (_pairs(c) * c["heads"] * c["dim"] * 4, c["streams"] * c["rows"] * c["heads"] * keys,
            c["streams"] * keys * c["kv_heads"] * c["dim"])


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "attention", "copy"])
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (32, 32, 64), (28, 4, 128), (16, 2, 64), (12, 12, 128), (10, 1, 64)])
    c = {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "heads": heads, "kv_heads": kv, "dim": dim,
         "page": rng.choice([16, 32, 64, 64, 128])}
    if op == "copy":
        c |= {"layers": rng.choice([1, 4, 26]), "pages": rng.randrange(40, 500)}
        c["copies"] = _log(rng, 1, c["pages"] // 2)
        return c
    c |= {"streams": _log(rng, 1, 48), "gap": rng.randrange(0, 400), "less": rng.randrange(0, 9)}
    if op == "append":
        c |= {"src": rng.choice(["fp32", c["dtype"]]), "norm": rng.random() < 0.5, "pos": _log(rng, 1, 20000)}
        c["rows"] = 1 if rng.random() < 0.3 else max(1, min(_log(rng, 2, 1000), 4000 // c["streams"]))
        return c
    kind = rng.choice(["token", "draft", "chunk", "prompt"])
    c["rows"] = {"token": 1, "draft": rng.randrange(2, 17), "chunk": _log(rng, 16, 1000), "prompt": _log(rng, 32, 2000)}[kind]
    c["pos"] = 0 if kind == "prompt" else _log(rng, 1, 16000)
    c["window"] = rng.choice([0, 0, 750, _log(rng, 16, 8192)])
    c["sinks"] = rng.choice([0, 1, 4, 7]) if c["window"] else 0
    most = (4.5e11, 1.2e9, 5.0e8)
    while c["streams"] > 1 and any(a > b for a, b in zip(_cost(c), most)):
        c["streams"] = max(1, c["streams"] * 2 // 3)
    while c["rows"] > 1 and any(a > b for a, b in zip(_cost(c), most)):
        c["rows"] = max(1, c["rows"] * 2 // 3)
    return c


def _positions(c):
    return [max(0, c["pos"] - s * c["gap"]) for s in range(c["streams"])]


def _counts(c):
    return [max(1, c["rows"] - s * c["less"]) for s in range(c["streams"])]


def _pairs(c):
    """(row, key) pairs that are visible."""
    total = 0
    for p, n in zip(_positions(c), _counts(c)):
        for at in range(p, p + n):
            low = max(0, at - c["window"] + 1) if c["window"] else 0
            total += at + 1 - low + min(low, c["sinks"])
    return total


def _keys(c):
    """Keys that some row of their stream sees."""
    total = 0
    for p, n in zip(_positions(c), _counts(c)):
        low = max(0, p - c["window"] + 1) if c["window"] else 0
        total += p + n - low + min(low, c["sinks"])
    return total


def work(c):
    row = c["kv_heads"] * c["dim"]
    if c["op"] == "copy":
        n = c["copies"] * c["layers"] * (c["page"] * row * 2 + 8 * c["kv_heads"])
        return {"bytes": 2 * n, "flops": n}
    n, h, b = sum(_counts(c)), c["heads"] * c["dim"], SIZE[c["dtype"]]
    if c["op"] == "append":
        return {"bytes": n * ((h + 2 * row) * SIZE[c["src"]] + h * b + 2 * row), "flops": n * (h + 2 * row) * (8 if c["norm"] else 4)}
    return {"bytes": 2 * _keys(c) * row + 2 * n * h * b + 4 * n * c["heads"], "flops": 4 * _pairs(c) * h}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def prepare(c, seed):
    dev = "cuda"
    cpu = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, page, kv, dim = TYPES[c["dtype"]], c["page"], c["kv_heads"], c["dim"]

    def normal(*shape, to=dtype, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(to)

    st = {"case": c}
    if c["op"] == "copy":
        layers, pages = c["layers"], c["pages"]
        order = torch.randperm(pages, generator=cpu)
        st["src"] = order[: c["copies"]].to(dev, torch.int32)
        st["dst"] = order[c["copies"]: 2 * c["copies"]].to(dev, torch.int32)
    else:
        # the streams' pages lie anywhere in the pool, a few of which are free; -1 stands behind a stream's last page
        layers, counts, positions = 1, _counts(c), _positions(c)
        held = [-(-(p + n) // page) for p, n in zip(positions, counts)]
        pages, width = sum(held) + 5, max(held) + 1
        order = torch.randperm(pages, generator=cpu)
        table = torch.full((c["streams"], width), -1, dtype=torch.int64)
        for s, n in enumerate(held):
            table[s, :n] = order[sum(held[:s]): sum(held[:s]) + n]
        st["table"] = table.to(dev, torch.int32)
        st["pos"] = torch.tensor(positions, dtype=torch.int32, device=dev)
        st["start"] = torch.tensor([sum(counts[:s]) for s in range(len(counts) + 1)], dtype=torch.int32, device=dev)
        st["n"], st["most"] = sum(counts), max(counts)
    # values of about 1: e4m3 numbers of about 100 under scales of 2^-8 to 2^-6
    for name in ("k", "v"):
        st[name] = torch.empty(layers, pages, kv, page, dim, dtype=torch.uint8, device=dev)
        for layer in st[name]:
            layer.copy_((torch.randn(layer.shape, generator=gen, device=dev) * 100).clamp_(-LARGEST, LARGEST).to(E4M3).view(torch.uint8))
        st[name + "_scale"] = torch.exp2(torch.randint(-8, -5, (layers, pages, kv), generator=gen, device=dev).float())
    if c["op"] == "append":
        st["qkv"] = normal(st["n"], c["heads"] + 2 * kv, dim, to=TYPES[c["src"]], scale=2.0)
        st["gq"] = 1 + 0.1 * normal(dim, to=torch.float32) if c["norm"] else None
        st["gk"] = 1 + 0.1 * normal(dim, to=torch.float32) if c["norm"] else None
        st["q"] = torch.empty(st["n"], c["heads"], dim, dtype=dtype, device=dev)
    elif c["op"] == "attention":
        st["q"] = normal(st["n"], c["heads"], dim, scale=2.0)
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(st["n"], c["heads"], device=dev)
    if own:
        V = st["lib"] = _lib()
        st["stream"] = torch.cuda.current_stream().cuda_stream or V.STREAM_LEGACY
        tab = st.get("table")
        st["cache"] = V.PagedCache(st["k"].data_ptr(), st["v"].data_ptr(), st["k_scale"].data_ptr(), st["v_scale"].data_ptr(),
                                   None if tab is None else tab.data_ptr(), table_stride=0 if tab is None else tab.shape[1],
                                   n_layers=layers, n_pages=pages, page_size=page, n_streams=c.get("streams", 1), n_kv_heads=kv,
                                   head_dim=dim)
        if c["op"] != "copy":
            st["rows"] = V.Rows(st["pos"].data_ptr(), st["start"].data_ptr(), None, n_rows=st["n"], max_rows=st["most"])
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(st):
    c = st["case"]
    if own:
        _run_own(st, c)
    elif c["op"] == "append":
        _plain_append(st, c)
    elif c["op"] == "attention":
        return _plain_attention(st, c)
    else:
        _plain_copy(st, c)
    if c["op"] == "attention":
        return {"out": st["out"], "lse": st["lse"]}
    held = {"k": st["k"].view(E4M3), "v": st["v"].view(E4M3), "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    return held | {"q": st["q"]} if c["op"] == "append" else held


def _run_own(st, c):
    V, stream = st["lib"], st["stream"]
    if c["op"] == "append":
        V.rope_append_paged_dev(st["cache"], 0, st["rows"], st["qkv"].data_ptr(), c["src"], c["heads"], st["qkv"].stride(0),
                                None if st["gq"] is None else st["gq"].data_ptr(), None if st["gk"] is None else st["gk"].data_ptr(),
                                EPS, THETA, st["q"].data_ptr(), c["dtype"], stream)
    elif c["op"] == "attention":
        V.attention_paged_dev(st["cache"], 0, st["rows"], st["q"].data_ptr(), c["dtype"], c["heads"], c["window"], c["sinks"], 0.0,
                              st["out"].data_ptr(), st["lse"].data_ptr(), stream)
    else:
        V.kv_copy_pages_dev(st["cache"], st["src"].data_ptr(), st["dst"].data_ptr(), c["copies"], stream)


def _rows(st):
    """(stream, index in its stream) of every row."""
    start = st["start"].long()
    row = torch.arange(st["n"], device=start.device)
    s = torch.searchsorted(start, row, right=True) - 1
    return s, row - start[s]


def _plain_store(st, c, name, x, s, at):
    """The rows' values x of one KV tensor at the positions `at` of their streams."""
    pool, scale, page = st[name][0], st[name + "_scale"][0], c["page"]
    to, slot = st["table"].long()[s, at // page], at % page
    pages, kv = scale.shape
    index = to[:, None].expand(-1, kv)
    most = torch.zeros_like(scale).scatter_reduce_(0, index, x.abs().amax(-1), "amax")
    m, e = torch.frexp(most.double() / LARGEST)
    need = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp_(min=LEAST_EXP).double()).float()
    first = torch.full((pages,), page, device=x.device).scatter_reduce_(0, to, slot, "amin")   # the first new slot
    touched = (first < page)[:, None]
    new = torch.where(touched, torch.where((first == 0)[:, None], need, torch.maximum(scale, need)), scale)
    # what the pages that were being filled hold already
    pos = st["pos"].long()
    mine = st["table"].long()[torch.arange(len(pos), device=x.device), pos // page]
    old = pool[mine].view(E4M3).float() * (scale[mine] / new[mine])[:, :, None, None]
    before = torch.arange(page, device=x.device)[None] < (pos % page)[:, None]
    pool[mine] = torch.where(before[:, None, :, None], old.to(E4M3).view(torch.uint8), pool[mine])
    pool[to, :, slot] = (x / new[to][:, :, None]).to(E4M3).view(torch.uint8)
    scale.copy_(new)


def _plain_append(st, c):
    s, i = _rows(st)
    at = st["pos"].long()[s] + i
    x = st["qkv"].float()
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * st["gq"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * st["gk"]
    freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    angle = at.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(t):
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    _plain_store(st, c, "k", turn(k), s, at)
    _plain_store(st, c, "v", v, s, at)
    st["q"].copy_(turn(q))


def _plain_attention(st, c):
    """Rows padded to the longest stream's, keys in the order of their positions."""
    s, i = _rows(st)
    dev, most, page = s.device, st["most"], c["page"]
    streams, h, kv, d = c["streams"], c["heads"], c["kv_heads"], c["dim"]
    pos = st["pos"].long()
    table = st["table"].long()
    there = (table >= 0)[:, :, None].expand(-1, -1, page).flatten(1)

    def gather(name):
        x = st[name][0][table.clamp(min=0)].view(E4M3).float()                      # streams, pages, heads, slots, dims
        x = x * st[name + "_scale"][0][table.clamp(min=0)][..., None, None]
        return x.transpose(2, 3).flatten(1, 2).masked_fill_(~there[..., None, None], 0.0)

    key = torch.arange(there.shape[1], device=dev)
    at = pos[:, None] + torch.arange(most, device=dev)[None]
    seen = there[:, None, :] & (key <= at[:, :, None])
    if c["window"]:
        seen = seen & ((key > at[:, :, None] - c["window"]) | (key < c["sinks"]))
    q = torch.zeros(streams, most, h, d, device=dev)
    q[s, i] = st["q"].float()
    q = q.view(streams, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(streams, kv, -1, d)
    score = (q @ gather("k").permute(0, 2, 3, 1)).view(streams, kv, h // kv, most, -1) * (1.0 / math.sqrt(d))
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(streams, kv, -1, len(key)) @ gather("v").permute(0, 2, 1, 3)).view(streams, kv, h // kv, most, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(streams, most, h, d)[s, i]
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(streams, most, h)[s, i]
    return {"out": out.to(st["q"].dtype), "lse": lse}


def _plain_copy(st, c):
    src, dst = st["src"].long(), st["dst"].long()
    st["k"][:, dst], st["v"][:, dst] = st["k"][:, src], st["v"][:, src]
    st["k_scale"][:, dst], st["v_scale"][:, dst] = st["k_scale"][:, src], st["v_scale"][:, src]


# --------------------------------------------------------------------------
# 64 bits, from the definitions
# --------------------------------------------------------------------------

def _exact_e4m3(x):
    """The e4m3 number nearest to x, ties to even: steps of 2^(e - 3) of the value's power of two 2^e, of 2^-9 at least."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -40))).clamp(min=-6)
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, torch.where((x.abs() < torch.exp2(e)) & (e > -6), e - 1, e))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def exact(c, seed):
    st = prepare(c, seed)
    if c["op"] == "copy":
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            for name in ("k", "v", "k_scale", "v_scale"):
                st[name][:, b] = st[name][:, a].clone()
        return {"k": st["k"].view(E4M3), "v": st["v"].view(E4M3), "k_scale": st["k_scale"].double(), "v_scale": st["v_scale"].double()}
    counts, positions, table = _counts(c), _positions(c), st["table"].tolist()
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    held = {name: st[name][0].view(E4M3).double() for name in ("k", "v")}
    scale = {name: st[name + "_scale"][0].double() for name in ("k", "v")}
    if c["op"] == "append":
        freq = torch.tensor([THETA ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device="cuda")
        x, at, out = st["qkv"].double(), 0, []
        for s, (p, n) in enumerate(zip(positions, counts)):
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               torch.arange(p, p + n, dtype=torch.float64, device="cuda")[:, None] * freq)
            part, new = x[at:at + n], []
            for block, g in ((part[:, :h], st["gq"]), (part[:, h:h + kv], st["gk"])):
                if g is not None:
                    block = block / (block.square().mean(-1, keepdim=True) + EPS).sqrt() * g.double()
                z = torch.view_as_complex(block.reshape(n, -1, d // 2, 2).contiguous()) * turn[:, None]
                new.append(torch.view_as_real(z).reshape(n, -1, d))
            out.append(new[0])
            for name, rows in (("k", new[1]), ("v", part[:, h + kv:])):
                for j in range(p // page, (p + n - 1) // page + 1):
                    a, b = max(p, j * page), min(p + n, (j + 1) * page)
                    chunk = rows[a - p:b - p].transpose(0, 1)                       # heads, slots, dims
                    need = torch.tensor([2.0 ** max(LEAST_EXP, math.ceil(math.log2(max(m, 1e-300) / LARGEST)))
                                         for m in chunk.abs().amax((1, 2)).tolist()], dtype=torch.float64, device="cuda")
                    g, lo = table[s][j], a - j * page
                    was = scale[name][g].clone()
                    to = need if lo == 0 else torch.maximum(was, need)
                    held[name][g, :, :lo] = _exact_e4m3(held[name][g, :, :lo] * (was / to)[:, None, None])
                    held[name][g, :, lo:lo + b - a] = _exact_e4m3(chunk / to[:, None, None])
                    scale[name][g] = to
            at += n
        return {"q": torch.cat(out), "k": held["k"][None], "v": held["v"][None], "k_scale": scale["k"][None], "v_scale": scale["v"][None]}
    if _pairs(c) * h * d > 3e12:
        return None
    outs, lses, at = [], [], 0
    for s, (p, n) in enumerate(zip(positions, counts)):
        mine = torch.tensor(table[s][: -(-(p + n) // page)], device="cuda")
        here, j = p + torch.arange(n, device="cuda"), torch.arange(p + n, device="cuda")
        seen = j[None] <= here[:, None]
        if c["window"]:
            seen = seen & ((j[None] > here[:, None] - c["window"]) | (j < c["sinks"])[None])
        o, e = [], []
        for g in range(kv):
            k, v = (((held[name][mine, g] * scale[name][mine, g][:, None, None]).flatten(0, 1)[: p + n]) for name in ("k", "v"))
            for head in range(g * (h // kv), (g + 1) * (h // kv)):
                a = (st["q"][at:at + n, head].double() @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                z = torch.logsumexp(a, -1)
                e.append(z)
                o.append((a - z[:, None]).exp() @ v)
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(e, 1))
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
