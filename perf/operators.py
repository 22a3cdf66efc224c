"""The streaming-decode operators, measured: rotary append, attention with a
window and sinks, attention of a draft tree, cache commit and fork, token log
probabilities.

`run` computes one of them either through the library's entry points
(`own = True`) or in its plain form: elementary torch operations in 32 bits
(64 for rotation angles and long sums), rounded once at the end.  `exact`
computes the same outputs in 64 bits from the definitions, stream by stream.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
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
    return [
        # one decode step of eight streams of the decoder: fp32 q|k|v rows into fp32 rings
        {"name": "append-step", "op": "append", "dtype": "fp32", "src": "fp32", "streams": 8, "rows": 1, "less": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "cap": 1024, "sinks": 0, "pos": 740, "gap": 100, "norm": False,
         "tree": False},
        # prompt chunks of several streams, normalised heads, a 16-bit cache behind fp32 GEMM outputs
        {"name": "append-chunk", "op": "append", "dtype": "bf16", "src": "fp32", "streams": 4, "rows": 1021, "less": 100,
         "heads": 32, "kv_heads": 8, "dim": 128, "cap": 2048, "sinks": 4, "pos": 150000, "gap": 33333, "norm": True,
         "tree": False},
        # one token of a long-running transcription: the decoder's full window in its fp32 ring, four sinks
        {"name": "window-token", "op": "window", "dtype": "fp32", "streams": 1, "rows": 1, "less": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 9216, "sinks": 4, "pos": 100000, "gap": 0, "window": 8192},
        # one token each of many streams, 16-bit rings, ragged lengths
        {"name": "window-batch", "op": "window", "dtype": "bf16", "streams": 24, "rows": 1, "less": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 4100, "sinks": 4, "pos": 6000, "gap": 251, "window": 4096},
        # an encoder chunk: 32 heads of 64, window 750, every row its own window
        {"name": "window-encoder", "op": "window", "dtype": "fp16", "streams": 1, "rows": 1500, "less": 0, "heads": 32,
         "kv_heads": 32, "dim": 64, "cap": 2304, "sinks": 4, "pos": 3001, "gap": 0, "window": 750},
        # prompt chunks of two streams over a long cache
        {"name": "window-chunk", "op": "window", "dtype": "bf16", "streams": 2, "rows": 1024, "less": 27, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 5200, "sinks": 4, "pos": 20011, "gap": 7000, "window": 4096},
        # eight drafted tokens over a short fp32 ring, right after a stream's start
        {"name": "tree-few", "op": "tree", "dtype": "fp32", "streams": 1, "rows": 8, "less": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "cap": 1024, "sinks": 0, "pos": 740, "gap": 0, "window": 0},
        # a full draft tree for each of eight streams, long 16-bit rings
        {"name": "tree-wide", "op": "tree", "dtype": "bf16", "streams": 8, "rows": 64, "less": 3, "heads": 32, "kv_heads": 8,
         "dim": 128, "cap": 8300, "sinks": 4, "pos": 9001, "gap": 500, "window": 8192},
        # accepted paths of eight streams' trees, all 26 layers, fp32 rings
        {"name": "commit", "op": "commit", "dtype": "fp32", "streams": 8, "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "layers": 26, "cap": 256, "sinks": 4, "pos": 400, "gap": 17, "accept": 5},
        # two streams forked for a second hypothesis, all layers
        {"name": "fork", "op": "fork", "dtype": "bf16", "streams": 4, "heads": 32, "kv_heads": 8, "dim": 128, "layers": 26,
         "cap": 4100, "sinks": 4, "pos": 9000, "gap": 3001, "pairs": 2},
        # confidence of one emitted token over the decoder's vocabulary
        {"name": "logprobs-step", "op": "logprobs", "dtype": "fp32", "rows": 1, "vocab": 131072, "top": 5},
        # scoring a whole transcript
        {"name": "logprobs-pass", "op": "logprobs", "dtype": "bf16", "rows": 1001, "vocab": 131072, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _attention_cost(c):
    keys = _pairs(c)
    return keys * c["heads"] * c["dim"] * 4


def draw(rng):
    op = rng.choice(["append", "window", "window", "tree", "tree", "commit", "fork", "logprobs"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 200000)
        rows = min(_log(rng, 1, 1024), max(1, 130_000_000 // vocab))
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 4, 5, 20, 32])}
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 32, 64), (28, 4, 128), (16, 2, 64), (12, 12, 128), (10, 1, 64)])
    c = {"op": op, "dtype": dtype, "streams": _log(rng, 1, 24), "heads": heads, "kv_heads": kv, "dim": dim,
         "sinks": rng.choice([0, 1, 4, 7, 16]), "gap": rng.randrange(0, 400)}
    if op == "append":
        c |= {"src": rng.choice(["fp32", dtype]), "rows": min(_log(rng, 1, 1000), 4000 // c["streams"]), "less": rng.randrange(0, 9),
              "pos": _log(rng, 1, 400000), "norm": rng.random() < 0.5, "tree": False}
        if c["rows"] <= 64 and rng.random() < 0.4:
            c["tree"] = True
        c["cap"] = c["rows"] + c["sinks"] + _log(rng, 16, 1000)
        return c
    if op == "window":
        c |= {"rows": 1 if rng.random() < 0.5 else _log(rng, 2, 1000), "window": rng.choice([0, 64, 750, _log(rng, 16, 8192)]),
              "pos": _log(rng, 1, 300000)}
    elif op == "tree":
        c |= {"rows": _log(rng, 2, 128), "window": rng.choice([0, 0, 8192, _log(rng, 16, 8192)]), "pos": _log(rng, 1, 50000)}
    elif op == "commit":
        c |= {"rows": _log(rng, 16, 128), "layers": rng.choice([1, 4, 26]), "pos": _log(rng, 1, 3000), "accept": rng.randrange(2, 8)}
        c["cap"] = c["rows"] + c["sinks"] + _log(rng, 16, 150)
        c["streams"] = min(c["streams"], 8)
        return c
    else:
        c |= {"streams": rng.randrange(2, 6), "layers": rng.choice([1, 4, 26]), "pos": _log(rng, 1, 20000)}
        c["pairs"] = rng.randrange(1, c["streams"] // 2 + 1)
        c["cap"] = c["sinks"] + _log(rng, 64, 3000)
        return c
    c["less"] = rng.randrange(0, 3)
    c["cap"] = c["sinks"] + c["rows"] + _log(rng, 32, 8192)
    while c["streams"] > 1 and (_attention_cost(c) > 5e11 / (8 if dtype == "fp32" else 1)
                                or c["streams"] * c["rows"] * heads * min(c["cap"], 9000) > 3e8):
        c["streams"] = max(1, c["streams"] // 2)
    while c["rows"] > 1 and (_attention_cost(c) > 5e11 / (8 if dtype == "fp32" else 1) or c["rows"] * heads * c["cap"] > 3e8):
        c["rows"] = max(1, c["rows"] // 2)
    return c


def _positions(c):
    return [max(0, c["pos"] - s * c["gap"]) for s in range(c["streams"])]


def _counts(c):
    return [max(1, c["rows"] - s * c.get("less", 0)) for s in range(c["streams"])]


def _accepted(c):
    return [c["accept"] - s % 2 for s in range(c["streams"])]


def _spans(c):
    """Per stream: (first position, rows, lowest held position past the sinks)."""
    ring = c["cap"] - c["sinks"]
    return [(p, n, max(c["sinks"], p + n - ring)) for p, n in zip(_positions(c), _counts(c))]


def _pairs(c):
    """(row, key) pairs that are visible; a tree counts its context and each node itself."""
    total = 0
    for p, n, held in _spans(c):
        for i in range(n):
            at = p if c["op"] == "tree" else p + i
            low = max(held, at - c["window"] + 1) if c["window"] else held
            upto = p - 1 if c["op"] == "tree" else at
            total += min(upto + 1, c["sinks"]) + max(0, upto + 1 - low) + (1 if c["op"] == "tree" else 0)
    return total


def _keys(c):
    """Keys that some row of their stream sees."""
    total = 0
    for p, n, held in _spans(c):
        low = max(held, p - c["window"] + 1) if c["window"] else held
        total += min(p + n, c["sinks"]) + max(0, p + n - low)
    return total


def work(c):
    b = SIZE[c["dtype"]]
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * b + c["rows"] * (12 + 8 * c["top"]), "flops": 5 * n}
    row = c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        n, h = sum(_counts(c)), c["heads"] * c["dim"]
        return {"bytes": n * ((h + 2 * row) * SIZE[c["src"]] + (h + 2 * row) * b), "flops": n * (h + row) * (8 if c["norm"] else 4)}
    if c["op"] == "commit":
        n = sum(a - 1 for a in _accepted(c)) * c["layers"] * row   # the root is in its place already
        return {"bytes": 4 * n * b, "flops": n}
    if c["op"] == "fork":
        held = [min(p, c["cap"]) for p in _positions(c)]
        n = sum(held[: c["pairs"]]) * c["layers"] * row
        return {"bytes": 4 * n * b, "flops": n}
    n = sum(_counts(c))
    return {"bytes": 2 * _keys(c) * row * b + 2 * n * c["heads"] * c["dim"] * b + 4 * n * c["heads"],
            "flops": 4 * _pairs(c) * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _parents(counts, g):
    """A drafted tree per stream: each node's parent is an earlier node of its stream or none (-1)."""
    out = []
    for n in counts:
        far = torch.randint(1, 9, (n,), generator=g)
        p = torch.arange(n) - far
        out.append(torch.clamp(p, min=-1))
    return torch.cat(out).to(torch.int32)


def prepare(c, seed):
    dev = "cuda"
    cpu = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[c["dtype"]]

    def normal(*shape, to=dtype, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(to)

    st = {"case": c}
    if c["op"] == "logprobs":
        st["logits"] = normal(c["rows"], c["vocab"], scale=3.0)
        st["tokens"] = torch.randint(0, c["vocab"], (c["rows"],), generator=cpu).to(dev, torch.int32)
        st["logprob"] = torch.empty(c["rows"], device=dev)
        st["entropy"] = torch.empty(c["rows"], device=dev)
        st["top_ids"] = torch.empty(c["rows"], c["top"], dtype=torch.int32, device=dev)
        st["top_logprob"] = torch.empty(c["rows"], c["top"], device=dev)
    else:
        layers = c.get("layers", 1)
        shape = (layers, c["streams"], c["cap"], c["kv_heads"], c["dim"])
        st["k"], st["v"] = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
        for t in (st["k"], st["v"]):   # layer by layer: no second copy of a large cache
            for layer in t:
                layer.copy_(torch.randn(layer.shape, generator=gen, device=dev))
        st["pos"] = torch.tensor(_positions(c), dtype=torch.int32, device=dev)
    if c["op"] in ("append", "window", "tree"):
        counts = _counts(c)
        n = sum(counts)
        st["start"] = torch.tensor([sum(counts[:s]) for s in range(len(counts) + 1)], dtype=torch.int32, device=dev)
        st["n"], st["most"] = n, max(counts)
        st["parent"] = _parents(counts, cpu).to(dev) if c["op"] == "tree" or c.get("tree") else None
        st["q"] = torch.empty(n, c["heads"], c["dim"], dtype=dtype, device=dev)
        if c["op"] == "append":
            st["qkv"] = normal(n, c["heads"] + 2 * c["kv_heads"], c["dim"], to=TYPES[c["src"]], scale=2.0)
            st["gq"] = 1 + 0.1 * normal(c["dim"], to=torch.float32) if c["norm"] else None
            st["gk"] = 1 + 0.1 * normal(c["dim"], to=torch.float32) if c["norm"] else None
        else:
            st["q"] = normal(n, c["heads"], c["dim"], scale=2.0)
            st["out"] = torch.empty_like(st["q"])
            st["lse"] = torch.empty(n, c["heads"], device=dev)
    if c["op"] == "commit":
        # an accepted path: the root, then nodes behind every row that the commit writes
        a, r = c["accept"], c["rows"]
        late = [sorted(torch.randperm(r - a, generator=cpu)[: a - 1].tolist()) for _ in range(c["streams"])]
        st["path"] = torch.tensor([[0] + [a + x for x in row] + [-1] * (8 - a) for row in late], dtype=torch.int32, device=dev)
        st["accepted"] = torch.tensor(_accepted(c), dtype=torch.int32, device=dev)
        st["new_pos"] = torch.empty_like(st["pos"])
    if c["op"] == "fork":
        st["src"] = list(range(c["pairs"]))
        st["dst"] = [c["pairs"] + i for i in range(c["pairs"])]
    if own:
        V = st["lib"] = _lib()
        st["stream"] = torch.cuda.current_stream().cuda_stream or V.STREAM_LEGACY
        if c["op"] != "logprobs":
            k = st["k"]
            st["cache"] = V.KvCache(k.data_ptr(), st["v"].data_ptr(), c["dtype"], n_layers=k.shape[0], n_streams=k.shape[1],
                                    cap=c["cap"], n_kv_heads=c["kv_heads"], head_dim=c["dim"], n_sink=c["sinks"])
        if c["op"] in ("append", "window", "tree"):
            par = st["parent"]
            st["rows"] = V.Rows(st["pos"].data_ptr(), st["start"].data_ptr(), None if par is None else par.data_ptr(),
                                n_rows=st["n"], max_rows=st["most"])
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(st):
    c = st["case"]
    if own:
        return _run_own(st, c)
    return {"append": _plain_append, "window": _plain_attention, "tree": _plain_attention, "commit": _plain_commit,
            "fork": _plain_fork, "logprobs": _plain_logprobs}[c["op"]](st, c)


def _run_own(st, c):
    V, op, stream = st["lib"], c["op"], st["stream"]
    if op == "logprobs":
        V.token_logprobs_dev(st["logits"].data_ptr(), c["dtype"], c["rows"], c["vocab"], c["vocab"], st["tokens"].data_ptr(),
                             c["top"], st["logprob"].data_ptr(), st["entropy"].data_ptr(), st["top_ids"].data_ptr(),
                             st["top_logprob"].data_ptr(), stream)
        return {"logprob": st["logprob"], "entropy": st["entropy"], "top_ids": st["top_ids"], "top_logprob": st["top_logprob"]}
    if op == "append":
        V.rope_append_dev(st["cache"], 0, st["rows"], st["qkv"].data_ptr(), c["src"], c["heads"], st["qkv"].stride(0),
                          None if st["gq"] is None else st["gq"].data_ptr(), None if st["gk"] is None else st["gk"].data_ptr(),
                          EPS, THETA, st["q"].data_ptr(), stream)
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    if op in ("window", "tree"):
        call = V.attention_window_dev if op == "window" else V.attention_tree_dev
        call(st["cache"], 0, st["rows"], st["q"].data_ptr(), c["heads"], c["window"], 0.0, st["out"].data_ptr(),
             st["lse"].data_ptr(), stream)
        return {"out": st["out"], "lse": st["lse"]}
    if op == "commit":
        V.kv_commit_dev(st["cache"], st["pos"].data_ptr(), st["path"].data_ptr(), st["path"].shape[1], st["accepted"].data_ptr(),
                        c["accept"], st["new_pos"].data_ptr(), stream)
        return {"k": st["k"], "v": st["v"], "pos": st["new_pos"]}
    V.kv_fork_dev(st["cache"], st["src"], st["dst"], st["pos"].data_ptr(), stream)
    return {"k": st["k"], "v": st["v"]}


def _slot(p, c):
    ring = c["cap"] - c["sinks"]
    return torch.where(p < c["sinks"], p, c["sinks"] + (p - c["sinks"]).remainder(ring))


def _rows(st):
    """(stream, index in its stream) of every row."""
    start = st["start"].long()
    row = torch.arange(st["n"], device=start.device)
    s = torch.searchsorted(start, row, right=True) - 1
    return s, row - start[s]


def _closure(st, s, i):
    """[streams, most, most] truth values: node b is an ancestor of node a, or a itself."""
    n = st["most"]
    eye = torch.eye(n, device=s.device).expand(len(st["pos"]), n, n)
    up = torch.zeros_like(eye, dtype=torch.float32).contiguous()
    par = st["parent"].long()
    up[s, i, par.clamp(min=0)] = (par >= 0).float()
    return torch.linalg.solve_triangular(eye - up, eye, upper=False, unitriangular=True) > 0.5


def _plain_append(st, c):
    s, i = _rows(st)
    pos = st["pos"].long()
    depth = i if st["parent"] is None else _closure(st, s, i).sum(-1)[s, i] - 1
    x = st["qkv"].float()
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * st["gq"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * st["gk"]
    freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    angle = (pos[s] + depth).double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(t):
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    to = _slot(pos[s] + i, c)
    st["k"][0, s, to] = turn(k).to(st["k"].dtype)
    st["v"][0, s, to] = v.to(st["v"].dtype)
    return {"q": turn(q).to(st["q"].dtype), "k": st["k"], "v": st["v"]}


def _plain_attention(st, c):
    """Rows padded to the longest stream's, keys in the order of their slots."""
    s, i = _rows(st)
    dev, most, ring = s.device, st["most"], c["cap"] - c["sinks"]
    streams, h, kv, d = c["streams"], c["heads"], c["kv_heads"], c["dim"]
    pos = st["pos"].long()
    count = (st["start"][1:] - st["start"][:-1]).long()
    # the position that each slot holds once the rows are in
    last = (pos + count - 1)[:, None]
    slot = torch.arange(c["cap"], device=dev)[None]
    held = torch.where(slot < c["sinks"], slot, last - (last - slot).remainder(ring))
    there = (held >= 0) & (held <= last) & ((slot < c["sinks"]) | (held >= c["sinks"]))
    row = torch.arange(most, device=dev)
    tree = st["parent"] is not None
    if tree:
        mine = _closure(st, s, i)
        depth = mine.sum(-1) - 1
        at = pos[:, None] + depth
    else:
        at = pos[:, None] + row[None]
    key = held[:, None, :]
    logical = key.expand(streams, 1, -1)
    seen = there[:, None, :] & (key <= at[:, :, None])
    if tree:
        node = (held - pos[:, None]).clamp(0, most - 1)
        draft = (held >= pos[:, None])[:, None, :]
        family = torch.gather(mine, 2, node[:, None, :].expand(streams, most, -1))
        seen = there[:, None, :] & torch.where(draft, family, key < pos[:, None, None])
        logical = torch.where(draft, (pos[:, None] + torch.gather(depth, 1, node))[:, None, :], key)
    if c["window"]:
        kept = (logical > at[:, :, None] - c["window"]) | (logical < c["sinks"])
        seen = seen & kept
    q = torch.zeros(streams, most, h, d, device=dev)
    q[s, i] = st["q"].float()
    q = q.view(streams, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(streams, kv, -1, d)
    k = st["k"][0].float().permute(0, 2, 3, 1)
    v = torch.where(there[..., None, None], st["v"][0].float(), 0.0).permute(0, 2, 1, 3)
    score = (q @ k).view(streams, kv, h // kv, most, -1) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = (score - top).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(streams, kv, -1, c["cap"]) @ v).view(streams, kv, h // kv, most, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(streams, most, h, d)[s, i]
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(streams, most, h)[s, i]
    return {"out": out.to(st["q"].dtype), "lse": lse}


def _plain_commit(st, c):
    a = torch.arange(c["accept"], device=st["path"].device)
    s, k = torch.nonzero(a[None] < st["accepted"][:, None], as_tuple=True)
    pos = st["pos"].long()
    frm, to = _slot(pos[s] + st["path"][s, k].long(), c), _slot(pos[s] + k, c)
    st["k"][:, s, to] = st["k"][:, s, frm]
    st["v"][:, s, to] = st["v"][:, s, frm]
    return {"k": st["k"], "v": st["v"], "pos": st["pos"] + st["accepted"]}


def _plain_fork(st, c):
    dev = st["pos"].device
    src, dst = torch.tensor(st["src"], device=dev), torch.tensor(st["dst"], device=dev)
    full = st["pos"].long()[src][:, None] > torch.arange(c["cap"], device=dev)[None]
    which, slot = torch.nonzero(full, as_tuple=True)   # the first pos slots are the ones in use
    st["k"][:, dst[which], slot] = st["k"][:, src[which], slot]
    st["v"][:, dst[which], slot] = st["v"][:, src[which], slot]
    return {"k": st["k"], "v": st["v"]}


def _plain_logprobs(st, c):
    x = st["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, dtype=torch.float64)
    spread = (e * (x - m)).sum(-1, dtype=torch.float64)
    logz = z.log()
    own_logit = torch.gather(x, 1, st["tokens"].long()[:, None])
    logprob = ((own_logit - m).double().squeeze(-1) - logz).float()
    entropy = (logz - spread / z).float()
    # one whole number orders by value, then by the lowest id
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (bits << 32) | (0x7FFFFFFF - torch.arange(c["vocab"], device=x.device))
    ids = 0x7FFFFFFF - (torch.topk(key, c["top"], dim=-1).values & 0xFFFFFFFF)
    top = ((torch.gather(x, 1, ids) - m).double() - logz[:, None]).float()
    return {"logprob": logprob, "entropy": entropy, "top_ids": ids.to(torch.int32), "top_logprob": top}


# --------------------------------------------------------------------------
# 64 bits, from the definitions
# --------------------------------------------------------------------------

def _exact_slot(p, c):
    return p if p < c["sinks"] else c["sinks"] + (p - c["sinks"]) % (c["cap"] - c["sinks"])


def _exact_depths(parent):
    depth = []
    for p in parent:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def exact(c, seed):
    st = prepare(c, seed)
    op = c["op"]
    if op == "logprobs":
        lp, ent, top = [], [], []
        for row, tok in zip(st["logits"], st["tokens"].tolist()):
            x = row.double()
            lz = torch.logsumexp(x, 0)
            p = x - lz
            lp.append(p[tok])
            ent.append(-(p.exp() * p).sum())
            top.append(torch.sort(p, descending=True).values[: c["top"]])
        return {"logprob": torch.stack(lp), "entropy": torch.stack(ent), "top_ids": None, "top_logprob": torch.stack(top)}
    positions = _positions(c)
    if op == "fork":
        for a, b in zip(st["src"], st["dst"]):
            p = positions[a]
            slots = sorted({_exact_slot(j, c) for j in list(range(min(p, c["sinks"]))) + list(range(max(0, p - c["cap"]), p))})
            st["k"][:, b, slots] = st["k"][:, a, slots].clone()
            st["v"][:, b, slots] = st["v"][:, a, slots].clone()
        return {"k": st["k"], "v": st["v"]}
    if op == "commit":
        path, took = st["path"].tolist(), st["accepted"].tolist()
        for s, p in enumerate(positions):
            for n in range(took[s]):
                a, b = _exact_slot(p + path[s][n], c), _exact_slot(p + n, c)
                st["k"][:, s, b] = st["k"][:, s, a].clone()
                st["v"][:, s, b] = st["v"][:, s, a].clone()
        return {"k": st["k"], "v": st["v"], "pos": None}
    counts, h, kv, d = _counts(c), c["heads"], c["kv_heads"], c["dim"]
    parent = None if st["parent"] is None else st["parent"].tolist()
    if op == "append":
        k, v = st["k"].double(), st["v"].double()
        freq = torch.tensor([THETA ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device=k.device)
        x, at, out = st["qkv"].double(), 0, []
        for s, (p, n) in enumerate(zip(positions, counts)):
            depth = list(range(n)) if parent is None else _exact_depths(parent[at:at + n])
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=k.device),
                               (torch.tensor([p + e for e in depth], dtype=torch.float64, device=k.device)[:, None] * freq))
            part, new = x[at:at + n], []
            for block, g in ((part[:, :h], st["gq"]), (part[:, h:h + kv], st["gk"])):
                if g is not None:
                    block = block / (block.square().mean(-1, keepdim=True) + EPS).sqrt() * g.double()
                z = torch.view_as_complex(block.reshape(n, -1, d // 2, 2).contiguous()) * turn[:, None]
                new.append(torch.view_as_real(z).reshape(n, -1, d))
            slots = [_exact_slot(p + j, c) for j in range(n)]
            out.append(new[0])
            k[0, s, slots], v[0, s, slots] = new[1], part[:, h + kv:]
            at += n
        return {"q": torch.cat(out), "k": k, "v": v}
    if _pairs(c) * h * d > 3e12:
        return None
    ring, at, outs, lses = c["cap"] - c["sinks"], 0, [], []
    for s, (p, n) in enumerate(zip(positions, counts)):
        end = p + n
        keys = list(range(min(end, c["sinks"]))) + list(range(max(c["sinks"], end - ring), end))
        slots = torch.tensor([_exact_slot(j, c) for j in keys], device="cuda")
        j = torch.tensor(keys, device="cuda")
        if op == "tree":
            par = parent[at:at + n]
            depth = _exact_depths(par)
            line = torch.zeros(n, n, dtype=torch.bool)
            for i in range(n):
                line[i, i] = True
                if par[i] >= 0:
                    line[i] |= line[par[i]]
            line = line.cuda()
            dep = torch.tensor(depth, device="cuda")
            logical = torch.where(j >= p, p + dep[(j - p).clamp(min=0)], j)
            mine = torch.where((j >= p)[None], line[:, (j - p).clamp(min=0)], True)
            here = p + dep
        else:
            here = p + torch.arange(n, device="cuda")
            logical, mine = j, j[None] <= here[:, None]
        if c["window"]:
            mine = mine & ((logical[None] > here[:, None] - c["window"]) | (logical < c["sinks"])[None])
        o, e = [], []
        for g in range(kv):
            k, v = st["k"][0, s, slots, g].double(), st["v"][0, s, slots, g].double()
            for head in range(g * (h // kv), (g + 1) * (h // kv)):
                a = st["q"][at:at + n, head].double() @ k.T / math.sqrt(d)
                a = a.masked_fill(~mine, -math.inf)
                z = torch.logsumexp(a, -1)
                e.append(z)
                o.append((a - z[:, None]).exp() @ v)
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(e, 1))
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
