"""What the serving operators of the library are measured on: rotary positions and
their tables, a KV cache that is quantised as it is written, attention over that cache
(single tokens, prompt chunks, trees of drafted tokens) and log probabilities.

`listed()` names the cases, `draw(rng)` makes another one of the same ranges, `prepare`
builds what a program holds before the call, `run` is one pass through an operator (its
plain form, or with `own` the library's entry points), `work` the bytes and operations
such a pass cannot do without, and `exact` its results in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # The tables of a model with a 4096-token context, made when it is loaded.
        dict(name="tables_4k", op="tables", count=4096, first=0, half=32, base=500000.0,
             scaling="none", factor=1.0),
        # The tables of a context extended 32 times, all 131072 positions.
        dict(name="tables_yarn_128k", op="tables", count=131072, first=0, half=64, base=10000.0,
             scaling="yarn", factor=32.0),
        # One decoded token of 32 sequences, far positions: latency counts.
        dict(name="rotate_decode", op="rotate", batch=32, seq=1, heads=40, d=128, half=64,
             interleaved=False, far=130000, pad=0),
        # The query heads of an odd-length prompt inside fused q/k/v rows, pairs
        # side by side, part of the head.
        dict(name="rotate_prompt", op="rotate", batch=1, seq=8191, heads=32, d=128, half=32,
             interleaved=True, far=8191, pad=2048),
        # One token of each of 64 sequences written, rotated, to an e4m3 cache and read back.
        dict(name="cache_decode", op="cache", fmt="e4m3", batch=64, new_lo=1, new_hi=1,
             past_lo=1000, past_hi=8000, kv_heads=8, d=128, page=64, half=64, interleaved=False),
        # Four prompts of unequal lengths written to an int8 cache and read back.
        dict(name="cache_prompt", op="cache", fmt="int8", batch=4, new_lo=1001, new_hi=4096,
             past_lo=0, past_hi=0, kv_heads=8, d=128, page=64, half=64, interleaved=False),
        # A tree of 25 drafted tokens of one chat over an int4 cache: the smallest attention.
        dict(name="attend_tree", op="attend", fmt="int4", batch=1, new_lo=25, new_hi=25,
             past_lo=1900, past_hi=1900, heads=32, kv_heads=8, d=128, page=64, half=64,
             interleaved=False, tree=True),
        # One token of each of 64 sequences over their e4m3 caches.
        dict(name="attend_decode", op="attend", fmt="e4m3", batch=64, new_lo=1, new_hi=1,
             past_lo=2000, past_hi=8000, heads=32, kv_heads=8, d=128, page=64, half=64,
             interleaved=False, tree=False),
        # One token over a 131071-token int8 cache.
        dict(name="attend_long", op="attend", fmt="int8", batch=1, new_lo=1, new_hi=1,
             past_lo=131071, past_hi=131071, heads=32, kv_heads=8, d=128, page=128, half=0,
             interleaved=False, tree=False),
        # Chunks of two prompts over what is already cached: the most arithmetic.
        dict(name="attend_prompt", op="attend", fmt="int8", batch=2, new_lo=1500, new_hi=2048,
             past_lo=4000, past_hi=6144, heads=32, kv_heads=8, d=64, page=64, half=32,
             interleaved=False, tree=False),
        # Decoded tokens' log probabilities with 20 alternatives each.
        dict(name="logprobs_decode", op="logprobs", rows=8, vocab=151936, top=20, masked=False,
             coarse=False),
        # A whole prompt's, from logits rounded to bf16 (equal values) with masked tokens.
        dict(name="logprobs_prompt", op="logprobs", rows=1000, vocab=128256, top=8, masked=True,
             coarse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "rotate", "cache", "cache", "attend", "attend", "attend", "attend",
                     "logprobs", "logprobs"])
    if op == "tables":
        count = _log(rng, 256, 131072)
        return dict(op=op, count=count, first=rng.randint(0, 131072 - count),
                    half=rng.randint(8, 64), base=float(rng.choice([10000, 500000, 1000000])),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                    factor=float(rng.choice([2, 4, 8, 32])))
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    half = rng.choice([0, d // 4, d // 2, d // 2])
    inter = rng.random() < 0.3
    if op == "rotate":
        batch = _log(rng, 1, 64)
        seq = rng.choice([1, _log(rng, 2, 8191 // batch)])
        return dict(op=op, batch=batch, seq=seq, heads=rng.randint(1, 32) * 128 // max(d, 128), d=d,
                    half=half or d // 2, interleaved=inter, far=rng.choice([8191, 130000]),
                    pad=rng.choice([0, 0, 64, 2048]))
    if op == "logprobs":
        vocab = _log(rng, 1000, 151936)
        rows = _log(rng, 1, min(2048, 1000 * 128256 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, 64]),
                    masked=rng.random() < 0.3, coarse=rng.random() < 0.3)
    fmt = rng.choice(["int8", "e4m3", "int4"])
    kv = rng.choice([1, 2, 4, 8, 8])
    if op == "cache":
        batch = _log(rng, 1, 64)
        hi = rng.choice([1, _log(rng, 2, 8192 // batch)])
        past = rng.choice([0, _log(rng, 1, 8000)])
        return dict(op=op, fmt=fmt, batch=batch, new_lo=(hi + 1) // 2, new_hi=hi,
                    past_lo=past // 2, past_hi=past, kv_heads=kv, d=d, page=page, half=half,
                    interleaved=inter)
    group = rng.choice([1, 2, 4, 4, 7, 8])
    form = rng.choice(["one", "tree", "prompt"])
    # Bounded so that neither the cached bytes nor the products exceed the listed ones.
    if form == "one":
        batch = _log(rng, 1, 64)
        hi, past = 1, _log(rng, 16, min(131071, 64 * 4096 * 1024 // (batch * kv * d)))
    elif form == "tree":
        batch = _log(rng, 1, 8)
        hi, past = rng.randint(4, 64), _log(rng, 16, 8000)
    else:
        batch = _log(rng, 1, 4)
        hi = _log(rng, 16, min(2048, 2048 * 2 * 32 * 64 // (batch * kv * group * d)))
        past = rng.choice([0, _log(rng, 16, 6144)])
    return dict(op=op, fmt=fmt, batch=batch, new_lo=(hi + 1) // 2, new_hi=hi,
                past_lo=(past + 1) // 2, past_hi=past, heads=kv * group, kv_heads=kv, d=d,
                page=page, half=half, interleaved=inter, tree=form == "tree")


# ------------------------------------------------------------------ inputs


def _lengths(c):
    """New rows and cached tokens of each sequence: the case's, whatever the seed."""
    rng = random.Random(c["batch"] * 1000003 + c["past_hi"] * 31 + c["new_hi"])
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]
    past = [rng.randint(c["past_lo"], c["past_hi"]) for _ in range(c["batch"])]
    return new, past


def _inv_freq(c):
    """The scaled frequencies of a rotary table and the factor on its values."""
    half, base, f, length = c["half"], c["base"], c["factor"], 4096.0
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    inv = base ** (-i / half)
    if c["scaling"] == "linear":
        return inv / f, 1.0
    if c["scaling"] == "ntk":
        return (base * f ** (half / (half - 1))) ** (-i / half), 1.0
    if c["scaling"] == "yarn":
        at = [half * math.log(length / (beta * 2 * math.pi)) / math.log(base) for beta in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), 2 * half - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    if c["scaling"] == "bands":
        turns = length * inv / (2 * math.pi)  # rotations over the original length
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv / f * (1 - keep) + inv * keep, 1.0
    return inv, 1.0


def _tree(c, g, new, words=1):
    """Random trees of drafted tokens: each row's ancestors and itself as bits, its depth."""
    n = torch.tensor(new, device=DEV)
    top, batch = max(new), len(new)
    at = torch.arange(top, device=DEV)
    parent = (torch.rand(batch, top, generator=g, device=DEV) * (at + 1)).long() - 1  # -1: the root
    link = (parent[:, :, None] == at).double() + torch.eye(top, device=DEV, dtype=torch.float64)
    seen = torch.linalg.matrix_power(link, 64) > 0.5
    bits = (seen.long() << at).sum(-1)  # at most 64 drafted tokens: one word a row
    rows = at < n[:, None]
    return bits[rows].view(-1, words).contiguous(), (seen.sum(-1) - 1)[rows].to(torch.int32)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _sequences(c, g):
    """The packed rows of a batch, its page table and positions, three padding rows behind."""
    new, past = _lengths(c)
    rows = sum(new) + 3
    start = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    past_t = torch.tensor(past, device=DEV, dtype=torch.int32)
    n = torch.tensor(new, device=DEV)
    width = max(-(-(a + b) // c["page"]) for a, b in zip(new, past))
    pages = c["batch"] * width
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(c["batch"], width)
    seq = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), n)
    i = torch.arange(sum(new), device=DEV) - start[:-1].long()[seq]
    t = dict(new=new, past=past, rows=rows, start=start, past_t=past_t, table=table, pages=pages,
             seq=seq, i=i, max_new=c["new_hi"], max_len=c["new_hi"] + c["past_hi"])
    t["positions"] = (past_t.long()[seq] + i).to(torch.int32)
    if c.get("tree"):
        t["bits"], depth = _tree(c, g, new)
        t["positions"] = past_t[seq] + depth
    pad = torch.zeros(3, device=DEV, dtype=torch.int32)
    t["positions"] = torch.cat([t["positions"], pad])
    if "bits" in t:
        t["bits"] = torch.cat([t["bits"], torch.zeros(3, 1, device=DEV, dtype=torch.int64)])
    return t


def _rope_tables(c, count):
    pos = torch.arange(count, device=DEV, dtype=torch.float64)[:, None]
    freq = 500000.0 ** (-torch.arange(c["half"], device=DEV, dtype=torch.float64) / c["half"])
    return torch.cos(pos * freq).float(), torch.sin(pos * freq).float()


def _keys(g, rows, c):
    """Keys and values as layers make them: some channels of the keys are larger."""
    k, v = (_normal(g, rows, c["kv_heads"], c["d"]) for _ in range(2))
    return k * torch.exp(0.6 * _normal(g, c["kv_heads"], c["d"])), v


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if c["op"] == "tables":
        # (What is read is the case itself; the seed moves the first position.)
        return dict(first=max(0, min(c["first"] + int(seed) % 997, 200000)))
    if c["op"] == "rotate":
        x = _normal(g, c["batch"], c["seq"], c["heads"] * c["d"] + c["pad"])
        last = torch.randint(c["seq"] - 1, max(c["far"], c["seq"]), (c["batch"], 1), generator=g,
                             device=DEV)
        pos = (last - c["seq"] + 1 + torch.arange(c["seq"], device=DEV)).to(torch.int32)
        cos, sin = _rope_tables(c, max(c["far"], c["seq"]))
        return dict(x=x, pos=pos, cos=cos, sin=sin)
    if c["op"] == "logprobs":
        x = 2.5 * _normal(g, c["rows"], c["vocab"])
        x[:, :: max(1, c["vocab"] // 7)] += 6.0 * torch.rand(c["rows"], 1, generator=g, device=DEV)
        if c["coarse"]:
            x = x.to(torch.bfloat16).float()
        tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=DEV)
        if c["masked"]:  # a grammar's mask, never over the given token
            x[torch.rand(c["rows"], c["vocab"], generator=g, device=DEV) < 0.4] = -math.inf
            x[torch.arange(c["rows"], device=DEV), tokens] = 1.0
        return dict(x=x, tokens=tokens.to(torch.int32))
    t = _sequences(c, g)
    if c["half"]:
        t["cos"], t["sin"] = _rope_tables(c, t["max_len"])
    if c["op"] == "cache":
        t["k"], t["v"] = _keys(g, t["rows"], c)
        return t
    # What earlier steps and this step's write have put into the cache, and the queries.
    t["total"] = [a + b for a, b in zip(t["new"], t["past"])]
    t["all_k"], t["all_v"] = _keys(g, sum(t["total"]), c)
    t["q"] = _normal(g, t["rows"], c["heads"], c["d"])
    return t


# ------------------------------------------------------------- plain forms


def _rotate(x, cos, sin, interleaved):
    """Pairs of the first 2 * half elements turned by their angle, in 64 bits, rounded once."""
    half = cos.shape[-1]
    a, rest = x[..., : 2 * half].double(), x[..., 2 * half:]
    cos, sin = cos.double(), sin.double()
    p, q = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., :half], a[..., half:])
    u, w = p * cos - q * sin, q * cos + p * sin
    y = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([y.float(), rest], -1)


def _quantise(x, fmt):
    """Codes, scale and (int4) middle of each vector along the last dimension."""
    if fmt == "int4":
        hi, lo = x.amax(-1, keepdim=True).double(), x.amin(-1, keepdim=True).double()
        mid, h = ((hi + lo) / 2).float(), ((hi - lo) / 30).float()
        u = (x.double() - mid.double()) / torch.where(h > 0, h, 1.0).double()
        return ((u + 15) / 2).round().clamp(0, 15).to(torch.uint8), h, mid
    scale = (x.abs().amax(-1, keepdim=True).double() / (127 if fmt == "int8" else 448)).float()
    u = x.double() / torch.where(scale > 0, scale, 1.0).double()
    if fmt == "int8":
        return u.round().clamp(-127, 127).to(torch.int8), scale, None
    step = torch.ldexp(torch.ones_like(u), (torch.frexp(u)[1] - 1).clamp(min=-6) - 3)
    return ((u / step).round() * step).clamp(-448, 448).float().to(torch.float8_e4m3fn), scale, None


def _values(code, scale, mid):
    """What the codes stand for."""
    if mid is None:
        return code.float() * scale
    return mid + (2 * code.float() - 15) * scale


def _pages(t, c, codes, scale, mid, slot):
    """Codes and scales of packed rows in pages, each row at its slot."""
    n = t["pages"] * c["page"]
    out = []
    for x in (codes, scale, mid):
        if x is None:
            out.append(None)
            continue
        b = torch.zeros((n,) + x.shape[1:], device=DEV, dtype=torch.uint8 if x.element_size() == 1 else x.dtype)
        b[slot] = x.view(torch.uint8) if x.element_size() == 1 else x
        out.append(b.view(x.dtype))
    return out


def _slots(t, c, seq, pos):
    return t["table"][seq, pos // c["page"]].long() * c["page"] + pos % c["page"]


def _plain_attend(s):
    c, t = s["c"], s["t"]
    b, n, heads, kv, d = c["batch"], max(t["new"]), c["heads"], c["kv_heads"], c["d"]
    group, length = heads // kv, max(t["total"])
    rows = t["seq"].numel()
    q = t["q"][:rows]
    if c["half"]:
        pos = t["positions"][:rows].long()
        q = _rotate(q, t["cos"][pos][:, None], t["sin"][pos][:, None], c["interleaved"])
    qb = torch.zeros(b, n, heads, d, device=DEV)
    qb[t["seq"], t["i"]] = q
    qb = qb.view(b, n, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b * kv, group * n, d)
    at = torch.arange(length, device=DEV)
    slot = _slots(t, c, torch.arange(b, device=DEV)[:, None], at.clamp(max=t["table"].shape[1] * c["page"] - 1)[None])

    def cached(x):
        # (8-bit floats are gathered as bytes.)
        byte = x[0].element_size() == 1
        code = (x[0].view(torch.uint8) if byte else x[0])[slot].view(x[0].dtype)
        y = _values(code, x[1][slot], None if x[2] is None else x[2][slot])
        return y.permute(0, 2, 1, 3).reshape(b * kv, length, d)

    k, v = cached(s["kc"]), cached(s["vc"])
    score = torch.matmul(qb, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
    total = torch.tensor(t["total"], device=DEV)[:, None, None]
    past = t["past_t"].long()[:, None, None]
    i = torch.arange(n, device=DEV)[None, :, None]
    key = at[None, None, :]
    if c["tree"]:
        bits = torch.zeros(b, n, device=DEV, dtype=torch.int64)
        bits[t["seq"], t["i"]] = t["bits"][:rows, 0]
        drafted = (bits[:, :, None] >> (key - past).clamp(0, 63)) & 1
        seen = (key < total) & ((key < past) | (drafted == 1))
    else:
        seen = (key <= past + i) & (key < total)
    score = score.view(b, kv, group, n, length)
    score = torch.where(seen[:, None, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    z = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(b * kv, group * n, length), v).view(b, kv, group, n, d) / z
    y = y.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)
    out = torch.zeros(t["rows"], heads, d, device=DEV)
    out[:rows] = y[t["seq"], t["i"]]
    return out


def _plain(s):
    c, t = s["c"], s["t"]
    if c["op"] == "tables":
        inv, a = _inv_freq(c)
        angle = (t["first"] + torch.arange(c["count"], device=DEV, dtype=torch.float64))[:, None] * inv
        return (torch.cos(angle) * a).float(), (torch.sin(angle) * a).float()
    if c["op"] == "rotate":
        x = t["x"][..., : c["heads"] * c["d"]].view(c["batch"], c["seq"], c["heads"], c["d"])
        pos = t["pos"].long()
        return _rotate(x, t["cos"][pos][:, :, None], t["sin"][pos][:, :, None], c["interleaved"])
    if c["op"] == "logprobs":
        x, top = t["x"], c["top"]
        e = x - x.amax(-1, keepdim=True)
        p = torch.exp(e)
        z = p.sum(-1, keepdim=True)
        lp = e - torch.log(z)
        h = -(torch.where(p > 0, lp, 0.0) * p).sum(-1, keepdim=True) / z
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
        given = lp.gather(1, t["tokens"].long()[:, None])
        return given[:, 0], h[:, 0], ids.to(torch.int32), lp.gather(1, ids)
    if c["op"] == "cache":
        rows = t["seq"].numel()
        k, v = t["k"][:rows], t["v"][:rows]
        pos = t["positions"][:rows].long()
        if c["half"]:
            k = _rotate(k, t["cos"][pos][:, None], t["sin"][pos][:, None], c["interleaved"])
        out = []
        for x in (k, v):
            y = torch.zeros(t["rows"], c["kv_heads"], c["d"], device=DEV)
            y[:rows] = _values(*_quantise(x, c["fmt"]))
            out.append(y)
        return tuple(out)
    return _plain_attend(s)


# -------------------------------------------------------- the library's calls


def _ops():
    from onnx_runtime_dart_amd import ops
    return ops


def _context():
    """The thread's library context, on torch's stream."""
    ctx = _ops().default_context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return ctx


def _batch(t, c, start, past, rows, max_new, max_len):
    """The library's description of a batch of sequences (device arrays by address)."""
    return _ops().SeqBatch(batch=c["batch"], rows=rows, max_new=max_new, max_len=max_len,
                           row_start_ptr=start.data_ptr(), past_ptr=past.data_ptr(),
                           page_table_ptr=t["table"].data_ptr(), table_stride=t["table"].shape[1])


def _own_prepare(s):
    ops = _ops()
    c, t = s["c"], s["t"]
    s["ctx"] = _context()
    if c["op"] == "tables":
        s["cos"], s["sin"] = (torch.empty(c["count"], c["half"], device=DEV) for _ in range(2))
        s["scaling"] = ops.RopeScaling(c["scaling"], factor=c["factor"], original_length=4096)
    if c["op"] == "rotate":
        s["y"] = torch.empty(c["batch"], c["seq"], c["heads"], c["d"], device=DEV)
        s["rope"] = ops.Rope(t["cos"].data_ptr(), t["sin"].data_ptr(), max_pos=t["cos"].shape[0],
                             half_rot=c["half"], interleaved=c["interleaved"],
                             positions_ptr=t["pos"].data_ptr())
        row = c["heads"] * c["d"] + c["pad"]
        s["strides"] = (c["seq"] * row, row, c["d"])
    if c["op"] == "logprobs":
        n, top = c["rows"], c["top"]
        s["given"], s["entropy"] = (torch.empty(n, device=DEV) for _ in range(2))
        s["ids"] = torch.empty(n, top, device=DEV, dtype=torch.int32)
        s["tops"] = torch.empty(n, top, device=DEV)
    if c["op"] not in ("cache", "attend"):
        return s
    s["cache"] = ops.KvCache(t["pages"], kv_heads=c["kv_heads"], head_size=c["d"],
                             page_size=c["page"], fmt=c["fmt"], ctx=s["ctx"])
    s["batch"] = _batch(t, c, t["start"], t["past_t"], t["rows"], t["max_new"], t["max_len"])
    s["rope"] = ops.Rope(t["cos"].data_ptr(), t["sin"].data_ptr(), max_pos=t["cos"].shape[0],
                         half_rot=c["half"], interleaved=c["interleaved"],
                         positions_ptr=t["positions"].data_ptr()) if c["half"] else None
    if c["op"] == "cache":
        s["ky"], s["vy"] = (torch.zeros(t["rows"], c["kv_heads"], c["d"], device=DEV) for _ in range(2))
        return s
    s["y"] = torch.zeros(t["rows"], c["heads"], c["d"], device=DEV)
    # What earlier steps left in the cache: written once, as they write it.
    start = torch.tensor([0] + t["total"], device=DEV).cumsum(0).to(torch.int32)
    none = torch.zeros(c["batch"], device=DEV, dtype=torch.int32)
    total = sum(t["total"])
    s["cache"].append_dev(_batch(t, c, start, none, total, t["max_len"], t["max_len"]),
                          t["all_k"].data_ptr(), t["all_v"].data_ptr())
    torch.cuda.synchronize()
    return s


def _own_run(s):
    ops = _ops()
    c, t = s["c"], s["t"]
    if c["op"] == "tables":
        ops.rotary_tables_dev(s["cos"].data_ptr(), s["sin"].data_ptr(), t["first"], c["count"],
                              c["half"], base=c["base"], scaling=s["scaling"], ctx=s["ctx"])
        return s["cos"], s["sin"]
    if c["op"] == "rotate":
        ops.rotary_embedding_dev(t["x"].data_ptr(), c["batch"], c["seq"], c["heads"], c["d"],
                                 s["rope"], s["y"].data_ptr(), x_strides=s["strides"], ctx=s["ctx"])
        return s["y"]
    if c["op"] == "logprobs":
        ops.token_logprobs_dev(t["x"].data_ptr(), c["rows"], c["vocab"], tokens_ptr=t["tokens"].data_ptr(),
                               logprob_ptr=s["given"].data_ptr(), entropy_ptr=s["entropy"].data_ptr(),
                               top=c["top"], top_ids_ptr=s["ids"].data_ptr(),
                               top_logprobs_ptr=s["tops"].data_ptr(), ctx=s["ctx"])
        return s["given"], s["entropy"], s["ids"], s["tops"]
    if c["op"] == "cache":
        s["cache"].append_dev(s["batch"], t["k"].data_ptr(), t["v"].data_ptr(), rope=s["rope"])
        s["cache"].read_dev(s["batch"], s["ky"].data_ptr(), s["vy"].data_ptr())
        return s["ky"], s["vy"]
    s["cache"].attend_dev(s["batch"], t["q"].data_ptr(), s["y"].data_ptr(), c["heads"], rope=s["rope"],
                          tree_ptr=t["bits"].data_ptr() if c["tree"] else 0, tree_words=1 if c["tree"] else 0)
    return s["y"]


def prepare(case, seed):
    c = case
    t = _inputs(c, seed)
    s = dict(c=c, t=t)
    if own:
        s = _own_prepare(s)
    elif c["op"] == "attend":
        total = torch.tensor(t["total"], device=DEV)
        seq = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), total)
        first = torch.cat([total.new_zeros(1), total.cumsum(0)[:-1]])
        pos = torch.arange(seq.numel(), device=DEV) - first[seq]
        slot = _slots(t, c, seq, pos)
        s["kc"] = _pages(t, c, *_quantise(t["all_k"], c["fmt"]), slot)
        s["vc"] = _pages(t, c, *_quantise(t["all_v"], c["fmt"]), slot)
    for name in ("all_k", "all_v"):
        t.pop(name, None)
    return s


def run(state):
    return _own_run(state) if own else _plain(state)


# ------------------------------------------------------ bytes and operations


def work(case):
    c = case
    if c["op"] == "tables":
        n = c["count"] * c["half"]
        return dict(bytes=8 * n, flops=4 * n)
    if c["op"] == "rotate":
        n = c["batch"] * c["seq"]
        # (A table row is read once for each distinct position.)
        return dict(bytes=8 * n * c["heads"] * c["d"] + n * (8 * c["half"] + 4), flops=6 * n * c["heads"] * c["half"])
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return dict(bytes=4 * n + c["rows"] * (12 + 8 * c["top"]), flops=6 * n)
    new, past = _lengths(c)
    scales = 8 if c["fmt"] == "int4" else 4
    token = 2 * c["kv_heads"] * (c["d"] * (4 if c["fmt"] == "int4" else 8) // 8 + scales)
    if c["op"] == "cache":
        n = sum(new)
        vectors = 2 * c["kv_heads"] * c["d"] * 4
        return dict(bytes=n * (2 * vectors + 2 * token + 8 * c["half"]), flops=n * 2 * c["kv_heads"] * c["d"] * 4)
    keys = sum(new) + sum(past)
    if c["tree"]:
        pairs = sum(n * p + n * (n + 1) // 4 for n, p in zip(new, past))
    else:
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    return dict(bytes=keys * token + sum(new) * (8 * c["heads"] * c["d"] + 8 * c["half"]),
                flops=4 * c["heads"] * c["d"] * pairs)


# ------------------------------------------------------- results in 64 bits


def _exact_turn(x, cos, sin, interleaved):
    """Each pair as a complex number times cos + i sin; the result is an fp32 tensor's."""
    half = cos.shape[-1]
    y = x.double().clone()
    w = torch.complex(cos.double(), sin.double())
    at = torch.arange(half, device=DEV)
    a, b = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
    z = torch.complex(y[..., a], y[..., b]) * w
    y[..., a], y[..., b] = z.real, z.imag
    return y.float().double()


def _exact_cached(x, fmt):
    """What a cache of this format gives back for the vectors x (64 bits, of fp32 values)."""
    if fmt == "int4":
        top, low = x.max(-1, keepdim=True)[0], x.min(-1, keepdim=True)[0]
        m, h = ((top + low) * 0.5).float().double(), ((top - low) / 30.0).float().double()
        n = torch.floor(torch.where(h > 0, (x - m) / h, 0.0) * 0.5 + 7.5 + 0.5)
        # (Halves go to the even code.)
        half = torch.where(h > 0, (x - m) / h, 0.0) * 0.5 + 7.5
        n = torch.where((n - half == 0.5) & (n % 2 == 1), n - 1, n).clamp(0, 15)
        return m + (2 * n - 15) * h
    s = (x.abs().max(-1, keepdim=True)[0] / (127.0 if fmt == "int8" else 448.0)).float().double()
    u = torch.where(s > 0, x / s, 0.0)
    if fmt == "int8":
        return torch.round(u).clamp(-127, 127) * s
    # e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6.
    a = u.abs().clamp(min=2.0**-6)
    step = 2.0 ** (torch.floor(torch.log2(a)) - 3)
    step = torch.where(a >= 16 * step, 2 * step, torch.where(a < 8 * step, step / 2, step))
    return (torch.round(u / step) * step).clamp(-448, 448) * s


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    if c["op"] == "tables":
        inv, a = _inv_freq(c)
        turns = (t["first"] + torch.arange(c["count"], device=DEV, dtype=torch.float64))[:, None] * inv / (2 * math.pi)
        angle = (turns - torch.floor(turns)) * (2 * math.pi)
        return a * torch.cos(angle), a * torch.sin(angle)
    if c["op"] == "rotate":
        x = t["x"][..., : c["heads"] * c["d"]].reshape(c["batch"], c["seq"], c["heads"], c["d"])
        pos = t["pos"].long()
        return _exact_turn(x, t["cos"][pos].unsqueeze(2), t["sin"][pos].unsqueeze(2), c["interleaved"])
    if c["op"] == "logprobs":
        given, entropy, tops = [], [], []
        for i in range(c["rows"]):
            x = t["x"][i].double()
            m = x.max()
            log_z = torch.log(torch.exp(x - m).sum()) + m
            seen = x[x > -math.inf] - log_z
            given.append(x[int(t["tokens"][i])] - log_z)
            entropy.append(-(torch.exp(seen) * seen).sum())
            tops.append(torch.sort(x, descending=True)[0][: c["top"]] - log_z)
        return torch.stack(given), torch.stack(entropy), None, torch.stack(tops)
    rows = t["seq"].numel()
    pos = t["positions"][:rows].long()
    if c["op"] == "cache":
        k, v = t["k"][:rows].double(), t["v"][:rows].double()
        if c["half"]:
            k = _exact_turn(k, t["cos"][pos].unsqueeze(1), t["sin"][pos].unsqueeze(1), c["interleaved"])
        out = []
        for x in (k, v):
            y = torch.zeros(t["rows"], c["kv_heads"], c["d"], device=DEV, dtype=torch.float64)
            y[:rows] = _exact_cached(x, c["fmt"])
            out.append(y)
        return tuple(out)
    q = t["q"][:rows].double()
    if c["half"]:
        q = _exact_turn(q, t["cos"][pos].unsqueeze(1), t["sin"][pos].unsqueeze(1), c["interleaved"])
    out = torch.zeros(t["rows"], c["heads"], c["d"], device=DEV, dtype=torch.float64)
    group, row, key = c["heads"] // c["kv_heads"], 0, 0
    for n, p in zip(t["new"], t["past"]):
        sees = torch.ones(n, n + p, device=DEV, dtype=torch.bool).tril(p)
        if c["tree"]:
            drafted = torch.arange(n, device=DEV)
            sees[:, p:] = (t["bits"][row:row + n] >> drafted) & 1 != 0
        for h in range(c["kv_heads"]):
            k, v = (_exact_cached(t[name][key:key + n + p, h].double(), c["fmt"]) for name in ("all_k", "all_v"))
            for j in range(h * group, (h + 1) * group):
                s = q[row:row + n, j] @ k.T.contiguous() / math.sqrt(c["d"])
                s = s.masked_fill(~sees, -math.inf)
                out[row:row + n, j] = torch.softmax(s, -1) @ v
        row, key = row + n, key + n + p
    return out
