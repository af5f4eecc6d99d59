"""What the operators around a batch of requests are measured on: the verification of drafted
tokens, the pages of the quantised KV cache (copied, compacted, forked and fitted to lengths)
and low-rank adapters beside a shared projection.

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
        # Four drafted tokens of one chat, small vocabulary: latency counts.
        dict(name="verify_one", op="verify", batch=1, new_lo=5, new_hi=5, vocab=32000, tree=False,
             draft=True, greedy=0.0),
        # Four to eight drafted tokens of each of 64 chats, some of them greedy.
        dict(name="verify_batch", op="verify", batch=64, new_lo=5, new_hi=9, vocab=151936, tree=False,
             draft=True, greedy=0.2),
        # Trees of 25 tokens that a draft head proposed, for 8 chats.
        dict(name="verify_tree", op="verify", batch=8, new_lo=25, new_hi=25, vocab=128256, tree=True,
             draft=False, greedy=0.1),
        # q, k and v of a small layer for four requests with an adapter each: the smallest.
        dict(name="adapt_few", op="adapt", k=1024, ns="2048 1024 1024", slots=4, rank=8, fmt="f16",
             prompts="", tokens=4, none=0.0),
        # One decoded token of each of 64 requests, most with adapters of their own.
        dict(name="adapt_decode", op="adapt", k=2048, ns="2048", slots=96, rank=32, fmt="f32",
             prompts="", tokens=64, none=0.1),
        # Prompts of unequal lengths together with decoded tokens of other requests.
        dict(name="adapt_mixed", op="adapt", k=2048, ns="2048 512 512", slots=32, rank=16, fmt="f16",
             prompts="1203 777 401 64 1", tokens=48, none=0.1),
        # Gate and up of long prompts, wide adapters: the most arithmetic.
        dict(name="adapt_prompts", op="adapt", k=2048, ns="8192 8192", slots=8, rank=64, fmt="f32",
             prompts="4095 2500 1596", tokens=0, none=0.0),
        # 25 drafted tokens of 64 chats written; those that were accepted move together.
        dict(name="compact_drafts", op="compact", fmt="int8", batch=64, new_lo=25, new_hi=25,
             past_lo=1000, past_hi=4000, keep=0.16, evict=False, kv_heads=8, d=128, page=64),
        # A copy of long sequences keeps half of its tokens.
        dict(name="compact_long", op="compact", fmt="e4m3", batch=4, new_lo=7001, new_hi=8192,
             past_lo=0, past_hi=0, keep=0.5, evict=True, kv_heads=8, d=128, page=64),
        # Pages of an int4 cache copied (a prompt that becomes another request's own).
        dict(name="copy_pages", op="copy", fmt="int4", pages=128, kv_heads=8, d=128, page=64),
        # One prompt becomes 4 answers: pages are shared, the last ones copied when written.
        dict(name="fork_one", op="fork", fmt="int8", parents=1, children=4, past_lo=1000, past_hi=1000,
             new=1, spare=1.0, kv_heads=8, d=128, page=16),
        # Beams of 16 searches change places, too few pages for some of the last.
        dict(name="fork_beams", op="fork", fmt="int8", parents=64, children=64, past_lo=500,
             past_hi=4000, new=4, spare=0.9, kv_heads=8, d=128, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["verify", "verify", "verify", "adapt", "adapt", "adapt", "adapt", "compact",
                     "compact", "copy", "fork"])
    if op == "verify":
        vocab = _log(rng, 1000, 151936)
        tree = rng.random() < 0.35
        hi = _log(rng, 8, 64) if tree else _log(rng, 1, 17)
        draft = not tree and rng.random() < 0.7
        # Bounded by the logits of the largest listed case.
        most = 64 * 7 * 2 * 151936 // (vocab * hi * (2 if draft else 1))
        return dict(op=op, batch=_log(rng, 1, max(1, min(256, most))), new_lo=(hi + 1) // 2, new_hi=hi,
                    vocab=vocab, tree=tree, draft=draft, greedy=rng.choice([0.0, 0.2, 1.0]))
    if op == "adapt":
        k = _log(rng, 128, 4096)
        ns = [_log(rng, 64, 8192) for _ in range(rng.choice([1, 1, 2, 3, 4]))]
        ns = [n // len(ns) + 1 for n in ns]
        rank = rng.choice([1, 4, 8, 16, 16, 32, 64, rng.randint(1, 128)])
        slots = _log(rng, 1, 96)
        form = rng.choice(["tokens", "prompts", "both"])
        tokens = 0 if form == "prompts" else _log(rng, 1, 512)
        # Bounded by the arithmetic of the largest listed case.
        most = max(16, 8191 * (2 * 2048 + 16384) // (k * len(ns) + sum(ns)) * 64 // max(rank, 64))
        left = _log(rng, 16, min(8191, most))
        prompts = []
        while form != "tokens" and left > 0 and len(prompts) < 8:
            prompts.append(rng.randint(1, left))
            left -= prompts[-1]
        return dict(op=op, k=k, ns=" ".join(map(str, ns)), slots=slots, rank=rank,
                    fmt=rng.choice(["f32", "f16"]), prompts=" ".join(map(str, prompts)), tokens=tokens,
                    none=rng.choice([0.0, 0.1, 0.5]))
    d = rng.choice([64, 80, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    fmt = rng.choice(["int8", "e4m3", "int4"])
    if op == "copy":
        most = max(1, 4 * 8192 * 1024 // (kv * d * page))
        return dict(op=op, fmt=fmt, pages=_log(rng, 1, most), kv_heads=kv, d=d, page=page)
    if op == "fork":
        parents = _log(rng, 1, 64)
        past = _log(rng, 16, 4000)
        return dict(op=op, fmt=fmt, parents=parents, children=_log(rng, 1, 128), past_lo=(past + 1) // 2,
                    past_hi=past, new=rng.choice([1, 1, 4, 64]), spare=rng.choice([0.5, 0.9, 1.0, 1.5]),
                    kv_heads=kv, d=d, page=page)
    evict = rng.random() < 0.4
    if evict:
        batch = _log(rng, 1, 8)
        hi = _log(rng, 16, min(8192, 4 * 8192 * 1024 // (batch * kv * d)))
        past = 0
    else:
        batch = _log(rng, 1, 64)
        hi = rng.randint(1, 64)
        past = rng.choice([0, _log(rng, 1, 4000)])
    return dict(op=op, fmt=fmt, batch=batch, new_lo=(hi + 1) // 2, new_hi=hi, past_lo=past // 2,
                past_hi=past, keep=rng.choice([0.1, 0.3, 0.5, 0.9]), evict=evict, kv_heads=kv, d=d,
                page=page)


# ------------------------------------------------------------------ inputs


def _sizes(c, n, lo, hi, salt):
    """n numbers of the case, whatever the seed."""
    rng = random.Random(n * 1000003 + hi * 31 + salt)
    return [rng.randint(lo, hi) for _ in range(n)]


def _ints(text):
    return [int(x) for x in text.split()]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _int(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def _starts(new):
    return _int([sum(new[:i]) for i in range(len(new) + 1)])


def _logits(g, rows, vocab):
    x = 2.5 * _normal(g, rows, vocab)
    # A few likely tokens, as trained models have them.
    at = torch.randint(0, vocab // 6, (rows, 6), generator=g, device=DEV) + vocab // 6 * torch.arange(6, device=DEV)
    return x.scatter_add_(1, at, 5.0 + 4.0 * torch.rand(rows, 6, generator=g, device=DEV))


def _verify_inputs(c, g):
    new = _sizes(c, c["batch"], c["new_lo"], c["new_hi"], 1)
    rows, vocab = sum(new), c["vocab"]
    start = _starts(new)
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
    i = torch.arange(rows, device=DEV) - start[:-1].long()[seq]
    temp = 0.5 + 0.7 * torch.rand(len(new), generator=g, device=DEV)
    temp[torch.rand(len(new), generator=g, device=DEV) < c["greedy"]] = 0.0
    t = dict(new=new, rows=rows, start=start, seq=seq, i=i, temp=temp)
    t["target"] = _logits(g, rows, vocab)
    drafted = 0.9 * t["target"] + 0.8 * _normal(g, rows, vocab)
    if c["tree"]:
        # A row hangs under an earlier one, with the next of that one's likely tokens.
        up = (torch.rand(rows, generator=g, device=DEV) ** 2 * i).long()
        same = (seq[:, None] == seq[None]) & (up[:, None] == up[None]) & (i[None] < i[:, None]) & (i[None] > 0)
        nth = same.sum(1).clamp(max=vocab - 1)
        above = (start[:-1].long()[seq] + up)
        likely = drafted.topk(min(64, vocab), dim=1)[1]
        tokens = likely[above, nth]
        t["parent"] = torch.where(i > 0, up, -1).to(torch.int32)
    else:
        above = (torch.arange(rows, device=DEV) - 1).clamp(min=0)
        warm = torch.where(temp > 0, temp, 1.0)[seq][:, None]
        noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device=DEV).clamp(1e-9, 1 - 1e-7)))
        noise *= (temp > 0)[seq][:, None]
        tokens = (drafted / warm + noise).argmax(1)[above]
    t["tokens"] = tokens.to(torch.int32)
    t["uniform"] = torch.rand(rows, generator=g, device=DEV)
    if c["draft"]:
        t["draft"] = drafted
    return t


def _adapt_inputs(c, g):
    # The rows of the prompts, then single tokens; requests take adapters at random.
    rng = random.Random(c["k"] * 31 + c["rank"] * 7 + c["tokens"])
    slot = []
    for n in _ints(c["prompts"]) + [1] * c["tokens"]:
        slot += [-1 if rng.random() < c["none"] else rng.randrange(c["slots"])] * n
    # (Decoded tokens are in no order of their adapters.)
    rows, k, r = len(slot), c["k"], c["rank"]
    t = dict(rows=rows, host_slot=slot, slot=_int(slot), x=_normal(g, rows, k))
    t["base"] = [_normal(g, rows, n) for n in _ints(c["ns"])]
    kind = torch.float16 if c["fmt"] == "f16" else torch.float32
    t["a"] = [(_normal(g, c["slots"], r, k) / math.sqrt(k)).to(kind) for _ in _ints(c["ns"])]
    t["b"] = [(0.3 * _normal(g, c["slots"], n, r) / math.sqrt(r)).to(kind) for n in _ints(c["ns"])]
    t["scale"] = [float(2.0 ** rng.randint(-1, 1)) for _ in range(c["slots"])]
    return t


def _keys(g, rows, c):
    """Keys and values as layers make them: some channels of the keys are larger."""
    k, v = (_normal(g, rows, c["kv_heads"], c["d"]) for _ in range(2))
    return k * torch.exp(0.6 * _normal(g, c["kv_heads"], c["d"])), v


def _table(g, need, width, first=0):
    """Pages for sequences of `need` pages each from shuffled ones; -1 behind."""
    total = sum(need)
    order = first + torch.randperm(total, generator=g, device=DEV)
    table = torch.full((len(need), width), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, total


def _compact_inputs(c, g):
    b, page = c["batch"], c["page"]
    new = _sizes(c, b, c["new_lo"], c["new_hi"], 2)
    past = _sizes(c, b, c["past_lo"], c["past_hi"], 3)
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    t = dict(new=new, past=past, rows=sum(new), start=_starts(new), past_t=_int(past))
    t["table"], t["pages"] = _table(g, need, max(need))
    if c["evict"]:  # the copy's own pages
        t["first"] = t["table"]
        t["table"] = torch.where(t["first"] < 0, -1, t["first"] + t["pages"])
        t["from"] = torch.arange(t["pages"], device=DEV, dtype=torch.int32)
        t["to"] = t["from"] + t["pages"]
        t["pages"] *= 2
    rng = random.Random(sum(new) * 7 + b)
    kept, count = [], []
    for n in new:
        keep = [0] + [i for i in range(1, n) if rng.random() < c["keep"]]
        kept += keep + [-1] * (n - len(keep))
        count.append(len(keep))
    t["kept"], t["count"], t["counts"] = _int(kept), _int(count), count
    t["k"], t["v"] = _keys(g, t["rows"], c)
    return t


def _fork_inputs(c, g):
    page, n = c["page"], c["new"]
    past = _sizes(c, c["parents"], c["past_lo"], c["past_hi"], 4)
    rng = random.Random(c["parents"] * 131 + c["children"])
    parent = [rng.randrange(c["parents"]) for _ in range(c["children"])]
    need = [-(-p // page) for p in past]
    # Pages that the children will ask for, and the share of them that is free.
    ask = sum(-(-(past[p] + n) // page) - past[p] // page for p in parent)
    t = dict(past=past, parent=_int(parent), past_t=_int(past), grown=[past[p] for p in parent])
    t["table"], held = _table(g, need, max(need))
    t["pages"] = held + max(1, int(ask * c["spare"]))
    # (The first pages are not all held: free ones lie between.)
    move = torch.randperm(t["pages"], generator=g, device=DEV).to(torch.int32)
    t["table"] = torch.where(t["table"] < 0, -1, move[t["table"].clamp(min=0).long()])
    t["width"] = -(-(max(past) + n) // page)
    refs = torch.zeros(t["pages"] + 1, device=DEV, dtype=torch.int32)
    refs[torch.where(t["table"] < 0, t["pages"], t["table"]).long().flatten()] = 1
    t["refs0"] = refs[:-1].contiguous()
    t["start"] = _starts([n] * c["children"])
    t["k"], t["v"] = _keys(g, sum(past), c)
    # The positions whose pages are copied when written: each child's last page.
    tail = [p % page for p in t["grown"]]
    t["tail"], t["tail_start"], t["tail_past"] = tail, _starts(tail), _int([p - q for p, q in zip(t["grown"], tail)])
    return t


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if c["op"] == "copy":
        n = c["pages"]
        order = torch.randperm(2 * n, generator=g, device=DEV).to(torch.int32)
        k, v = _keys(g, n * c["page"], c)
        return {"pages": 2 * n, "from": order[:n].contiguous(), "to": order[n:].contiguous(), "k": k, "v": v,
                "rows": n * c["page"], "start": _int([0, n * c["page"]]), "past_t": _int([0])}
    return dict(verify=_verify_inputs, adapt=_adapt_inputs, compact=_compact_inputs,
                fork=_fork_inputs)[c["op"]](c, g)


# ------------------------------------------------------------- plain forms


def _plain_verify(c, t):
    """All rows' distributions in 64 bits (borders of a cumulated vocabulary lie closer than
    32 bits tell apart), the rows in order, the last token of each sequence."""
    b, rows, vocab = c["batch"], t["rows"], c["vocab"]
    start, n = t["start"][:-1].long(), torch.tensor(t["new"], device=DEV)
    warm = torch.where(t["temp"] > 0, t["temp"], 1.0).double()

    def likely(x):
        e = torch.exp((x.double() - x.amax(1, keepdim=True).double()) / warm[t["seq"]][:, None])
        return e / e.sum(1, keepdim=True)

    p = likely(t["target"])
    q = likely(t["draft"]) if c["draft"] else None
    best = t["target"].argmax(1)
    greedy = t["temp"] <= 0
    at = torch.arange(b, device=DEV)
    cur = torch.zeros(b, device=DEV, dtype=torch.long)
    left = torch.ones(b, device=DEV, dtype=torch.float64)  # what rejected tokens leave of p
    kept = torch.full((rows + 1,), -1, device=DEV, dtype=torch.long)  # (the last: of rows that none has)
    out = kept.clone()
    count = torch.where(n > 0, 1, 0)
    kept[torch.where(n > 0, start, rows)] = 0
    gone = torch.zeros(b, c["new_hi"], device=DEV, dtype=torch.bool)  # rejected at cur
    for i in range(1, c["new_hi"]):
        row = (start + i).clamp(max=rows - 1)
        node = (start + cur).clamp(max=rows - 1)
        up = t["parent"][row].long() if c["tree"] else torch.full_like(cur, i - 1)
        here = (i < n) & (up == cur)
        x = t["tokens"][row].long()
        px = p[node, x]
        earlier = t["tokens"][(start[:, None] + torch.arange(c["new_hi"], device=DEV)).clamp(max=rows - 1)].long()
        px = torch.where((gone & (earlier == x[:, None])).any(1), 0.0, px)
        u = t["uniform"][row].double()
        took = u * q[node, x] < px if c["draft"] else u * left < px
        took = torch.where(greedy, best[node] == x, took & (px > 0)) & here
        left = torch.where(took, 1.0, torch.where(here, left - px, left))
        gone = torch.where(took[:, None], False, gone)
        gone[:, i] |= here & ~took
        cur = torch.where(took, i, cur)
        out[torch.where(took, start + count - 1, rows)] = x
        kept[torch.where(took, start + count, rows)] = i
        count = count + took
    node = (start + cur).clamp(max=rows - 1)
    w = p[node]
    if c["draft"]:
        rest = torch.clamp(w - q[node], min=0.0)
        w = torch.where((gone.any(1) & (rest.sum(1) > 2.0**-40))[:, None], rest, w)
    else:
        for i in range(1, c["new_hi"]):
            x = t["tokens"][(start + i).clamp(max=rows - 1)].long()
            w[at, x] = torch.where(gone[:, i], 0.0, w[at, x])
    total = w.cumsum(1)
    u = t["uniform"][start.clamp(max=rows - 1)].double()
    last = (total <= (u * total[:, -1])[:, None]).sum(1).clamp(max=vocab - 1)
    last = torch.where(greedy, best[node], last)
    out[torch.where(n > 0, start + count - 1, rows)] = last
    return out[:-1].to(torch.int32), kept[:-1].to(torch.int32), count.to(torch.int32)


def _plain_adapt(c, t):
    order = torch.argsort(t["slot"], stable=True)
    x = t["x"][order]
    out = []
    for i in range(len(_ints(c["ns"]))):
        y = t["base"][i][order]
        at = t["host_slot"].count(-1)
        for s in range(c["slots"]):
            n = t["host_slot"].count(s)
            if n:
                low = torch.matmul(x[at:at + n], t["a"][i][s].float().T)
                y[at:at + n] += t["scale"][s] * torch.matmul(low, t["b"][i][s].float().T)
            at += n
        z = torch.empty_like(y)
        z[order] = y
        out.append(z)
    return tuple(out)


def _quantise(x, fmt):
    """Codes (a byte each), scale and (int4) middle of each vector along the last dimension."""
    if fmt == "int4":
        hi, lo = x.amax(-1, keepdim=True).double(), x.amin(-1, keepdim=True).double()
        mid, h = ((hi + lo) / 2).float(), ((hi - lo) / 30).float()
        u = (x.double() - mid.double()) / torch.where(h > 0, h, 1.0).double()
        return [((u + 15) / 2).round().clamp(0, 15).to(torch.uint8), h, mid]
    scale = (x.abs().amax(-1, keepdim=True).double() / (127 if fmt == "int8" else 448)).float()
    u = x.double() / torch.where(scale > 0, scale, 1.0).double()
    if fmt == "int8":
        return [u.round().clamp(-127, 127).to(torch.int8).view(torch.uint8), scale]
    step = torch.ldexp(torch.ones_like(u), (torch.frexp(u)[1] - 1).clamp(min=-6) - 3)
    u = ((u / step).round() * step).clamp(-448, 448).float()
    return [u.to(torch.float8_e4m3fn).view(torch.uint8), scale]


def _values(parts, fmt):
    """What codes stand for."""
    code, scale = parts[:2]
    if fmt == "int4":
        return parts[2] + (2 * code.float() - 15) * scale
    return code.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float() * scale


def _slots(c, table, seq, pos):
    return table[seq, pos // c["page"]].long() * c["page"] + pos % c["page"]


def _packed(new, past):
    """Sequence and position of each row."""
    n = torch.tensor(new, device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), n)
    first = torch.repeat_interleave(n.cumsum(0) - n, n)
    return seq, torch.arange(sum(new), device=DEV) - first + past.long()[seq]


def _plain_read(s, table, new, past):
    seq, pos = _packed(new, past)
    slot = _slots(s["c"], table, seq, pos)
    return tuple(_values([x[slot] for x in cache], s["c"]["fmt"]) for cache in s["cache"])


def _plain_copy(s):
    for cache in s["cache"]:
        for x in cache:
            x = x.view((-1, s["c"]["page"]) + x.shape[1:])
            x[s["t"]["to"].long()] = x[s["t"]["from"].long()]


def _plain_compact(s):
    c, t = s["c"], s["t"]
    seq, pos = _packed(t["new"], t["past_t"])
    if c["evict"]:
        _plain_copy(s)
    else:
        slot = _slots(c, t["table"], seq, pos)
        for cache, rows in zip(s["cache"], (t["k"], t["v"])):
            for x, y in zip(cache, _quantise(rows, c["fmt"])):
                x[slot] = y
    i = pos - t["past_t"].long()[seq]
    stays = i < t["count"].long()[seq]
    source = torch.where(stays, t["kept"].long(), i) + t["past_t"].long()[seq]
    a, b = _slots(c, t["table"], seq, source), _slots(c, t["table"], seq, pos)
    for cache in s["cache"]:
        for x in cache:
            x[b] = x[a]
    return (t["past_t"] + t["count"],) + _plain_read(s, t["table"], t["counts"], t["past_t"])


def _plain_fork(s):
    c, t = s["c"], s["t"]
    page, n, kids = c["page"], c["new"], c["children"]
    s["refs"].copy_(t["refs0"])
    refs = s["refs"]

    def count(table, held, by):
        refs.index_add_(0, table.clamp(min=0).long().flatten(), torch.where(held, by, 0).to(torch.int32).flatten())

    # The children hold their parents' pages, the parents none.
    parent = t["parent"].long()
    past = t["past_t"][parent]
    col = torch.arange(t["width"], device=DEV)
    table = torch.full((kids, t["width"]), -1, device=DEV, dtype=torch.int32)
    width = min(t["width"], t["table"].shape[1])
    table[:, :width] = t["table"][parent][:, :width]
    table = torch.where(col < ((past + page - 1) // page)[:, None], table, -1)
    count(t["table"], t["table"] >= 0, -1)
    count(table, table >= 0, 1)
    # Pages for the new positions, and own ones where a shared last page is written.
    have, want = (past + page - 1) // page, (past + n + page - 1) // page
    at = torch.arange(kids, device=DEV)
    last = table[at, (past // page).clamp(max=t["width"] - 1).long()].long()
    writes = past % page != 0
    same = (last[:, None] == last[None]) & writes[:, None] & writes[None]
    copy = writes & (same.tril(-1).sum(1) + 1 < refs[last.clamp(min=0)])
    need = copy + want - have
    end = need.cumsum(0)
    free = torch.argsort((refs != 0).to(torch.int32), stable=True)
    # (One that needs no page waits for those before it to leave a page that they share.)
    alone = ~writes | (refs[last.clamp(min=0)] <= 1)
    given = ((need == 0) & alone) | (end <= (refs == 0).sum())
    first = end - need
    at_copy = free[first.clamp(max=t["pages"] - 1)]
    copy = copy & given
    fresh = free[(first[:, None] + copy[:, None] + col - have[:, None]).clamp(0, t["pages"] - 1)]
    new = given[:, None] & (col >= have[:, None]) & (col < want[:, None])
    table = torch.where(new, fresh.to(torch.int32), table)
    table = torch.where(copy[:, None] & (col == (past // page)[:, None]), at_copy[:, None].to(torch.int32), table)
    count(fresh, new, 1)
    count(at_copy, copy, 1)
    count(last, copy, -1)
    source = torch.where(copy, last, t["pages"])  # (the last: a page that none has)
    target = torch.where(copy, at_copy, t["pages"])
    for cache in s["cache"]:
        for x in cache:
            x = x.view((-1, page) + x.shape[1:])
            x[target] = x[source]
    return (past, table, refs, given.to(torch.int32)) + _plain_read(s, table, t["tail"], t["tail_past"])


def _plain(s):
    c, t = s["c"], s["t"]
    if c["op"] == "verify":
        return _plain_verify(c, t)
    if c["op"] == "adapt":
        return _plain_adapt(c, t)
    if c["op"] == "compact":
        return _plain_compact(s)
    if c["op"] == "fork":
        return _plain_fork(s)
    _plain_copy(s)
    return _plain_read(s, t["to"][None], [t["rows"]], t["past_t"])


def _plain_prepare(s):
    """The cache as earlier steps left it, one page more behind it."""
    c, t = s["c"], s["t"]
    if c["op"] in ("verify", "adapt"):
        return s
    n = (t["pages"] + 1) * c["page"]
    s["cache"] = []
    for rows in (t["k"], t["v"]):
        parts = _quantise(rows, c["fmt"])
        s["cache"].append([torch.zeros((n,) + x.shape[1:], device=DEV, dtype=x.dtype) for x in parts])
        if c["op"] == "compact" and not c["evict"]:
            continue
        table, new = _written(c, t)
        seq, pos = _packed(new, torch.zeros(len(new), device=DEV, dtype=torch.int32))
        slot = _slots(c, table, seq, pos)
        for x, y in zip(s["cache"][-1], parts):
            x[slot] = y
    if c["op"] == "fork":
        s["refs"] = t["refs0"].clone()
    return s


def _written(c, t):
    """Where the rows of k and v lie before the call: pages, and lengths of the sequences."""
    if c["op"] == "copy":
        return t["from"][None], [t["rows"]]
    return (t["first"], t["new"]) if c["op"] == "compact" else (t["table"], t["past"])


# -------------------------------------------------------- the library's calls


def _ops():
    from onnx_runtime_dart_amd import ops
    return ops


def _context():
    """The thread's library context, on torch's stream."""
    ctx = _ops().default_context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return ctx


def _batch(table, start, past, batch, rows, max_new, max_len):
    """The library's description of a batch of sequences (device arrays by address)."""
    return _ops().SeqBatch(batch=batch, rows=rows, max_new=max_new, max_len=max_len,
                           row_start_ptr=start.data_ptr(), past_ptr=past.data_ptr(),
                           page_table_ptr=table.data_ptr(), table_stride=table.shape[1])


def _own_prepare(s):
    ops = _ops()
    c, t = s["c"], s["t"]
    s["ctx"] = _context()
    if c["op"] == "verify":
        s["out"], s["kept"] = (torch.empty(t["rows"], device=DEV, dtype=torch.int32) for _ in range(2))
        s["count"] = torch.empty(c["batch"], device=DEV, dtype=torch.int32)
        s["drafts"] = ops.Drafts(
            batch=c["batch"], rows=t["rows"], max_new=c["new_hi"], vocab=c["vocab"],
            row_start_ptr=t["start"].data_ptr(), tokens_ptr=t["tokens"].data_ptr(),
            parent_ptr=t["parent"].data_ptr() if c["tree"] else 0, target_ptr=t["target"].data_ptr(),
            draft_ptr=t["draft"].data_ptr() if c["draft"] else 0, temperature_ptr=t["temp"].data_ptr(),
            uniform_ptr=t["uniform"].data_ptr())
        return s
    if c["op"] == "adapt":
        s["y"] = [torch.empty_like(x) for x in t["base"]]
        s["adapters"] = ops.Adapters(c["k"], _ints(c["ns"]), slots=c["slots"], max_rank=c["rank"], fmt=c["fmt"],
                                     ctx=s["ctx"])
        for i in range(c["slots"]):
            a, b = ([x[i].float() for x in t[name]] for name in ("a", "b"))
            s["adapters"].set_dev(i, c["rank"], [x.data_ptr() for x in a], [x.data_ptr() for x in b],
                                  scale=t["scale"][i])
        torch.cuda.synchronize()
        return s
    s["cache"] = ops.KvCache(t["pages"], kv_heads=c["kv_heads"], head_size=c["d"], page_size=c["page"],
                             fmt=c["fmt"], ctx=s["ctx"])
    if c["op"] != "compact" or c["evict"]:
        # What earlier steps left in the cache.
        table, new = _written(c, t)
        start, none = _starts(new), _int([0] * len(new))
        s["cache"].append_dev(_batch(table, start, none, len(new), sum(new), max(new), max(new)),
                              t["k"].data_ptr(), t["v"].data_ptr())
        torch.cuda.synchronize()
    if c["op"] == "copy":
        s["read"] = _batch(t["to"][None], t["start"], t["past_t"], 1, t["rows"], t["rows"], t["rows"])
        rows = t["rows"]
    elif c["op"] == "compact":
        longest = c["new_hi"] + c["past_hi"]
        s["batch"] = _batch(t["table"], t["start"], t["past_t"], c["batch"], t["rows"], c["new_hi"], longest)
        rows = sum(t["counts"])
        s["read_start"] = _starts(t["counts"])
        s["read"] = _batch(t["table"], s["read_start"], t["past_t"], c["batch"], rows, max(t["counts"]), longest)
        s["past"] = torch.empty_like(t["past_t"])
    else:
        kids, longest = c["children"], c["past_hi"] + c["new"]
        s["refs"] = t["refs0"].clone()
        s["past"], s["given"] = (torch.empty(kids, device=DEV, dtype=torch.int32) for _ in range(2))
        s["table"] = torch.empty(kids, t["width"], device=DEV, dtype=torch.int32)
        s["before"] = _batch(t["table"], t["start"], t["past_t"], c["parents"], 0, 0, c["past_hi"])
        s["batch"] = _batch(s["table"], t["start"], s["past"], kids, kids * c["new"], c["new"], longest)
        rows = sum(t["tail"])
        s["read"] = _batch(s["table"], t["tail_start"], t["tail_past"], kids, rows, max(t["tail"]), longest)
    s["k"], s["v"] = (torch.zeros(rows, c["kv_heads"], c["d"], device=DEV) for _ in range(2))
    return s


def _own_run(s):
    ops = _ops()
    c, t = s["c"], s["t"]
    if c["op"] == "verify":
        ops.verify_drafts_dev(s["drafts"], s["out"].data_ptr(), s["kept"].data_ptr(), s["count"].data_ptr(),
                              ctx=s["ctx"])
        return s["out"], s["kept"], s["count"]
    if c["op"] == "adapt":
        s["adapters"].apply_dev(t["x"].data_ptr(), t["rows"], t["slot"].data_ptr(),
                                [x.data_ptr() for x in t["base"]], [y.data_ptr() for y in s["y"]])
        return tuple(s["y"])
    cache = s["cache"]
    if c["op"] == "copy" or c["op"] == "compact" and c["evict"]:
        cache.copy_pages_dev(t["from"].data_ptr(), t["to"].data_ptr(), t["from"].numel())
    head = ()
    if c["op"] == "compact":
        if not c["evict"]:
            cache.append_dev(s["batch"], t["k"].data_ptr(), t["v"].data_ptr())
        cache.compact_dev(s["batch"], t["kept"].data_ptr(), t["count"].data_ptr(), past_out_ptr=s["past"].data_ptr())
        head = (s["past"],)
    if c["op"] == "fork":
        s["refs"].copy_(t["refs0"])
        cache.fork_dev(s["before"], t["parent"].data_ptr(), c["children"], s["past"].data_ptr(),
                       s["table"].data_ptr(), t["width"], s["refs"].data_ptr())
        cache.fit_dev(s["batch"], s["refs"].data_ptr(), s["given"].data_ptr())
        head = (s["past"], s["table"], s["refs"], s["given"])
    cache.read_dev(s["read"], s["k"].data_ptr(), s["v"].data_ptr())
    return head + (s["k"], s["v"])


def prepare(case, seed):
    t = _inputs(case, seed)
    s = dict(c=case, t=t)
    return _own_prepare(s) if own else _plain_prepare(s)


def run(state):
    return _own_run(state) if own else _plain(state)


# ------------------------------------------------------ bytes and operations


def work(case):
    c = case
    if c["op"] == "verify":
        rows = sum(_sizes(c, c["batch"], c["new_lo"], c["new_hi"], 1))
        n = (rows + (rows - c["batch"] if c["draft"] else 0)) * c["vocab"]
        return dict(bytes=4 * n + 20 * rows, flops=4 * n)
    if c["op"] == "adapt":
        rows = sum(_ints(c["prompts"])) + c["tokens"]
        el, out = (2 if c["fmt"] == "f16" else 4), sum(_ints(c["ns"]))
        used = min(c["slots"], len(_ints(c["prompts"])) + c["tokens"])
        one = c["rank"] * (c["k"] * len(_ints(c["ns"])) + out)
        return dict(bytes=4 * rows * (c["k"] + 2 * out) + used * one * el, flops=2 * rows * one)
    token = 2 * c["kv_heads"] * (c["d"] * (4 if c["fmt"] == "int4" else 8) // 8 + (8 if c["fmt"] == "int4" else 4))
    vector = 2 * c["kv_heads"] * c["d"] * 4
    if c["op"] == "copy":
        n = c["pages"] * c["page"]
        return dict(bytes=n * (3 * token + vector), flops=n * 2 * c["kv_heads"] * c["d"])
    if c["op"] == "compact":
        n = sum(_sizes(c, c["batch"], c["new_lo"], c["new_hi"], 2))
        kept = int(n * c["keep"]) + c["batch"]
        write = n * 2 * token if c["evict"] else n * (vector + token)
        return dict(bytes=write + kept * (3 * token + vector), flops=n * 2 * c["kv_heads"] * c["d"])
    past = sum(_sizes(c, c["parents"], c["past_lo"], c["past_hi"], 4)) // c["parents"]
    tail = c["children"] * c["page"] // 2
    pages = (c["parents"] + c["children"]) * past // c["page"]
    return dict(bytes=tail * (3 * token + vector) + 12 * pages, flops=tail * 2 * c["kv_heads"] * c["d"])


# ------------------------------------------------------- results in 64 bits


def _exact_cached(x, fmt):
    """What a cache of this format gives back for the vectors x (64 bits, of fp32 values)."""
    x = x.double()
    if fmt == "int4":
        top, low = x.max(-1, keepdim=True)[0], x.min(-1, keepdim=True)[0]
        m, h = ((top + low) * 0.5).float().double(), ((top - low) / 30.0).float().double()
        half = torch.where(h > 0, (x - m) / h, 0.0) * 0.5 + 7.5
        n = torch.floor(half + 0.5)
        # (Halves go to the even code.)
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
    if c["op"] == "verify":
        return None  # (whole numbers)
    t = _inputs(c, seed)
    if c["op"] == "adapt":
        out = []
        slot = t["slot"].long()
        for i, n in enumerate(_ints(c["ns"])):
            y = t["base"][i].double()
            for s in sorted(set(t["host_slot"]) - {-1}):
                rows = torch.nonzero(slot == s)[:, 0]
                whole = t["b"][i][s].double() @ t["a"][i][s].double()
                y[rows] += t["scale"][s] * (t["x"][rows].double() @ whole.T.contiguous())
            out.append(y)
        return tuple(out)
    rows, at = [], 0
    if c["op"] == "compact":
        kept = t["kept"].tolist()
        for n, m in zip(t["new"], t["counts"]):
            rows += [at + j for j in kept[at:at + m]]
            at += n
        head = (None,)
    elif c["op"] == "fork":
        first = [sum(t["past"][:i]) for i in range(c["parents"])]
        for p in t["parent"].tolist():
            rows += range(first[p] + t["past"][p] - t["past"][p] % c["page"], first[p] + t["past"][p])
        head = (None,) * 4
    else:
        rows, head = range(t["rows"]), ()
    at = torch.tensor(list(rows), device=DEV, dtype=torch.long)
    return head + tuple(_exact_cached(x[at], c["fmt"]) for x in (t["k"], t["v"]))
