"""The serving operators together, as a program runs them: prompts and drafted trees written
to the paged cache, attended to, verified, the rows that stay moved together, sequences forked and
fitted with pages, against a cache that only ever held what was emitted."""
import ctypes as C

import numpy as np
import pytest

import drafts_reference as R
import kv_reference as K
from hip_graph import Captured

pytestmark = pytest.mark.gpu
KV, HEADS, D, PAGE, VOCAB, RANK = 2, 4, 64, 16, 300, 4


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


class Model:
    """One layer: token embeddings through q, k and v with each request's adapter, attention, logits."""

    def __init__(self, ops, rng):
        self.ops = ops
        self.emb, self.out = rng.standard_normal((VOCAB, D)), rng.standard_normal((HEADS * D, VOCAB)) * 0.3
        ns = [HEADS * D, KV * D, KV * D]
        self.w = [(rng.standard_normal((D, n)) / np.sqrt(D)).astype(np.float32) for n in ns]
        self.ad = ops.Adapters(D, ns, slots=3, max_rank=RANK)
        for s in range(3):
            self.ad.set(s, [rng.standard_normal((RANK, D)).astype(np.float32) / 8 for _ in ns],
                        [rng.standard_normal((n, RANK)).astype(np.float32) for n in ns], scale=0.5)
        self.cos, self.sin = ops.rotary_tables(512, D // 2, base=1e4)

    def qkv(self, tokens, slots):
        x = self.emb[tokens].astype(np.float32)
        y = self.ad.apply(x, slots, [x @ w for w in self.w])
        return [t.reshape(len(tokens), -1, D) for t in y]

    def step(self, cache, tokens, slots, where, tree=None, pos=None):
        """Writes the rows, attends; their logits, keys and values."""
        q, k, v = self.qkv(tokens, slots)
        rope = (self.cos, self.sin, False) if pos is None else (self.cos, self.sin, False, pos)
        cache.append(k, v, **where, rope=rope)
        y = cache.attend(q, **where, rope=rope, tree=tree)
        return (y.reshape(len(tokens), -1) @ self.out).astype(np.float32), k, v


def trees(rng, new):
    """Parents, ancestors' bits and depths of packed rows."""
    parent, bits, depth = [], [], []
    for n in new:
        b, d = [1], [0]
        parent.append(-1)
        for i in range(1, n):
            up = int(rng.integers(0, i))
            parent.append(up)
            b.append(b[up] | 1 << i)
            d.append(d[up] + 1)
        bits += b
        depth += d
    return np.array(parent), np.array(bits, np.uint64)[:, None], np.array(depth)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("tree", [True, False])
def test_speculative_decoding(ops, fmt, tree):
    rng = np.random.default_rng(1)
    m = Model(ops, rng)
    cache = ops.KvCache(120, kv_heads=KV, head_size=D, page_size=PAGE, fmt=fmt)
    pages, table, refs = 120, np.full((2, 10), -1, np.int32), np.zeros(120, np.int32)

    # Two prompts, then five answers of them.
    prompts = [rng.integers(0, VOCAB, n) for n in (37, 20)]
    start, past = np.array([0, 37, 57]), np.zeros(2, np.int32)
    table, refs, granted = cache.fit(row_start=start, past=past, page_table=table, refs=refs)
    assert granted.all()
    slots = np.repeat([0, 1], [37, 20])
    _, k, v = m.step(cache, np.concatenate(prompts), slots, dict(row_start=start, past=past, page_table=table))
    parents = [0, 0, 1, 0, 1]
    past, table, refs = cache.fork(parents, past=[37, 20], page_table=table, refs=refs)
    assert refs.max() == 3
    slot = np.array([0, 1, -1, 0, 1])  # (answers may differ in their adapters: earlier keys stay)
    told = [[int(rng.integers(0, VOCAB))] for _ in parents]  # the last emitted token, not yet cached
    seen = [list(prompts[p]) for p in parents]
    keys, values = ([list(t[start[p]:start[p + 1]]) for p in parents] for t in (k, v))
    for step in range(6):
        new = rng.integers(1, 20, 5)
        start = np.r_[0, np.cumsum(new)]
        table, refs, granted = cache.fit(row_start=start, past=past, page_table=table, refs=refs)
        assert granted.all()
        up, bits, depth = trees(rng, new) if tree else (None, None, np.concatenate([np.arange(n) for n in new]))
        tokens = rng.integers(0, VOCAB, start[-1])
        tokens[start[:-1]] = [t[-1] for t in told]
        where = dict(row_start=start, past=past, page_table=table)
        rows = np.repeat(slot, new)
        pos = np.repeat(past, new) + depth
        logits, k, v = m.step(cache, tokens, rows, where, bits, pos)
        uniform = (rng.random(start[-1]) * 0.02).astype(np.float32)  # (small ones, so that drafts stay)
        temp = np.array([1, 0, 1.5, 3, 1], np.float32)
        args = dict(parent=up, temperature=temp)
        got = ops.op_verify_drafts(logits, tokens, uniform, start, **args)
        for g, w in zip(got, R.verify(logits, tokens, uniform, start, **args)):
            np.testing.assert_array_equal(g, w)
        out, kept, count = got
        past = cache.compact(kept, count, **where)
        for b in range(5):
            s, c = start[b], count[b]
            assert kept[s] == 0 and out[s + c - 1] >= 0
            seen[b] += [told[b][-1]] + list(out[s:s + c - 1])
            told[b] += list(out[s:s + c])
            keys[b] += list(k[s + kept[s:s + c]])
            values[b] += list(v[s + kept[s:s + c]])
        np.testing.assert_array_equal(past, [len(t) for t in seen])
    assert not cache.refused()
    held, n = np.unique(table[table >= 0], return_counts=True)
    np.testing.assert_array_equal(refs[held], n)

    # What the cache holds is, bit for bit, what a cache of each answer alone holds.
    start = np.r_[0, np.cumsum(past)]
    got = cache.read(start[-1], row_start=start, past=np.zeros(5, np.int32), page_table=table)
    alone = ops.KvCache(200, kv_heads=KV, head_size=D, page_size=PAGE, fmt=fmt)
    own = np.arange(5 * 12).reshape(5, 12)
    pos = np.concatenate([np.arange(n) for n in past])
    where = dict(row_start=start, past=np.zeros(5, np.int32), page_table=own)
    alone.append(*(np.concatenate(t) for t in (keys, values)), **where, rope=(m.cos, m.sin, False, pos))
    for g, w in zip(got, alone.read(start[-1], **where)):
        np.testing.assert_array_equal(g, w)

    # The best two answers go on; in the end nothing is held.
    past, table, refs = cache.fork([3, 2, 3], past=past, page_table=table, refs=refs)
    assert (refs > 0).sum() == sum(-(-int(past[i]) // PAGE) for i in (0, 1))
    table, refs, granted = cache.fit(row_start=[0, 0, 0, 0], past=[0, 0, 0], page_table=table, refs=refs)
    assert (refs == 0).all() and (table == -1).all() and granted.all()


def test_captured_steps_leave_out_whom_fit_does_not_serve(ops):
    # A and B share their last page, C holds all others.  The step's calls get past -1 for those that are not
    # granted: nothing of theirs is written, so the page they share stays as it is.
    rng = np.random.default_rng(32)
    with Captured(ops) as g:
        cache = ops.KvCache(3, kv_heads=1, head_size=D, page_size=PAGE, fmt="int8", ctx=g.ctx)
        whole = dict(row_start=PAGE * np.arange(4), past=np.zeros(3), page_table=np.arange(3)[:, None])
        k, v = rng.standard_normal((2, 3 * PAGE, 1, D)).astype(np.float32)
        cache.append(k, v, **whole)
        held = [x.reshape(3, PAGE, 1, D) for x in cache.read(3 * PAGE, **whole)]
        table = np.array([[0, -1], [0, -1], [1, 2]], np.int32)
        refs, past = np.array([2, 1, 1], np.int32), np.array([5, 5, 20], np.int32)
        start, kept, count = np.array([0, 2, 4, 6]), np.array([1, -1, 0, 1, 1, -1]), np.array([1, 2, 1])
        d = {name: g.buffer(np.ascontiguousarray(a, np.int32)) for name, a in dict(
            start=start, past=past, step=past, table=table, refs=refs, granted=np.zeros(3), kept=kept,
            count=count).items()}
        f = {name: g.buffer(np.zeros((6, 1, D), np.float32)) for name in ("k", "v", "q", "y")}

        def batch(lengths):
            return ops.SeqBatch(batch=3, rows=6, max_new=2, max_len=2 * PAGE, row_start_ptr=d["start"].ptr,
                                past_ptr=d[lengths].ptr, page_table_ptr=d["table"].ptr, table_stride=2)

        def fit():
            cache.fit_dev(batch("past"), d["refs"].ptr, d["granted"].ptr)

        def step():
            cache.append_dev(batch("step"), f["k"].ptr, f["v"].ptr)
            cache.attend_dev(batch("step"), f["q"].ptr, f["y"].ptr, 1)
            cache.compact_dev(batch("step"), d["kept"].ptr, d["count"].ptr, past_out_ptr=d["step"].ptr)

        fit()
        g.put(d["step"], np.full(3, -1, np.int32))
        step()  # (workspaces, nobody's rows)
        assert cache.refused()
        fit, step = g.capture(fit), g.capture(step)
        for served in ([0, 0, 1], [0, 0, 1], [1, 1, 1], [1, 1, 1]):
            rows = {name: rng.standard_normal((6, 1, D)).astype(np.float32) for name in ("k", "v", "q")}
            for name, x in rows.items():
                g.put(f[name], x)
            g.put(f["y"], np.full((6, 1, D), 77, np.float32))
            fit()
            g.wait()
            granted, table = (d[n].to_array(sh, np.int32) for n, sh in (("granted", (3,)), ("table", (3, 2))))
            np.testing.assert_array_equal(granted, served)
            g.put(d["step"], np.where(granted, past, -1).astype(np.int32))
            step()
            g.wait()
            np.testing.assert_array_equal(d["step"].to_array((3,), np.int32), np.where(granted, past + count, -1))
            y = f["y"].to_array((6, D), np.float32)
            assert ((y == 77).all(1) == np.repeat(1 - granted, 2)).all()
            if served[0] and past[0] == 5:  # A has a copy now
                for x in held:
                    x[table[0, 0]] = x[0]
            now = [x.reshape(3, PAGE, 1, D) for x in cache.read(3 * PAGE, **whole)]
            mine = np.zeros((3, PAGE), bool)  # places that may change
            for b in np.nonzero(granted)[0]:
                for p in range(past[b], past[b] + 2):
                    mine[table[b, p // PAGE], p % PAGE] = True
                for j, i in enumerate(kept[2 * b:2 * b + count[b]]):
                    at = table[b, (past[b] + j) // PAGE], (past[b] + j) % PAGE
                    for x, new in zip(now, (rows["k"], rows["v"])):
                        np.testing.assert_array_equal(x[at], K.cached(new[2 * b + i][None], "int8")[0])
            for x, was in zip(now, held):
                np.testing.assert_array_equal(x[~mine], was[~mine])
            held = now
            assert cache.refused() == (not granted.all())
            past = np.where(granted, past + count, past).astype(np.int32)
            if served == [0, 0, 1] and past[2] == 22:
                past[2] = 10  # C gives its second page back
            g.put(d["past"], past)
        cache.release()


def test_contexts_at_once(ops):
    # Two contexts with streams of their own use the same adapters and cache; nothing of one call waits
    # for the other's.
    rng = np.random.default_rng(31)
    ad = ops.Adapters(200, [300], slots=4, max_rank=8)
    for s in range(4):
        ad.set(s, *([rng.standard_normal(sh).astype(np.float32)] for sh in ((8, 200), (300, 8))))
    rows, seqs, n = 1200, 12, 6
    x, base = (rng.standard_normal((rows, k)).astype(np.float32) for k in (200, 300))
    slot = rng.integers(-1, 4, rows).astype(np.int32)
    want = ad.apply(x, slot, [base])[0]
    logits = rng.standard_normal((seqs * n, 4000)).astype(np.float32)
    start, tokens = np.arange(0, seqs * n + 1, n), rng.integers(0, 4000, seqs * n)
    uniform = rng.random(seqs * n).astype(np.float32)
    drawn = R.verify(target=logits, tokens=tokens, uniform=uniform, row_start=start, parent=None, draft=None)
    cache = ops.KvCache(8, kv_heads=2, head_size=64, page_size=64, fmt="int8")
    k, v = rng.standard_normal((2, 512, 2, 64)).astype(np.float32)
    where = dict(row_start=64 * np.arange(9), past=np.zeros(8), page_table=np.arange(8)[:, None])
    cache.append(k, v, **where)
    held = cache.read(512, **where)
    with Captured(ops) as one, Captured(ops) as two:
        sides = []
        for g, src, dst in ((one, [0, 1], [2, 3]), (two, [4, 5], [6, 7])):
            d = {name: g.buffer(a) for name, a in dict(
                x=x, base=base, slot=slot, y=np.zeros_like(base), logits=logits, start=start.astype(np.int32),
                tokens=tokens.astype(np.int32), uniform=uniform, out=np.zeros(seqs * n, np.int32),
                kept=np.zeros(seqs * n, np.int32), count=np.zeros(seqs, np.int32),
                src=np.array(src, np.int32), dst=np.array(dst, np.int32)).items()}
            # (The handles are the default context's: calls on others go by the C entries.)
            sides.append((g, d, ops.Drafts(
                batch=seqs, rows=seqs * n, max_new=n, vocab=4000, row_start_ptr=d["start"].ptr,
                tokens_ptr=d["tokens"].ptr, target_ptr=d["logits"].ptr, uniform_ptr=d["uniform"].ptr)))
        from onnx_runtime_dart_amd._lib import check, lib
        for _ in range(6):
            for g, d, drafts in sides:
                check(lib.mg_adapters_apply_f32_dev(g.ctx.handle, ad.handle, d["x"].ptr, rows, d["slot"].ptr,
                                                    (C.c_void_p * 1)(d["base"].ptr), (C.c_void_p * 1)(d["y"].ptr)))
                ops.verify_drafts_dev(drafts, d["out"].ptr, d["kept"].ptr, d["count"].ptr, ctx=g.ctx)
                check(lib.mg_kv_cache_copy_pages_dev(g.ctx.handle, cache.handle, d["src"].ptr, d["dst"].ptr, 2))
        for g, d, _ in sides:
            g.wait()
            np.testing.assert_array_equal(d["y"].to_array(want.shape, np.float32), want)
            for name, w in zip(("out", "kept", "count"), drawn):
                np.testing.assert_array_equal(d[name].to_array(w.shape, np.int32), w)
    for got, was in zip(cache.read(512, **where), held):
        pages = was.reshape((8, 64) + was.shape[1:]).copy()
        pages[[2, 3, 6, 7]] = pages[[0, 1, 4, 5]]
        np.testing.assert_array_equal(got.reshape(pages.shape), pages)
