"""The serving operators together, as a program runs them: prompts and drafted trees written
to the paged cache, attended to, verified, the rows that stay moved together, sequences forked and
fitted with pages, against a cache that only ever held what was emitted."""
import numpy as np
import pytest

import drafts_reference as R

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
