"""The quantised KV cache against its formulas (bit for bit) and the attention over it
against 64 bits: formats, head and page sizes, ragged batches, trees of drafted tokens,
rows that see nothing, what lies in unseen places, bad pages, streams and captured graphs."""
import ctypes as C

import numpy as np
import pytest

import kv_reference as R
from onnx_runtime_dart_amd.errors import ArgumentError, UnsupportedError

pytestmark = pytest.mark.gpu

FMTS = ["int8", "e4m3", "int4"]


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def same(got, want):
    np.testing.assert_array_equal(got, want)


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def tables(rng, n, half):
    t = rng.uniform(0, 6, (n, half))
    return np.cos(t).astype(np.float32), np.sin(t).astype(np.float32)


# ------------------------------------------------------------ write and read


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d, kv, page", [(1, 1, 16), (3, 2, 16), (16, 5, 32), (64, 8, 64), (80, 4, 64),
                                         (96, 3, 128), (128, 8, 64), (130, 1, 16), (192, 2, 32),
                                         (201, 3, 256), (256, 4, 128)])
def test_round_trip(ops, fmt, d, kv, page):
    rng = np.random.default_rng(d)
    b = R.Batch(rng, [5, 1, 0, 38, 4], [0, 17, 3, 29, 4], page, extra_rows=2)
    k, v = normal(rng, b.rows, kv, d) * 3, normal(rng, b.rows, kv, d)
    cache = ops.KvCache(b.pages, kv_heads=kv, head_size=d, page_size=page, fmt=fmt)
    cache.append(k, v, **b.args())
    gk, gv = cache.read(b.rows, **b.args())
    same(gk[:-2], R.cached(k, fmt)[:-2])
    same(gv[:-2], R.cached(v, fmt)[:-2])
    assert not gk[-2:].any() and not gv[-2:].any()  # rows behind the last sequence
    assert not cache.refused()
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("inter", [False, True])
def test_keys_are_rotated_first(ops, fmt, inter):
    rng = np.random.default_rng(8)
    b = R.Batch(rng, [9, 30], [11, 0], 32)
    k, v = normal(rng, b.rows, 2, 96), normal(rng, b.rows, 2, 96)
    cos, sin = tables(rng, 60, 20)
    cache = ops.KvCache(b.pages, kv_heads=2, head_size=96, page_size=32, fmt=fmt)
    own = np.concatenate([11 + np.arange(9), np.arange(30)])
    given = rng.integers(0, 60, b.rows)
    given[4] = 60  # outside the tables: the key is NaN
    for pos, args in ((own, (cos, sin, inter)), (given, (cos, sin, inter, given))):
        cache.append(k, v, **b.args(), rope=args)
        gk, gv = cache.read(b.rows, **b.args())
        same(gk, R.cached(R.rotate(k, cos, sin, pos, inter), fmt))
        same(gv, R.cached(v, fmt))
    cache.release()


SPECIAL = {
    "zeros": lambda r, s: np.zeros(s), "constant": lambda r, s: np.full(s, -2.5),
    "integers": lambda r, s: r.integers(-15, 16, s), "halves": lambda r, s: r.integers(-60, 61, s) / 4,
    "tiny": lambda r, s: r.standard_normal(s) * 1e-39, "least": lambda r, s: r.integers(-3, 4, s) * 1.4e-45,
    "huge": lambda r, s: r.uniform(-3.4e38, 3.4e38, s), "steps": lambda r, s: r.integers(-448, 449, s) / 8,
    "one": lambda r, s: np.eye(s[-1])[r.integers(0, s[-1], s[:-1])] * 3,
    "minus zero": lambda r, s: np.where(r.random(s) < 0.5, -0.0, 1.0)}


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", SPECIAL)
def test_special_values(ops, fmt, kind):
    rng = np.random.default_rng(21)
    b = R.Batch(rng, [23], [2], 16)
    k, v = (np.asarray(SPECIAL[kind](rng, (23, 3, 64)), np.float32) for _ in range(2))
    cache = ops.KvCache(b.pages, kv_heads=3, head_size=64, page_size=16, fmt=fmt)
    cache.append(k, v, **b.args())
    gk, gv = cache.read(b.rows, **b.args())
    same(gk, R.cached(k, fmt))
    same(gv, R.cached(v, fmt))
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
def test_non_finite_vectors(ops, fmt):
    rng = np.random.default_rng(22)
    b = R.Batch(rng, [9], [0], 16)
    k, v = normal(rng, 9, 2, 80), normal(rng, 9, 2, 80)
    k[0, 0, 79], k[3, 1, 0], v[5, 0, 40], v[6, 1, 7] = np.nan, np.inf, -np.inf, np.nan
    cache = ops.KvCache(b.pages, kv_heads=2, head_size=80, page_size=16, fmt=fmt)
    cache.append(k, v, **b.args())
    gk, gv = cache.read(9, **b.args())
    same(gk, R.cached(k, fmt))
    same(gv, R.cached(v, fmt))
    assert np.isnan(gk[0, 0]).all() and np.isnan(gv[6, 1]).all() and np.isfinite(gk[0, 1]).all()
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("cuts", [[1] * 11, [2, 3, 1, 5], [5, 6], [4, 4, 3]], ids=str)
def test_appended_piece_by_piece(ops, fmt, cuts):
    # Tokens of one group of four arrive in different calls; none disturbs its neighbours.
    rng = np.random.default_rng(23)
    whole = R.Batch(rng, [11, 11], [6, 5], 16)
    k, v = normal(rng, 22, 2, 64), normal(rng, 22, 2, 64)
    cache = ops.KvCache(whole.pages, kv_heads=2, head_size=64, page_size=16, fmt=fmt)
    at = 0
    for n in cuts:
        rows = np.concatenate([np.arange(at, at + n), 11 + np.arange(at, at + n)])
        cache.append(k[rows], v[rows], row_start=[0, n, 2 * n], past=whole.past + at,
                     page_table=whole.page_table)
        at += n
    gk, gv = cache.read(22, **whole.args())
    same(gk, R.cached(k, fmt))
    same(gv, R.cached(v, fmt))
    cache.release()


def device(ops, *arrays):
    return [ops.DeviceBuffer.from_array(a) for a in arrays]


def seq_batch(ops, b, dev, max_new=None, max_len=None, rows=None):
    return ops.SeqBatch(batch=len(b.new), rows=b.rows if rows is None else rows,
                        max_new=max(b.new) if max_new is None else max_new,
                        max_len=int((b.past + b.new).max()) if max_len is None else max_len,
                        row_start_ptr=dev[0].ptr, past_ptr=dev[1].ptr, page_table_ptr=dev[2].ptr,
                        table_stride=b.page_table.shape[1])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d, pad, offset", [(64, 64, 0), (64, 1, 0), (128, 0, 1), (128, 4, 4), (70, 6, 2)])
def test_strided_rows(ops, fmt, d, pad, offset):
    # k and v inside fused rows, at addresses of 4, 8 and 16 bytes; read back into others.
    rng = np.random.default_rng(24)
    b = R.Batch(rng, [6, 9], [3, 0], 16)
    kv = 2
    row = 2 * kv * d + pad
    mem = normal(rng, offset + b.rows * row)
    fused = mem[offset:].reshape(b.rows, row)
    dev = device(ops, b.row_start, b.past, b.page_table, mem, np.full(mem.shape, 7, np.float32))
    cache = ops.KvCache(b.pages, kv_heads=kv, head_size=d, page_size=16, fmt=fmt)
    s = seq_batch(ops, b, dev)
    at = 4 * offset
    cache.append_dev(s, dev[3].ptr + at, dev[3].ptr + at + 4 * kv * d, k_stride=row, v_stride=row)
    cache.read_dev(s, dev[4].ptr + at, dev[4].ptr + at + 4 * kv * d, k_stride=row, v_stride=row)
    want = np.full(mem.shape, 7, np.float32)
    w = want[offset:].reshape(b.rows, row)
    w[:, :kv * d] = R.cached(fused[:, :kv * d].reshape(-1, kv, d), fmt).reshape(b.rows, -1)
    w[:, kv * d:2 * kv * d] = R.cached(fused[:, kv * d:2 * kv * d].reshape(-1, kv, d), fmt).reshape(
        b.rows, -1)
    same(dev[4].to_array(mem.shape, np.float32), want)
    for x in dev:
        x.free()
    cache.release()


def test_refused_sequences_and_pages(ops):
    # What the host rules refuse (shown for these arrays by kv_cache_slots first), the kernels
    # refuse too: nothing is written, rows stay as they were, and the cache remembers.
    rng = np.random.default_rng(25)
    row_start = np.array([0, 2, 5, 9, 12], np.int32)
    past = np.array([0, -3, 14, 0], np.int32)
    table = np.array([[3, 2], [1, 0], [9, 1], [-1, 5]], np.int32)
    slots, refused = ops.kv_cache_slots(row_start, past, table, rows=13, max_new=4, max_len=30,
                                        pages=6, page_size=16)
    want = np.full(13, -1)
    want[:2], want[7:9] = [48, 49], [16, 17]
    same(slots, want)
    assert refused
    k, v, q = normal(rng, 13, 1, 64), normal(rng, 13, 1, 64), normal(rng, 13, 2, 64)
    seven = np.full((13, 1, 64), 7, np.float32)
    dev = device(ops, row_start, past, table, k, v, seven, seven, q, np.full(q.shape, 7, np.float32))
    cache = ops.KvCache(6, kv_heads=1, head_size=64, page_size=16)
    s = ops.SeqBatch(batch=4, rows=13, max_new=4, max_len=30, row_start_ptr=dev[0].ptr,
                     past_ptr=dev[1].ptr, page_table_ptr=dev[2].ptr, table_stride=2)
    cache.append_dev(s, dev[3].ptr, dev[4].ptr)
    assert cache.refused() and not cache.refused()
    cache.read_dev(s, dev[5].ptr, dev[6].ptr)
    assert cache.refused()
    gk = dev[5].to_array(seven.shape, np.float32)
    same(gk[slots >= 0], R.cached(k, "int8")[slots >= 0])
    assert (gk[2:5] == 7).all() and (gk[12:] == 7).all()  # the refused sequence, no sequence
    assert np.isnan(gk[5:7]).all() and np.isnan(gk[9:12]).all()  # no such page
    cache.attend_dev(s, dev[7].ptr, dev[8].ptr, 2)
    assert cache.refused()
    y = dev[8].to_array(q.shape, np.float32)
    assert np.isfinite(y[:2]).all() and (y[2:5] == 7).all() and (y[12:] == 7).all()
    assert np.isnan(y[5:12]).all()
    # A whole cache read shows that nothing else was written.
    ck, cv = cache.read(96, row_start=[0, 96], past=[0], page_table=[[0, 1, 2, 3, 4, 5]])
    written = np.zeros(96, bool)
    written[slots[slots >= 0]] = True
    assert not ck[~written].any() and not cv[~written].any()
    assert not cache.refused()
    for x in dev:
        x.free()
    cache.release()


# --------------------------------------------------------------- attention


def filled(ops, rng, b, kv, d, fmt, scale=1.0, **kw):
    """A cache that holds all positions of the batch, and what it gives back for them."""
    n = [int(x) for x in b.past + b.new]
    k, v = normal(rng, sum(n), kv, d) * np.float32(scale), normal(rng, sum(n), kv, d)
    cache = ops.KvCache(b.pages, kv_heads=kv, head_size=d, page_size=b.page, fmt=fmt, **kw)
    cache.append(k, v, row_start=np.concatenate([[0], np.cumsum(n)]), past=np.zeros(len(n)),
                 page_table=b.page_table)
    cut = np.cumsum(n)[:-1]
    return cache, np.split(R.cached(k, fmt), cut), np.split(R.cached(v, fmt), cut)


def check_rows(y, q, b, ks, vs, scale, tree=None, tol=1.0):
    for i, (k, v) in enumerate(zip(ks, vs)):
        r = slice(b.row_start[i], b.row_start[i + 1])
        see = R.visible(b.new[i], int(b.past[i]), None if tree is None else tree[r])
        want = R.attend(q[r], k, v, see, scale)
        err = np.abs(y[r] - want).max(initial=0)
        assert err <= tol * R.bound(q[r], k, v, scale), (i, err, R.bound(q[r], k, v, scale))


# new, past, heads, kv heads, head size, page, format
CASES = [
    ([1], [0], 1, 1, 64, 16, "int8"), ([1, 1, 1], [1, 30, 31], 4, 2, 64, 16, "int8"),
    ([1], [32], 8, 1, 128, 32, "e4m3"), ([1, 1], [127, 128], 16, 1, 128, 64, "int4"),
    ([1, 0, 1], [129, 5, 0], 12, 4, 96, 16, "e4m3"), ([1], [1000], 7, 7, 80, 64, "int4"),
    ([1] * 9, [3, 700, 64, 63, 65, 1, 0, 2000, 255], 32, 8, 128, 64, "e4m3"),
    ([1, 1], [5000, 17], 4, 4, 256, 128, "int8"), ([1], [300], 6, 3, 192, 32, "int4"),
    ([1], [77], 3, 1, 1, 16, "int8"), ([1], [77], 32, 1, 201, 16, "e4m3"),
    ([2], [0], 8, 8, 64, 16, "int4"), ([17], [0], 1, 1, 64, 16, "int8"),
    ([5, 3], [40, 90], 12, 4, 128, 64, "e4m3"), ([33], [100], 2, 1, 128, 16, "int4"),
    ([64, 1, 20], [0, 64, 7], 8, 2, 64, 64, "int8"), ([65], [31], 7, 1, 96, 32, "e4m3"),
    ([130], [0], 4, 1, 128, 64, "int8"), ([200, 77], [13, 300], 8, 2, 128, 128, "int4"),
    ([90], [50], 4, 2, 256, 64, "e4m3"), ([100], [500], 4, 2, 192, 16, "int8"),
    ([40, 300], [3000, 0], 4, 1, 64, 256, "e4m3")]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_causal(ops, case):
    new, past, heads, kv, d, page, fmt = case
    rng = np.random.default_rng(sum(new) + sum(past) + d)
    b = R.Batch(rng, new, past, page, extra_rows=1)
    cache, ks, vs = filled(ops, rng, b, kv, d, fmt, 1.5)
    q = normal(rng, b.rows, heads, d)
    y = cache.attend(q, **b.args())
    check_rows(y, q, b, ks, vs, 1 / np.sqrt(d))
    assert not y[-1:].any()
    y2 = cache.attend(q, **b.args(), scale=0.37)
    check_rows(y2, q, b, ks, vs, np.float32(0.37))
    cache.release()


@pytest.mark.parametrize("max_bytes", [0, -1])
@pytest.mark.parametrize("fmt", FMTS)
def test_split_keys_and_no_workspace(ops, fmt, max_bytes):
    # Keys split over workgroups, and the same call without room for partial results.
    rng = np.random.default_rng(31)
    ctx = ops.Context()
    b = R.Batch(rng, [1, 1], [4097, 600], 64)
    cache, ks, vs = filled(ops, rng, b, 2, 128, fmt, ctx=ctx)
    q = normal(rng, b.rows, 8, 128)
    dev = device(ops, b.row_start, b.past, b.page_table, q, np.zeros_like(q))
    ctx.set_control(max_bytes=max_bytes)
    cache.attend_dev(seq_batch(ops, b, dev, max_len=9000), dev[3].ptr, dev[4].ptr, 8)
    y = (ctx.synchronize(), dev[4].to_array(q.shape, np.float32))[1]
    check_rows(y, q, b, ks, vs, 1 / np.sqrt(128))
    for x in dev:
        x.free()
    cache.release()
    ctx.close()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [40, 3]], ids=str)
def test_queries_are_rotated(ops, new, inter):
    rng = np.random.default_rng(32)
    b = R.Batch(rng, new, [70, 200], 32)
    cache, ks, vs = filled(ops, rng, b, 2, 96, "int8")
    q = normal(rng, b.rows, 4, 96)
    cos, sin = tables(rng, 300, 30)
    own = np.concatenate([p + np.arange(n) for n, p in zip(b.new, b.past)])
    given = rng.integers(0, 300, b.rows)
    for pos, args in ((own, (cos, sin, inter)), (given, (cos, sin, inter, given))):
        y = cache.attend(q, **b.args(), rope=args)
        check_rows(y, R.rotate(q, cos, sin, pos, inter), b, ks, vs, 1 / np.sqrt(96))
    given[1] = -1
    y = cache.attend(q, **b.args(), rope=(cos, sin, inter, given))
    assert np.isnan(y[1]).all() and np.isfinite(np.delete(y, 1, 0)).all()
    cache.release()


def tree_words(rng, n, words):
    """Random trees: each row's ancestors and itself; some rows see nothing drafted."""
    out = np.zeros((n, words), np.uint64)
    for i in range(n):
        p = rng.integers(-1, i) if i else -1
        if p >= 0:
            out[i] = out[p]
        out[i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return out


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new, past, heads, kv, d, words", [
    ([4], [0], 4, 4, 64, 1), ([25], [190], 8, 2, 128, 1), ([64, 10], [33, 0], 4, 1, 96, 1),
    ([7, 0, 16], [500, 9, 31], 16, 2, 64, 1), ([130, 5], [64, 127], 2, 1, 128, 3),
    ([70], [0], 8, 1, 256, 2), ([12], [2100], 4, 2, 128, 4)])
def test_trees(ops, fmt, new, past, heads, kv, d, words):
    rng = np.random.default_rng(sum(new))
    b = R.Batch(rng, new, past, 32, extra_rows=1)
    cache, ks, vs = filled(ops, rng, b, kv, d, fmt)
    q = normal(rng, b.rows, heads, d)
    tree = np.zeros((b.rows, words), np.uint64)
    for i, n in enumerate(new):
        tree[b.row_start[i]:b.row_start[i + 1]] = tree_words(rng, n, words)
    tree[1] = 0  # a row that sees only what is before the tree
    # Bits of places without a row mean nothing.
    tree[b.row_start[1] - 1, -1] |= np.uint64(1) << np.uint64(63) if max(new) < 64 * words else np.uint64(0)
    y = cache.attend(q, **b.args(), tree=tree)
    check_rows(y, q, b, ks, vs, 1 / np.sqrt(d), tree)
    if past[0] == 0:
        assert not y[1].any()  # nothing visible: zeros
    assert not y[-1:].any()
    cache.release()


def test_a_chain_of_drafts_is_causal(ops):
    rng = np.random.default_rng(41)
    b = R.Batch(rng, [30], [77], 16)
    cache, ks, vs = filled(ops, rng, b, 2, 64, "int8")
    q = normal(rng, 30, 4, 64)
    tree = ((np.uint64(2) << np.arange(30, dtype=np.uint64)) - np.uint64(1))[:, None]
    check_rows(cache.attend(q, **b.args(), tree=tree), q, b, ks, vs, 0.125)
    check_rows(cache.attend(q, **b.args()), q, b, ks, vs, 0.125)
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_non_finite_values_reach_their_viewers_only(ops, fmt, which, value):
    rng = np.random.default_rng(42)
    new, past = 20, 45
    b = R.Batch(rng, [new], [past], 16)
    k, v = normal(rng, 65, 2, 64), normal(rng, 65, 2, 64)
    (k if which == "k" else v)[past + 6, 1, 9] = value  # drafted row 6, KV head 1
    cache = ops.KvCache(b.pages, kv_heads=2, head_size=64, page_size=16, fmt=fmt)
    cache.append(k, v, row_start=[0, 65], past=[0], page_table=b.page_table)
    q = normal(rng, new, 4, 64)
    tree = tree_words(rng, new, 1)
    for t in (tree, None):
        y = cache.attend(q, **b.args(), tree=t)
        sees = R.visible(new, past, t)[:, past + 6]
        bad = np.isnan(y).all(-1)
        assert (np.isnan(y).any(-1) == bad).all()
        want = np.zeros((new, 4), bool)
        want[sees, 2:] = True
        same(bad, want)
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
def test_what_lies_behind_a_sequence_is_not_seen(ops, fmt):
    # Places past the length hold NaN and huge vectors of an earlier, longer sequence.
    rng = np.random.default_rng(43)
    b = R.Batch(rng, [1, 3], [50, 18], 32)
    cache = ops.KvCache(b.pages, kv_heads=1, head_size=64, page_size=32, fmt=fmt)
    k, v = normal(rng, 128, 1, 64), normal(rng, 128, 1, 64)
    lengths = [51, 21]
    for i, n in enumerate(lengths):
        k[64 * i + n:64 * (i + 1)], v[64 * i + n:64 * (i + 1)] = 3e38, 3e38
        k[64 * i + n, 0, 0], v[64 * i + n + 1, 0, 3] = np.nan, np.inf
    table = np.full((2, 2), 0, np.int32)
    table[:, :b.page_table.shape[1]] = b.page_table
    cache.append(k, v, row_start=[0, 64, 128], past=[0, 0], page_table=table)
    q = normal(rng, 4, 4, 64)
    y = cache.attend(q, row_start=b.row_start, past=b.past, page_table=table)
    ks, vs = ([R.cached(t[64 * i:64 * i + n], fmt) for i, n in enumerate(lengths)] for t in (k, v))
    check_rows(y, q, b, ks, vs, 0.125)
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
def test_scales_far_apart(ops, fmt):
    # Keys and values whose sizes span 2^-60 .. 2^60, rising and falling along the sequence;
    # queries from 1e-20 to 1e20 with scales that keep scores moderate.
    rng = np.random.default_rng(44)
    for sizes in (np.exp2(np.linspace(-60, 60, 200)), np.exp2(np.linspace(60, -60, 200)),
                  np.exp2(rng.uniform(-60, 60, 200))):
        b = R.Batch(rng, [1], [199], 16)
        k = normal(rng, 200, 1, 64)
        v = normal(rng, 200, 1, 64) * sizes[:, None, None].astype(np.float32)
        cache = ops.KvCache(b.pages, kv_heads=1, head_size=64, page_size=16, fmt=fmt)
        cache.append(k, v, row_start=[0, 200], past=[0], page_table=b.page_table)
        for size in (1e-20, 1e20):
            q = normal(rng, 1, 2, 64) * np.float32(size)
            scale = float(np.float32(0.125 / size))
            y = cache.attend(q, **b.args(), scale=scale)
            check_rows(y, q, b, [R.cached(k, fmt)], [R.cached(v, fmt)], scale)
        cache.release()
    # All values zero, and all scores far below zero or far above.
    b = R.Batch(rng, [3], [40], 16)
    cache, ks, vs = filled(ops, rng, b, 1, 64, fmt)
    q = normal(rng, 3, 1, 64)
    for scale in (0.0, 30.0, -30.0):
        check_rows(cache.attend(q, **b.args(), scale=scale), q, b, ks, vs, scale)
    cache.release()


# Many short prompts: workgroups of 64 rows; longer ones: of 128 (heads up to 128).
MANY = [(40, 16), (32, 64)]


def many(rng, count, most, page=16, past=100):
    """A batch of `count` sequences, up to `most` new rows each (some of them none or one)."""
    new = rng.integers(2, most + 1, count)
    new[0], new[1], new[2] = most, 0, 1
    return R.Batch(rng, [int(n) for n in new], rng.integers(0, past, count), page, extra_rows=1)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [33, 64, 128, 160, 256])
@pytest.mark.parametrize("count, most", MANY)
def test_many_rows(ops, fmt, d, count, most):
    rng = np.random.default_rng(d + count)
    b = many(rng, count, most, past=260)
    cache, ks, vs = filled(ops, rng, b, 8, d, fmt, 1.5)
    q = normal(rng, b.rows, 32, d)
    y = cache.attend(q, **b.args())
    check_rows(y, q, b, ks, vs, 1 / np.sqrt(d))
    assert not y[-1:].any()
    tree = np.zeros((b.rows, 1), np.uint64)
    for i, n in enumerate(b.new):
        tree[b.row_start[i]:b.row_start[i + 1]] = tree_words(rng, n, 1)
    tree[1] = 0
    cos, sin = tables(rng, 400, d // 2)
    pos = np.concatenate([p + np.arange(n) for n, p in zip(b.new, b.past)] + [[0]])
    y = cache.attend(q, **b.args(), tree=tree, rope=(cos, sin, False))
    check_rows(y, R.rotate(q, cos, sin, pos, False), b, ks, vs, 1 / np.sqrt(d), tree)
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kv, group, new, past, d", [(1, 16, 500, 8000, 128), (1, 8, 500, 3000, 256)])
def test_long_prompt_chunks(ops, fmt, kv, group, new, past, d):
    # Row blocks and key splits at once; a sample of the rows is compared.
    rng = np.random.default_rng(past)
    b = R.Batch(rng, [new], [past], 64)
    cache, ks, vs = filled(ops, rng, b, kv, d, fmt)
    q = normal(rng, new, kv * group, d)
    y = cache.attend(q, **b.args())
    see = R.visible(new, past)
    for r in (0, 1, 127, 128, 300, new - 1):
        want = R.attend(q[r:r + 1], ks[0], vs[0], see[r:r + 1], 1 / np.sqrt(d))
        assert np.abs(y[r] - want).max() <= R.bound(q[r], ks[0], vs[0], 1 / np.sqrt(d))
    cache.release()


def check_each_row(y, q, b, ks, vs, scale, tree=None):
    """As check_rows, a row's bound from its own query and what it sees alone."""
    for i, (k, v) in enumerate(zip(ks, vs)):
        r = slice(b.row_start[i], b.row_start[i + 1])
        see = R.visible(b.new[i], int(b.past[i]), None if tree is None else tree[r])
        want = R.attend(q[r], k, v, see, scale)
        for j, row in enumerate(range(r.start, r.stop)):
            for h in range(q.shape[1]):
                at = (row, slice(h, h + 1))
                err = np.abs(y[at] - want[j, h]).max()
                tol = R.bound(q[at], k[see[j]], v[see[j]], scale) if see[j].any() else 0
                assert err <= tol, (i, j, h, err, tol)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("count, most, d", [(2, 16, 64), (40, 16, 64), (32, 64, 64), (32, 64, 128),
                                            (2, 16, 256), (40, 16, 256)])
def test_rows_do_not_feel_one_another(ops, fmt, count, most, d):
    # Queries and values of neighbouring rows 2^40 and more apart: what a row does not see, and
    # how large another row's query is, costs it nothing.
    rng = np.random.default_rng(d + most)
    new = rng.integers(2, most + 1, count)
    new[0] = most
    b = R.Batch(rng, [int(n) for n in new], rng.integers(0, 40, count), 16)
    n = [int(x) for x in b.past + b.new]
    k, v = normal(rng, sum(n), 8, d), normal(rng, sum(n), 8, d)
    v *= np.exp2(rng.choice([-50, 0, 30], sum(n)))[:, None, None].astype(np.float32)
    cache = ops.KvCache(b.pages, kv_heads=8, head_size=d, page_size=16, fmt=fmt)
    cache.append(k, v, row_start=np.concatenate([[0], np.cumsum(n)]), past=np.zeros(count),
                 page_table=b.page_table)
    cut = np.cumsum(n)[:-1]
    ks, vs = np.split(R.cached(k, fmt), cut), np.split(R.cached(v, fmt), cut)
    q = normal(rng, b.rows, 32, d)
    q[rng.random((b.rows, 32)) < 0.1] *= np.float32(2.0**40)
    q[rng.random((b.rows, 32)) < 0.1] *= np.float32(2.0**-40)
    tree = np.zeros((b.rows, 1), np.uint64)
    for i, m in enumerate(b.new):
        tree[b.row_start[i]:b.row_start[i + 1]] = tree_words(rng, m, 1)
    for t in (None, tree):
        check_each_row(cache.attend(q, **b.args(), tree=t), q, b, ks, vs, 1 / np.sqrt(d), t)
    cache.release()


def test_pages_beyond_32_bit_offsets(ops):
    # A cache of more than 2^32 code bytes, the sequence in its last pages.
    rng = np.random.default_rng(45)
    kv, d, page = 8, 128, 256
    pages = 2**32 // (kv * d * page) + 40
    b = R.Batch(rng, [3, 1], [700, 300], page)
    b.page_table = pages - 1 - b.page_table
    for fmt in ("int8", "int4"):
        n = pages if fmt == "int8" else 2 * pages
        b.pages = n
        b.page_table = n - 1 - np.argsort(rng.random(b.page_table.size)).astype(np.int32).reshape(
            b.page_table.shape)
        cache, ks, vs = filled(ops, rng, b, kv, d, fmt)
        q = normal(rng, b.rows, 16, d)
        check_rows(cache.attend(q, **b.args()), q, b, ks, vs, 1 / np.sqrt(d))
        gk, gv = cache.read(b.rows, **b.args())
        same(gk, np.concatenate([k[-n_:] for k, n_ in zip(ks, b.new)]))
        assert not cache.refused()
        cache.release()


def test_strided_queries_and_outputs(ops):
    rng = np.random.default_rng(46)
    b = R.Batch(rng, [5, 70], [30, 2], 16)
    cache, ks, vs = filled(ops, rng, b, 2, 70, "int8")
    for pad, off in ((3, 1), (4, 0)):
        mem = normal(rng, off + b.rows * (4 * 70 + pad))
        q = mem[off:].reshape(b.rows, -1)[:, :280].reshape(b.rows, 4, 70)
        out = np.full(off + b.rows * (280 + 9), 7, np.float32)
        dev = device(ops, b.row_start, b.past, b.page_table, mem, out)
        cache.attend_dev(seq_batch(ops, b, dev), dev[3].ptr + 4 * off, dev[4].ptr + 4 * off, 4,
                         q_stride=280 + pad, y_stride=289)
        y = dev[4].to_array(out.shape, np.float32)
        rows = y[off:].reshape(b.rows, 289)
        assert (rows[:, 280:] == 7).all() and (y[:off] == 7).all()
        check_rows(rows[:, :280].reshape(q.shape), q, b, ks, vs, 1 / np.sqrt(70))
        for x in dev:
            x.free()
    cache.release()


def test_loose_bounds(ops):
    # Launches planned for more rows and longer sequences than the arrays hold give the
    # same kind of result, also where the bound passes the page table.
    rng = np.random.default_rng(47)
    b = R.Batch(rng, [2, 1], [40, 9], 16)
    cache, ks, vs = filled(ops, rng, b, 2, 64, "int8")
    q = normal(rng, 80, 8, 64)
    dev = device(ops, b.row_start, b.past, b.page_table, q, np.full_like(q, 7))
    for max_new, max_len in ((2, 42), (3, 43), (17, 5000), (80, 100000)):
        cache.attend_dev(seq_batch(ops, b, dev, max_new, max_len, rows=80), dev[3].ptr, dev[4].ptr, 8)
        y = dev[4].to_array(q.shape, np.float32)
        check_rows(y, q, b, ks, vs, 0.125)
        assert (y[3:] == 7).all()
    assert not cache.refused()
    for x in dev:
        x.free()
    cache.release()


def test_more_rows_than_a_launch_takes(ops):
    # Refused from the bounds alone, whatever the arrays hold.
    cache = ops.KvCache(1, kv_heads=4096, head_size=1, page_size=16)
    x = ops.DeviceBuffer.from_array(np.zeros(100, np.int32))
    s = ops.SeqBatch(batch=65535, rows=2**31 - 256, max_new=2**31 - 256, max_len=2**31 - 256,
                     row_start_ptr=x.ptr, past_ptr=x.ptr, page_table_ptr=x.ptr, table_stride=1)
    with pytest.raises(UnsupportedError):
        cache.attend_dev(s, x.ptr, x.ptr, 4096)
    with pytest.raises(UnsupportedError):
        cache.attend_dev(s, x.ptr, x.ptr, 8192)
    x.free()
    cache.release()


def test_shared_pages_and_contexts(ops):
    # Two sequences read one prefix page; two contexts (streams) use one cache in turn.
    rng = np.random.default_rng(48)
    k, v = normal(rng, 40, 1, 64), normal(rng, 40, 1, 64)
    a, c = ops.Context(), ops.Context()
    cache = ops.KvCache(5, kv_heads=1, head_size=64, page_size=16, ctx=a)
    cache.append(k[:16], v[:16], row_start=[0, 16], past=[0], page_table=[[4]])
    cache.append(k[16:], v[16:], row_start=[0, 10, 24], past=[16, 16], page_table=[[4, 0], [4, 2]])
    q = normal(rng, 2, 2, 64)
    args = dict(row_start=[0, 1, 2], past=[25, 29], page_table=[[4, 0], [4, 2]])
    y = cache.attend(q, **args)
    cache.ctx = c
    same(cache.attend(q, **args), y)
    cache.ctx = a
    b = R.Batch(rng, [1, 1], [25, 29], 16)
    kr, vr = R.cached(k, "int8"), R.cached(v, "int8")
    ks, vs = ([t[:26], np.concatenate([t[:16], t[26:]])] for t in (kr, vr))
    check_rows(y, q, b, ks, vs, 0.125)
    cache.release()
    a.close()
    c.close()


def test_repeated_calls_are_equal(ops):
    rng = np.random.default_rng(49)
    b = R.Batch(rng, [1] * 6, [3000, 10, 500, 77, 1200, 0], 64)
    cache, _, _ = filled(ops, rng, b, 4, 128, "e4m3")
    q = normal(rng, b.rows, 16, 128)
    y = cache.attend(q, **b.args())
    for _ in range(4):
        same(cache.attend(q, **b.args()), y)
    cache.release()


# --------------------------------------------------- the operators together


def test_a_decode_loop_with_drafts(ops):
    # Serving as a program does it: tables, a prompt, then steps that append a tree of
    # drafted tokens, attend, score the drafts from logits and keep one branch.
    rng = np.random.default_rng(50)
    heads, kv, d, half, page, vocab = 4, 2, 64, 32, 16, 500
    cos, sin = ops.rotary_tables(200, half, scaling=ops.RopeScaling("yarn", factor=4.0,
                                                                   original_length=64))
    head = normal(rng, heads * d, vocab)
    table = rng.permutation(9).astype(np.int32)[:8][None]
    cache = ops.KvCache(9, kv_heads=kv, head_size=d, page_size=page, fmt="int8")
    k, v, q = normal(rng, 37, kv, d), normal(rng, 37, kv, d), normal(rng, 37, heads, d)
    where = dict(row_start=[0, 37], past=[0], page_table=table)
    cache.append(k, v, **where, rope=(cos, sin, False))
    kc = R.cached(R.rotate(k, cos, sin, np.arange(37), False), "int8")
    vc = R.cached(v, "int8")
    b = R.Batch(rng, [37], [0], page)
    y = cache.attend(q, **where, rope=(cos, sin, False))
    check_rows(y, R.rotate(q, cos, sin, np.arange(37), False), b, [kc], [vc], 0.125)
    length = 37
    for n in (6, 9, 4):
        tree = tree_words(rng, n, 1)
        depth = np.array([bin(int(w)).count("1") - 1 for w in tree[:, 0]])
        pos = length + depth
        k, v, q = normal(rng, n, kv, d), normal(rng, n, kv, d), normal(rng, n, heads, d)
        where = dict(row_start=[0, n], past=[length], page_table=table)
        rope = (cos, sin, False, pos)
        cache.append(k, v, **where, rope=rope)
        kd, vd = R.cached(R.rotate(k, cos, sin, pos, False), "int8"), R.cached(v, "int8")
        # (Turned by the operator of its own, as a graph with its own node does.)
        qr = ops.op_rotary_embedding(q.reshape(1, n, -1), cos, sin, pos[None], num_heads=heads)
        y = cache.attend(qr.reshape(q.shape), **where, tree=tree)
        b = R.Batch(rng, [n], [length], page)
        check_rows(y, R.rotate(q, cos, sin, pos, False), b, [np.concatenate([kc, kd])],
                   [np.concatenate([vc, vd])], 0.125, tree)
        same(cache.attend(q, **where, tree=tree, rope=rope), y)
        logits = ops.op_matmul(y.reshape(n, -1), head)
        lp, ent, ids, tops = ops.op_token_logprobs(logits, rng.integers(0, vocab, n), top=3)
        z = logits.astype(np.float64)
        z = z - z.max(-1, keepdims=True)
        z = z - np.log(np.exp(z).sum(-1, keepdims=True))
        same(ids, np.argsort(-logits, -1, kind="stable")[:, :3])
        assert np.abs(tops - np.take_along_axis(z, ids.astype(np.int64), -1)).max() <= 1e-5
        # The branch of the last row is kept: its rows are written again, in order.
        keep = np.flatnonzero([(int(tree[-1, 0]) >> j) & 1 for j in range(n)])
        where = dict(row_start=[0, len(keep)], past=[length], page_table=table)
        cache.append(k[keep], v[keep], **where, rope=(cos, sin, False))
        kc = np.concatenate([kc, kd[keep]])
        vc = np.concatenate([vc, vd[keep]])
        length += len(keep)
        gk, gv = cache.read(length, row_start=[0, length], past=[0], page_table=table)
        same(gk, kc)
        same(gv, vc)
    assert not cache.refused()
    cache.release()


class Hip:
    """The HIP runtime that the library itself has loaded."""

    def __init__(self):
        with open("/proc/self/maps") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        self.lib = C.CDLL(path)

    def __getattr__(self, name):
        def call(*args):
            rc = getattr(self.lib, name)(*args)
            assert rc == 0, (name, rc)
        return call


@pytest.mark.parametrize("warm", [True, False])
def test_captured_steps(ops, warm):
    # A decode step (append, attend, score) captured once and replayed with other lengths:
    # the kernels read the lengths.  Cold: no workspace can be had while capturing.
    rng = np.random.default_rng(51)
    hip = Hip()
    ctx = ops.Context()
    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    hip.hipStreamCreate(C.byref(stream))
    ctx.set_stream(stream.value)
    kv, heads, d, page, vocab = 2, 8, 64, 32, 9000
    b = R.Batch(rng, [1, 1, 1], [900, 30, 400], page)
    cache, ks, vs = filled(ops, rng, b, kv, d, "int4", ctx=ctx)
    cos, sin = tables(rng, 1000, 32)
    q, k, v, x = normal(rng, 3, heads, d), normal(rng, 3, kv, d), normal(rng, 3, kv, d), normal(rng, 3, vocab)
    dev = device(ops, b.row_start, b.past, b.page_table, q, k, v, cos, sin, x,
                 np.array([1, 2, 3], np.int32), np.zeros_like(q), np.zeros(3, np.float32),
                 np.zeros(3, np.float32), np.zeros((3, 5), np.int32), np.zeros((3, 5), np.float32))
    s = seq_batch(ops, b, dev, max_len=901)
    rope = ops.Rope(dev[6].ptr, dev[7].ptr, max_pos=1000, half_rot=32)

    def step():
        cache.append_dev(s, dev[4].ptr, dev[5].ptr, rope=rope)
        cache.attend_dev(s, dev[3].ptr, dev[10].ptr, heads, rope=rope)
        ops.token_logprobs_dev(dev[8].ptr, 3, vocab, tokens_ptr=dev[9].ptr, logprob_ptr=dev[11].ptr,
                               entropy_ptr=dev[12].ptr, top=5, top_ids_ptr=dev[13].ptr,
                               top_logprobs_ptr=dev[14].ptr, ctx=ctx)

    def results():
        hip.hipStreamSynchronize(stream)
        return [dev[i].to_array(sh, t) for i, sh, t in (
            (10, q.shape, np.float32), (11, (3,), np.float32), (12, (3,), np.float32),
            (13, (3, 5), np.int32), (14, (3, 5), np.float32))]

    def put(i, a):
        hip.hipMemcpy(C.c_void_p(dev[i].ptr), a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes), 1)

    if warm:
        step()
        hip.hipStreamSynchronize(stream)
    hip.hipStreamBeginCapture(stream, 0)
    step()
    hip.hipStreamEndCapture(stream, C.byref(graph))
    hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0))
    for past in ([900, 30, 400], [10, 899, 64], [0, 1, 2]):
        b.past = np.array(past, np.int32)
        put(1, b.past)
        k, q = normal(rng, 3, kv, d), normal(rng, 3, heads, d)
        put(4, k)
        put(3, q)
        put(8, normal(rng, 3, vocab))
        hip.hipGraphLaunch(exe, stream)
        got = results()
        for i in range(10, 15):
            put(i, np.zeros(dev[i].nbytes // 4, np.int32))
        step()
        want = results()
        for g, w in zip(got, want):
            if warm:
                same(g, w)
            else:  # another split of the same sums
                np.testing.assert_allclose(g, w, rtol=0, atol=2e-5)
        assert got[0].any()
    hip.hipGraphExecDestroy(exe)
    hip.hipGraphDestroy(graph)
    for x in dev:
        x.free()
    cache.release()
    ctx.close()
    hip.hipStreamDestroy(stream)


def test_profile_names(ops):
    ctx = ops.Context()
    rng = np.random.default_rng(52)
    b = R.Batch(rng, [2], [3], 16)
    cache, _, _ = filled(ops, rng, b, 1, 64, "int8", ctx=ctx)
    ctx.set_profiling(True)
    cache.attend(normal(rng, 2, 1, 64), **b.args())
    cache.read(2, **b.args())
    ops.rotary_tables(4, 8, ctx=ctx)
    ops.op_token_logprobs(normal(rng, 2, 9), ctx=ctx)
    names = [n for n, _ in ctx.profile_records()]
    assert names == ["KvCacheAttention", "KvCacheRead", "RotaryTables", "TokenLogProbs"]
    cache.release()
    ctx.close()


@pytest.mark.parametrize("fmt", FMTS)
def test_sequences_without_rows(ops, fmt):
    # In a batch that others have rows of, the first and last sequences among them: nothing of
    # theirs is read, written or refused, wherever their pasts end and whatever their pages are.
    rng = np.random.default_rng(61)
    new, past = [0, 2, 0, 0, 1, 0], [5, 6, 31, 1, 3, 2]
    b = R.Batch(rng, new, past, 16)
    cache, ks, vs = filled(ops, rng, b, 2, 64, fmt)
    before = [cache.read(p, row_start=[0, p], past=[0], page_table=b.page_table[i:i + 1])
              for i, p in enumerate(past)]
    table = b.page_table.copy()
    table[2] = -1
    k, v = normal(rng, b.rows, 2, 64), normal(rng, b.rows, 2, 64)
    cos, sin = tables(rng, 40, 16)
    for rope in (None, (cos, sin, False)):
        cache.append(k, v, row_start=b.row_start, past=past, page_table=table, rope=rope)
        assert not cache.refused()
    gk, gv = cache.read(b.rows, row_start=b.row_start, past=past, page_table=table)
    assert not cache.refused()
    same(gv, R.cached(v, fmt))
    q = normal(rng, b.rows, 4, 64)
    y = cache.attend(q, row_start=b.row_start, past=past, page_table=table)
    assert np.isfinite(y).all() and not cache.refused()
    for i, p in enumerate(past):
        rk, rv = cache.read(p, row_start=[0, p], past=[0], page_table=b.page_table[i:i + 1])
        same(rk, before[i][0])
        same(rv, before[i][1])
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new, past", [
    ([1], [0]), ([1], [700]), ([3], [17]), ([20], [40]), ([2, 0, 1], [9, 8, 7])])
def test_more_new_rows_allowed_than_there_are(ops, fmt, new, past):
    # max_new above the rows of the whole batch, in all three calls.
    rng = np.random.default_rng(63)
    b = R.Batch(rng, new, past, 16)
    cache, ks, vs = filled(ops, rng, b, 2, 64, fmt)
    k, v, q = normal(rng, b.rows, 2, 64), normal(rng, b.rows, 2, 64), normal(rng, b.rows, 8, 64)
    out = np.zeros_like(k)
    dev = device(ops, b.row_start, b.past, b.page_table, k, v, out, out, q, np.zeros_like(q))
    for most in (b.rows, b.rows + 1, 33, 600):
        s = seq_batch(ops, b, dev, max_new=most, max_len=1000)
        cache.append_dev(s, dev[3].ptr, dev[4].ptr)
        cache.read_dev(s, dev[5].ptr, dev[6].ptr)
        same(dev[5].to_array(k.shape, np.float32), R.cached(k, fmt))
        same(dev[6].to_array(k.shape, np.float32), R.cached(v, fmt))
        for i in range(len(new)):
            r = slice(b.row_start[i], b.row_start[i + 1])
            ks[i][past[i]:], vs[i][past[i]:] = R.cached(k[r], fmt), R.cached(v[r], fmt)
        cache.attend_dev(s, dev[7].ptr, dev[8].ptr, 8)
        check_rows(dev[8].to_array(q.shape, np.float32), q, b, ks, vs, 0.125)
        assert not cache.refused()
    for x in dev:
        x.free()
    cache.release()


@pytest.mark.parametrize("past, max_len", [
    ([0], 131072), ([126], 131072), ([127], 131072), ([128], 131072), ([8191], 8192),
    ([8192], 131072), ([20000], 20001), ([20001], 131072), ([32766, 1, 0, 300], 32767),
    ([300, 32768, 4000], 2**31 - 256), ([513, 1023, 1024, 1025, 5000], 700000)])
def test_splits_share_a_sequence_out(ops, past, max_len):
    # Whatever the bound, every key counts once.
    rng = np.random.default_rng(sum(past))
    b = R.Batch(rng, [1] * len(past), past, 256)
    cache, ks, vs = filled(ops, rng, b, 2, 64, "int8")
    q = normal(rng, b.rows, 4, 64)
    dev = device(ops, b.row_start, b.past, b.page_table, q, np.zeros_like(q))
    cache.attend_dev(seq_batch(ops, b, dev, max_len=max_len), dev[3].ptr, dev[4].ptr, 4)
    check_rows(dev[4].to_array(q.shape, np.float32), q, b, ks, vs, 0.125)
    # All scores alike: a key left out or taken twice shows in the mean, by 1 / t of a value.  (Digits
    # round to 2^-22, a thousand tiles' sums walk by some 32 roundings of 2^-24.)
    cache.attend_dev(seq_batch(ops, b, dev, max_len=max_len), dev[3].ptr, dev[4].ptr, 4, scale=0.0)
    y = dev[4].to_array(q.shape, np.float32)
    for i, v in enumerate(vs):
        mean = v.astype(np.float64).mean(0).repeat(2, 0)
        assert np.abs(y[i] - mean).max() <= 2e-6 * np.abs(v).max()
    for x in dev:
        x.free()
    cache.release()


@pytest.mark.parametrize("max_bytes", [0, -1])
@pytest.mark.parametrize("new, heads", [(1, 2), (30, 2), (60, 32)])
def test_lengths_beyond_the_page_table(ops, new, heads, max_bytes):
    # Pasts of 2^31 and a little beyond the table: the rows that see missing pages are NaN, and
    # the call ends at the table; the sequence beside them is as ever.
    rng = np.random.default_rng(62)
    ctx = ops.Context()
    b = R.Batch(rng, [new] * 33, [100] * 33, 16)
    cache, ks, vs = filled(ops, rng, b, 8 if heads == 32 else 2, 64, "int8", ctx=ctx)
    past = b.past.copy()
    stride = b.page_table.shape[1]
    past[0], past[2] = 2**31 - 300, 16 * stride  # far and just beyond
    past[1] = 16 * stride - 1                     # its first row sees the whole table
    q = normal(rng, b.rows, heads, 64)
    dev = device(ops, b.row_start, past, b.page_table, q, np.full(q.shape, 7, np.float32))
    ctx.set_control(max_bytes=max_bytes)
    s = seq_batch(ops, b, dev, max_len=2**31 - 256)
    cache.attend_dev(s, dev[3].ptr, dev[4].ptr, heads)
    ctx.synchronize()
    y = dev[4].to_array(q.shape, np.float32)
    assert cache.refused()
    # (60 rows from 2^31 - 300 pass max_len: refused whole, rows as they were.)
    assert (np.isnan(y[:new]) if new <= 44 else y[:new] == 7).all()
    assert np.isnan(y[2 * new:3 * new]).all()
    assert np.isfinite(y[new]).all() and np.isnan(y[new + 1:2 * new]).all()
    for i in range(3, 33):
        r = slice(i * new, (i + 1) * new)
        want = R.attend(q[r], ks[i], vs[i], R.visible(new, 100), 0.125)
        assert np.abs(y[r] - want).max() <= R.bound(q[r], ks[i], vs[i], 0.125)
    ctx.set_control(max_bytes=-1)
    # Writing there is refused, whatever the bounds.
    k = normal(rng, b.rows, cache.kv_heads, 64)
    kd = ops.DeviceBuffer.from_array(k)
    cache.append_dev(s, kd.ptr, kd.ptr)
    assert cache.refused()
    gk, _ = cache.read(b.rows, **b.args())
    same(gk[3 * new:], R.cached(k, "int8")[3 * new:])
    for x in dev + [kd]:
        x.free()
    cache.release()
    ctx.close()


def test_host_numbers_beyond_32_bits(ops):
    cache = ops.KvCache(2, kv_heads=1, head_size=64, page_size=16)
    k = np.ones((1, 1, 64), np.float32)
    with pytest.raises(ArgumentError):
        cache.append(k, k, row_start=[0, 1], past=[2**32], page_table=[[0]])
    with pytest.raises(ArgumentError):
        cache.append(k, k, row_start=[0, 2**32 + 1], past=[0], page_table=[[0]])
    cache.append(k, k, row_start=[0, 1], past=[0], page_table=[[2**32 + 1]])
    assert cache.refused()
    cos = np.ones((4, 8), np.float32)
    cache.append(k, k, row_start=[0, 1], past=[0], page_table=[[1]],
                 rope=(cos, 0 * cos, False, [2**32 + 1]))
    gk, gv = cache.read(1, row_start=[0, 1], past=[0], page_table=[[1]])
    assert np.isnan(gk).all() and (np.abs(gv - 1) < 0.01).all()
    # Nothing to write, nothing to read.
    none = np.zeros((0, 1, 64), np.float32)
    cache.append(none, none, row_start=[0], past=[], page_table=np.zeros((0, 3), np.int32))
    cache.append(none, none, row_start=[0, 0], past=[5], page_table=[[1]])
    assert cache.attend(none, row_start=[0, 0], past=[5], page_table=[[1]]).shape == (0, 1, 64)
    assert not cache.refused()
    cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("base", [1.0, -1.0, 1.0000001192, -3e-20, 7e6, 2.0**100])
def test_nearly_constant_vectors(ops, fmt, base):
    # Extremes 1 to 40 units in the last place apart, on both parities: the middle's rounding
    # leaves one of them outside middle +- 15 steps (INT4), where the code is the last one.
    rng = np.random.default_rng(26)
    n, d = 80, 64
    first = np.full((n, 2, 1), np.float32(base)).view(np.int32) + (np.arange(n) % 2)[:, None, None]
    steps = (1 + np.arange(n) // 2)[:, None, None]
    b = R.Batch(rng, [n], [3], 16)
    cache = ops.KvCache(b.pages, kv_heads=2, head_size=d, page_size=16, fmt=fmt)
    for part in (rng.integers(0, 2, (n, 2, d)), rng.random((n, 2, d))):
        part[..., :2] = [0, 1]  # (both extremes are there)
        bits = first + np.rint(rng.permuted(part.astype(np.float64), axis=-1) * steps)
        k = bits.astype(np.int32).view(np.float32)
        v = k[..., ::-1].copy()
        cache.append(k, v, **b.args())
        gk, gv = cache.read(n, **b.args())
        same(gk, R.cached(k, fmt))
        same(gv, R.cached(v, fmt))
    cache.release()


@pytest.mark.parametrize("max_bytes", [0, -1])
@pytest.mark.parametrize("count, heads", [(1, 2), (40, 32)])
@pytest.mark.parametrize("past, stride", [(16, 1), (0, 0), (5, 1), (15, 1), (17, 1), (700, 44), (704, 44),
                                          (705, 44)])
def test_drafts_beyond_the_page_table(ops, count, heads, past, stride, max_bytes):
    # Positions past the table read as NaN, in whatever rows see them: also in those that see
    # one far behind the table's end and none of the first ones there.
    rng = np.random.default_rng(past + count)
    ctx = ops.Context()
    new, kv, page = 64, 8 if heads == 32 else 2, 16
    total = past + new
    pages = -(-total // page)
    b = R.Batch(rng, [new] * count, [past] * count, page)
    cache, ks, vs = filled(ops, rng, b, kv, 64, "int8", ctx=ctx)
    table = np.ascontiguousarray(b.page_table[:, :stride])
    q = normal(rng, b.rows, heads, 64)
    tree = np.zeros((b.rows, 1), np.uint64)
    own = np.uint64(1) << np.arange(new, dtype=np.uint64)
    for i in range(count):
        tree[i * new:(i + 1) * new, 0] = own
    tree[3], tree[5] = 0, 1  # one that sees the past alone, one that sees the first draft
    dev = device(ops, b.row_start, b.past, table if stride else np.zeros(1, np.int32), q,
                 np.full(q.shape, 7, np.float32), tree)
    s = ops.SeqBatch(batch=count, rows=b.rows, max_new=new, max_len=pages * page,
                     row_start_ptr=dev[0].ptr, past_ptr=dev[1].ptr, page_table_ptr=dev[2].ptr,
                     table_stride=stride)
    ctx.set_control(max_bytes=max_bytes)
    cache.attend_dev(s, dev[3].ptr, dev[4].ptr, heads, tree_ptr=dev[5].ptr, tree_words=1)
    ctx.synchronize()
    y = dev[4].to_array(q.shape, np.float32)
    assert cache.refused()
    for i in range(min(count, 3)):
        r = slice(i * new, (i + 1) * new)
        see = R.visible(new, past, tree[r])
        lost = see[:, stride * page:].any(-1)
        assert np.isnan(y[r][lost]).all()
        want = R.attend(q[r], ks[i], vs[i], see, 0.125)
        err = np.abs(y[r][~lost] - want[~lost]).max(initial=0)
        assert err <= R.bound(q[r], ks[i], vs[i], 0.125)
    ctx.set_control(max_bytes=-1)
    for x in dev:
        x.free()
    cache.release()
    ctx.close()
