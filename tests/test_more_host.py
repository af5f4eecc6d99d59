"""Verification of drafted tokens, pages of the KV cache, low-rank adapters: what is refused
before any device is touched, what needs none, and the references of their tests on small
cases that are plain to see."""
import ctypes as C

import numpy as np
import pytest

import drafts_reference as R
import pages_reference as PR
from onnx_runtime_dart_amd import ops
from onnx_runtime_dart_amd.errors import ArgumentError, UnsupportedError
from test_kv_host import BUF, CACHE, CTX, Handle, P, seqs

lib = ops.lib
# A stand-in for a handle of adapters: device, format, projections, largest rank, K, kp, slots, bytes, N.
ADAPTERS = Handle(0, 0, 2, 8, 64, 0, 64, 0, 4, 0, 0, 0, 16, 0, 24, 0)


def drafts(**kw):
    base = dict(batch=2, rows=8, max_new=4, vocab=100, row_start_ptr=P, tokens_ptr=P, target_ptr=P,
                uniform_ptr=P)
    return ops.Drafts(**{**base, **kw})


def verify(out=P, kept=P, count=P, ctx=CTX.ptr, **kw):
    return lib.mg_verify_drafts_f32_dev(ctx, C.byref(drafts(**kw)), out, kept, count)


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(batch=65536), dict(rows=-1), dict(rows=2**31), dict(max_new=-1), dict(vocab=0),
    dict(vocab=2**31), dict(target_stride=99), dict(target_stride=-1), dict(draft_ptr=P, draft_stride=99),
    dict(target_stride=2**41), dict(row_start_ptr=0), dict(tokens_ptr=0), dict(target_ptr=0),
    dict(uniform_ptr=0), dict(out=None), dict(kept=None), dict(count=None), dict(ctx=None)], ids=str)
def test_drafts_out_of_bounds(bad):
    assert verify(**bad) == 1


def test_drafts_that_are_not_supported():
    assert verify(rows=2000, max_new=1025) == 2
    assert verify(draft_ptr=P, parent_ptr=P) == 2
    assert verify(batch=65535, rows=10**6, max_new=1000, vocab=10**6) == 2
    assert verify(batch=0, row_start_ptr=0, tokens_ptr=0, target_ptr=0, uniform_ptr=0, out=None, kept=None,
                  count=None) == 0


def test_drafts_beyond_a_launch():
    # 2^24 - 1 workgroups of 256 threads: four runs of 2048 logits each, of every row that a sequence may have.
    assert verify(batch=16384, rows=2**24, max_new=1024, vocab=2048) == 2
    assert verify(batch=16384, rows=2**24, max_new=1024, vocab=1) == 2
    assert verify(batch=8192, rows=2**24, max_new=1024, vocab=8192, draft_ptr=P) == 2
    assert verify(batch=8192, rows=2**24, max_new=1024, vocab=8193) == 2
    assert verify(batch=65535, rows=2**24, max_new=257, vocab=100) == 2


def copy(n=3, src=P, dst=P, cache=CACHE.ptr, ctx=CTX.ptr):
    return lib.mg_kv_cache_copy_pages_dev(ctx, cache, src, dst, n)


def compact(s=None, kept=P, count=P, past=P, cache=CACHE.ptr):
    return lib.mg_kv_cache_compact_dev(CTX.ptr, cache, C.byref(s or seqs()), kept, count, past)


def fork(s=None, parent=P, n=2, past=P + 64, table=P + 128, stride=4, refs=P, cache=CACHE.ptr):
    return lib.mg_kv_cache_fork_dev(CTX.ptr, cache, C.byref(s or seqs()), parent, n, past, table, stride, refs)


def fit(s=None, refs=P, granted=P, cache=CACHE.ptr):
    return lib.mg_kv_cache_fit_dev(CTX.ptr, cache, C.byref(s or seqs()), refs, granted)


OTHER = Handle(1, 0, 6, 2, 64, 64)


def test_pages_out_of_bounds():
    assert copy(n=-1) == copy(n=2**31) == copy(src=None) == copy(dst=None) == copy(cache=OTHER.ptr) == 1
    assert copy(cache=None) == copy(ctx=None) == 1
    assert copy(n=0, src=None, dst=None) == 0 and copy(n=2**30) == 2
    for call in (compact, fork, fit):
        assert call(cache=OTHER.ptr) == call(cache=None) == 1
        for bad in (dict(batch=-1), dict(batch=65536), dict(rows=2**31), dict(max_len=3), dict(table_stride=-1)):
            assert call(seqs(**bad)) == 1
    none = seqs(batch=0, row_start_ptr=0, past_ptr=0, page_table_ptr=0)
    assert compact(none, kept=None, count=None) == fit(none, refs=None, granted=None) == 0
    assert fork(none, n=0, parent=None, past=None, table=None, refs=None) == 0
    assert compact(kept=None) == compact(count=None) == 1
    assert compact(seqs(rows=0, row_start_ptr=0)) == 1  # (past_out is asked for)
    assert compact(seqs(rows=0), kept=None, past=None) == 0
    assert compact(seqs(batch=65535), cache=Handle(0, 0, 6, 4096, 64, 64).ptr) == 2
    assert fork(parent=None) == fork(past=None) == fork(table=None) == fork(refs=None) == fork(n=-1) == 1
    assert fork(n=65536) == fork(stride=-1) == fork(stride=2**31) == 1
    assert fork(past=P) == fork(table=P) == 1  # the old batch's own arrays
    assert fork(seqs(past_ptr=0, rows=0, max_new=0)) == 1
    assert fit(refs=None) == fit(granted=None) == fit(seqs(row_start_ptr=0, rows=0, max_new=0)) == 1
    assert fit(seqs(batch=65535), cache=Handle(0, 0, 8, 4096, 256, 256).ptr) == 2


def create(k=64, n=1, ns=(8,), slots=2, rank=4, fmt=0, ctx=CTX.ptr):
    out = C.c_void_p()
    return lib.mg_adapters_create(ctx, k, n, (C.c_int64 * len(ns))(*ns), slots, rank, fmt, C.byref(out))


def pointers(*p):
    return (C.c_void_p * len(p))(*p)


def put(slot=1, rank=4, a=pointers(P, P), b=pointers(P, P), factor=1.0, h=ADAPTERS.ptr, call=lib.mg_adapters_set):
    return call(CTX.ptr, h, slot, rank, a, b, factor)


def apply(x=P, rows=3, slot=P, base=pointers(P, P), y=pointers(P, P), h=ADAPTERS.ptr):
    return lib.mg_adapters_apply_f32_dev(CTX.ptr, h, x, rows, slot, base, y)


def test_adapters_out_of_bounds():
    assert create(k=0) == create(k=2**24 + 1) == create(n=0) == create(n=5, ns=[8] * 5) == create(ns=[0]) == 1
    assert create(ns=[2**23 + 1]) == create(slots=0) == create(slots=4097) == create(rank=0) == 1
    assert create(rank=257) == create(fmt=2) == create(fmt=-1) == create(ctx=None) == 1
    for call in (lib.mg_adapters_set, lib.mg_adapters_set_dev):
        assert put(slot=-1, call=call) == put(slot=4, call=call) == put(rank=-1, call=call) == 1
        assert put(rank=9, call=call) == put(a=None, call=call) == put(b=None, call=call) == 1
        assert put(a=pointers(P, None), call=call) == put(b=pointers(None, P), call=call) == 1
        assert put(factor=float("nan"), call=call) == put(factor=float("inf"), call=call) == 1
        assert put(h=Handle(1, 0, 2, 8, 64).ptr, call=call) == 1
    assert apply(x=None) == apply(slot=None) == apply(base=None) == apply(y=None) == apply(rows=-1) == 1
    assert apply(base=pointers(P, None)) == apply(y=pointers(None, P)) == apply(rows=2**31) == 1
    assert apply(h=Handle(1, 0, 2, 8, 64).ptr) == 1
    assert apply(rows=0, x=None, slot=None, base=None, y=None) == 0


@pytest.mark.parametrize("k, n, rank", [(16384, 1, 64), (16384, 3, 16), (2048, 2, 256), (300, 1, 5)])
def test_adapters_workspace_holds_a_short_last_round(k, n, rank):
    # Rows beyond 65536 go in rounds; a short one splits K into more parts, by the compute units there are.
    need = lib["_Z11mg_adapt_wsPK6mg_ctxRK11mg_adaptersl"]
    need.restype, need.argtypes = C.c_size_t, [C.c_void_p, C.c_void_p, C.c_int64]
    h = Handle(0, 0, n, rank, k, 0, k, 0, 4, 0, 0, 0, 8, 0)
    for cus in (1, 32, 80, 256, 304, 1000):
        ctx = Handle(*[0] * 22, cus)  # (compute units)
        for rows in (1, 50, 513, 700, 1216, 1217, 4000, 20000, 65535):
            assert need(ctx.ptr, h.ptr, 65536 + rows) >= need(ctx.ptr, h.ptr, rows)
            assert need(ctx.ptr, h.ptr, 65536 + rows) >= need(ctx.ptr, h.ptr, 65536)
    # (The field is the one that is meant.)
    if k > 512:
        few, many = (need(Handle(*[0] * 22, cus).ptr, h.ptr, 1216) for cus in (32, 256))
        assert few < many


def test_host_calls_check_their_arrays():
    x, u = np.zeros((3, 5), np.float32), np.zeros(3, np.float32)
    good = dict(target=x, tokens=[0, 1, 2], uniform=u, row_start=[0, 3], ctx=object())
    for bad in (dict(tokens=[0, 1]), dict(tokens=[0.0, 1.0, 2.0]), dict(uniform=[0, 1, 0]),
                dict(uniform=[0, -0.1, 0]), dict(uniform=[0, np.nan, 0]), dict(row_start=[0, 2]),
                dict(row_start=[1, 3]), dict(row_start=[0, 4, 3]), dict(row_start=[]), dict(target=x[0]),
                dict(draft=x[:2]), dict(parent=[0]), dict(temperature=[1, 1])):
        with pytest.raises(ArgumentError):
            ops.op_verify_drafts(**{**good, **bad})
    cache = ops.KvCache.__new__(ops.KvCache)
    cache.pages, cache.ctx = 4, object()
    for call in (lambda: cache.copy_pages([0, 1], [2]), lambda: cache.copy_pages([0.5], [1]),
                 lambda: cache.compact([0], [1], row_start=[0, 2], past=[0], page_table=[[0]]),
                 lambda: cache.compact([0], [1], row_start=[0, 1], past=[0], page_table=[0]),
                 lambda: cache.compact([0], [1], row_start=[0, 1], past=[-1], page_table=[[0]]),
                 lambda: cache.fork([0], past=[1], page_table=[[0]], refs=[1, 0, 0]),
                 lambda: cache.fit(row_start=[0, 1, 1], past=[1], page_table=[[0]], refs=[1, 0, 0, 0]),
                 lambda: cache.fit(row_start=[0, 1], past=[1], page_table=[[0]], refs=[1])):
        with pytest.raises(ArgumentError):
            call()
    with pytest.raises(ArgumentError):
        ops.Adapters(8, [8], slots=1, max_rank=1, fmt="bf16", ctx=object())
    h = ops.Adapters.__new__(ops.Adapters)
    h.k, h.ns, h.ctx = 8, [6, 4], object()
    a, b = [np.zeros((2, 8))] * 2, [np.zeros((6, 2)), np.zeros((4, 2))]
    for x, y in ((a[:1], b), (a, b[:1]), (a, b[::-1]), ([a[0], a[0][:1]], b), (a[0], b[0]), ([a[0][:0]] * 2, b)):
        with pytest.raises(ArgumentError):
            h.set(0, x, y)
    with pytest.raises(ArgumentError):
        h._pointers([P])
    good = dict(x=np.zeros((3, 8)), slots=[0, 1, 2], bases=[np.zeros((3, 6)), np.zeros((3, 4))])
    for bad in (dict(x=np.zeros((3, 7))), dict(slots=[0, 1]), dict(bases=[np.zeros((3, 6))])):
        with pytest.raises(ArgumentError):
            h.apply(**{**good, **bad})


# ------------------------------------------------------- the tests' references


def test_reference_emits_the_target_distribution():
    # Averaged over a fine grid of random numbers and over the drafted token, the first emitted token has
    # the target's distribution (to the grid's steps), with and without the draft's.
    rng = np.random.default_rng(0)
    v, n = 4, 300
    t, q = rng.standard_normal((2, 1, v)).astype(np.float32)
    p, w = R.weights(t[0], 1.0), R.weights(q[0], 1.0)
    grid = (np.arange(n) + 0.5) / n
    for draft in (np.tile(q, (2, 1)), None):
        share = np.zeros(v)
        for x in range(v):
            for u in grid:
                for u0 in grid[::10]:
                    out, _, count = R.verify(np.tile(t, (2, 1)), [0, x], [u0, u], [0, 2], draft=draft)
                    share[out[0]] += w[x] / n / (n / 10)
                    if count[0] == 2:  # (it does not depend on u0)
                        share[out[0]] += w[x] / n / (n / 10) * (n / 10 - 1)
                        break
        assert np.abs(share - p).max() < 2 * v / (n / 10)


def test_reference_of_trees_and_greedy():
    x = np.zeros((4, 3), np.float32)
    x[0] = [0, 0, -np.inf]
    # Two children of the root: token 0 is rejected at 1/2, then token 1 has all that is left.
    out, kept, count = R.verify(x, [9, 0, 1, 2], [0.9, 0.5, 0.99, 0.99], [0, 4], parent=[-1, 0, 0, 2])
    assert list(kept) == [0, 2, -1, -1] and count[0] == 2 and list(out) == [1, 1, -1, -1]
    out, kept, count = R.verify(x, [9, 0, 1, 2], [0.0, 0.49, 0, 0], [0, 4], parent=[-1, 0, 0, 1])
    assert list(kept) == [0, 1, 3, -1] and list(out) == [0, 2, 0, -1]
    out, kept, count = R.verify(x, [9, 1, 0, 0], [0.0, 0, 0, 0], [0, 4], parent=[-1, 0, 0, 2], temperature=[0])
    assert list(kept) == [0, 2, 3, -1] and list(out) == [0, 0, 0, -1]


def test_reference_of_pages():
    table = np.array([[3, 1, -1], [0, -1, -1]], np.int32)
    refs = np.array([1, 1, 0, 1, 0], np.int32)
    past, new, refs, bad = PR.fork([0, 0, -1], [20, 9], table, refs, 3, 16, 20)
    assert past.tolist() == [20, 20, 0] and new.tolist() == [[3, 1, -1], [3, 1, -1], [-1] * 3] and not bad
    assert refs.tolist() == [0, 2, 0, 2, 0]
    table, refs, granted, moves, bad = PR.fit([1, 13, 2], past, new, refs, 16)
    # The first gets a copy of page 1, the second keeps it and takes a new one, the third starts.
    assert table.tolist() == [[3, 0, -1], [3, 1, 2], [4, -1, -1]] and moves == [(1, 0)]
    assert refs.tolist() == [1, 1, 1, 2, 1] and granted.tolist() == [1, 1, 1] and not bad
    assert PR.copied([0, 1, 4], [1, 2, 4], 5) == ([], True)
    assert PR.copied([0, 3], [1, 2], 5) == ([(0, 1), (3, 2)], False)
