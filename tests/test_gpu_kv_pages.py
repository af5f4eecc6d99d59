"""Pages of the quantised KV cache: copies, rows that move together, shared and free pages,
against plain numpy; what a cache reads back is compared bit for bit."""
import numpy as np
import pytest

import kv_reference as K
import pages_reference as P
from hip_graph import Captured

pytestmark = pytest.mark.gpu
FORMATS = ("int8", "e4m3", "int4")


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


class Cache:
    """A cache whose every place has been written, and what it reads back [pages * page, ...]."""

    def __init__(self, ops, rng, pages, page, fmt="int8", heads=2, d=64, ctx=None):
        self.c = ops.KvCache(pages, kv_heads=heads, head_size=d, page_size=page, fmt=fmt, ctx=ctx)
        self.pages, self.page = pages, page
        k, v = rng.standard_normal((2, pages * page, heads, d)).astype(np.float32)
        self.c.append(k, v, **self.where())
        self.now = self.read()
        for got, x in zip(self.now, (k, v)):
            np.testing.assert_array_equal(got, K.cached(x, fmt))

    def where(self):
        n = self.pages
        return dict(row_start=np.arange(n + 1) * self.page, past=np.zeros(n, np.int32),
                    page_table=np.arange(n).reshape(n, 1))

    def read(self):
        return self.c.read(self.pages * self.page, **self.where())

    def check(self, free=()):
        """The cache holds what is expected (rows in free: anything finite)."""
        for got, want in zip(self.read(), self.now):
            assert np.isfinite(got).all()
            want = want.copy()
            want[list(free)] = got[list(free)]
            np.testing.assert_array_equal(got, want)


# -------------------------------------------------------------------- copies


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page, heads, d", [(16, 1, 1), (16, 3, 80), (64, 2, 128), (256, 1, 256), (32, 5, 192)])
def test_copies(ops, fmt, page, heads, d):
    rng = np.random.default_rng(page + d)
    c = Cache(ops, rng, 9, page, fmt, heads, d)
    src, dst = np.array([0, 3, 0, -1, 5, 7]), np.array([1, 2, 8, -1, 5, 4])
    c.c.copy_pages(src, dst)
    for x in c.now:
        x = x.reshape((9, page) + x.shape[1:])
        x[[1, 2, 8, 4]] = x[[0, 3, 0, 7]]
    c.check()
    assert not c.c.refused()


BAD = [([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0, 9], [1, 2]), ([0, 1], [9, 2]), ([-1, 1], [0, 2]),
       ([0, 1], [-1, 2]), ([0, 0, 3], [1, 1, 4]), ([3, 1, 2], [3, 3, 0]), ([0, 1], [1, 0]),
       ([2**31 - 1, 1], [3, 2]), ([4, 4, 4], [5, 5, 4])]


@pytest.mark.parametrize("src, dst", BAD, ids=str)
@pytest.mark.parametrize("many", [False, True])
def test_pairs_that_are_refused(ops, src, dst, many):
    c = Cache(ops, np.random.default_rng(1), 7, 16)
    if many:  # behind a thousand that are passed over
        src, dst = np.r_[np.full(1030, -1), src], np.r_[np.full(1030, -1), dst]
    done, refused = P.copied(src, dst, 7)
    assert refused
    c.c.copy_pages(src, dst)
    for x in c.now:
        x = x.reshape((7, 16) + x.shape[1:])
        for s, t in done:
            x[t] = x[s]
    c.check()
    assert c.c.refused() and not c.c.refused()


def test_long_lists(ops):
    rng = np.random.default_rng(2)
    c = Cache(ops, rng, 3000, 16, heads=1)
    order = rng.permutation(3000)
    src, dst = order[:1400], order[1400:2800]
    c.c.copy_pages(src, dst)
    for x in c.now:
        x = x.reshape((3000, 16) + x.shape[1:])
        x[dst] = x[src]
    c.check()
    assert not c.c.refused()


# ------------------------------------------------------------------- compact


def moved(c, b, kept, counts):
    """c.now with the rows that stay moved together; returns the places behind them."""
    free, at = [], 0
    for i, (n, past) in enumerate(zip(b.new, b.past)):
        slot = [int(b.page_table[i, p // c.page]) * c.page + p % c.page for p in range(past, past + n)]
        keep = kept[at:at + counts[i]]
        for x in c.now:
            x[slot[:len(keep)]] = x[[slot[k] for k in keep]]
        free += slot[len(keep):]
        at += n
    return free


def lists(rng, new, share=0.5):
    kept, counts = [], []
    for n in new:
        keep = np.nonzero(rng.random(n) < share)[0]
        kept += list(keep) + [-1] * (n - keep.size)
        counts.append(keep.size)
    return np.array(kept, np.int32), np.array(counts, np.int32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page, heads, d", [(16, 1, 1), (16, 3, 80), (64, 2, 128), (256, 1, 256), (32, 4, 192)])
@pytest.mark.parametrize("share", [0.0, 0.2, 0.6, 1.0])
def test_compact(ops, fmt, page, heads, d, share):
    rng = np.random.default_rng(page + d + int(10 * share))
    new, past = [25, 1, 0, 7, 64, 130, 300], [33, 0, 5, 14, 61, 2, 100]
    b = K.Batch(rng, new, past, page)
    c = Cache(ops, rng, b.pages, page, fmt, heads, d)
    kept, counts = lists(rng, new, share)
    got = c.c.compact(kept, counts, **b.args())
    np.testing.assert_array_equal(got, b.past + counts)
    c.check(moved(c, b, kept, counts))
    assert not c.c.refused()


@pytest.mark.parametrize("fmt", FORMATS)
def test_compact_long(ops, fmt):
    rng = np.random.default_rng(3)
    b = K.Batch(rng, [3001, 4000], [7, 0], 64)
    c = Cache(ops, rng, b.pages, 64, fmt, 1, 64)
    for share in (0.5, 0.97):
        kept, counts = lists(rng, b.new, share)
        c.c.compact(kept, counts, **b.args())
        c.check(moved(c, b, kept, counts))
        c.now = c.read()


@pytest.mark.parametrize("budget", [False, True])
def test_compact_long_in_place(ops, budget):
    # The new lengths over the old ones; without room for a workspace rows move in order.  The graph
    # is captured before the context has any workspace, then again after a call.
    rng = np.random.default_rng(28)
    with Captured(ops) as g:
        c = Cache(ops, rng, 40, 64, "int8", 2, 48, ctx=g.ctx)
        past = np.array([70, 0], np.int32)
        kept, counts = lists(rng, [700, 901], 0.6)
        table = rng.permutation(40)[:32].reshape(2, 16).astype(np.int32)
        d = [g.buffer(v) for v in (np.array([0, 700, 1601], np.int32), past, table, kept, counts)]
        s = ops.SeqBatch(batch=2, rows=1601, max_new=901, max_len=1024, row_start_ptr=d[0].ptr,
                         past_ptr=d[1].ptr, page_table_ptr=d[2].ptr, table_stride=16)

        def step():
            g.ctx.set_control(max_bytes=1000 if budget else -1)
            c.c.compact_dev(s, d[3].ptr, d[4].ptr, past_out_ptr=d[1].ptr)
            g.ctx.set_control(max_bytes=-1)

        for call in (g.capture(step), step, None):
            call = call or g.capture(step)
            for _ in range(3):
                b = K.Batch(rng, [700, 901], past, 64)
                b.page_table = table
                call()
                g.wait()
                free = moved(c, b, kept, counts)
                np.testing.assert_array_equal(d[1].to_array((2,), np.int32), past + counts)
                c.check(free)
                c.now = c.read()
                g.put(d[1], past)
                assert not c.c.refused()
        c.c.release()


def test_compact_without_moves_writes_nothing(ops):
    rng = np.random.default_rng(4)
    b = K.Batch(rng, [20, 30], [3, 50], 16)
    c = Cache(ops, rng, b.pages, 16)
    kept = np.r_[np.arange(20), np.arange(30)]
    c.c.compact(kept, [20, 11], **b.args())
    c.check()
    kept[:20], kept[20:] = np.r_[0, 19, np.full(18, -1)], np.r_[29, np.full(29, -1)]
    c.c.compact(kept, [2, 1], **b.args())  # the last row to the second and to the first place
    c.check(moved(c, b, kept, [2, 1]))


@pytest.mark.parametrize("kept, count", [([1, 1, 2], 3), ([2, 1, 0], 2), ([0, 3, 2], 2), ([-1, 1, 2], 2),
                                         ([0, 1, 2], 4), ([0, 1, 2], -1), ([0, 2, 2**30], 3)])
def test_lists_that_are_refused(ops, kept, count):
    rng = np.random.default_rng(5)
    b = K.Batch(rng, [3, 3], [20, 9], 16)
    c = Cache(ops, rng, b.pages, 16)
    got = c.c.compact(np.r_[kept, 1, 2, -1], [count, 2], **b.args())
    np.testing.assert_array_equal(got, b.past + [0, 2])
    good = np.r_[np.arange(3), 1, 2, -1]
    c.check(moved(c, b, good, [3, 2]))
    assert c.c.refused()


def test_compact_across_missing_pages(ops):
    # Rows from or to a page that is not there stay where they are, the others move.
    rng = np.random.default_rng(6)
    b = K.Batch(rng, [60], [4], 16)
    c = Cache(ops, rng, b.pages, 16)
    b.page_table[0, 2] = c.pages + 5
    kept = np.r_[np.arange(10, 60), np.full(10, -1)]
    before = [x.copy() for x in c.now]
    c.c.compact(kept, [50], **b.args())
    table = b.page_table[0]
    for x, old in zip(c.now, before):
        for j in range(50):
            to, at = 4 + j, 4 + 10 + j
            if to // 16 != 2 and at // 16 != 2:
                x[table[to // 16] * 16 + to % 16] = old[table[at // 16] * 16 + at % 16]
    free = [int(table[p // 16]) * 16 + p % 16 for p in range(54, 64)]
    c.check(free)
    assert c.c.refused()


# ---------------------------------------------------------- shared and free pages


def holdings(rng, past, page, pages, width):
    """A table of pages of their own, and refs."""
    need = [-(-int(p) // page) for p in past]
    order = rng.permutation(pages)
    table, refs, at = np.full((len(past), width), -1, np.int32), np.zeros(pages, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        refs[order[at:at + n]] += 1
        at += n
    return table, refs


@pytest.mark.parametrize("seed", range(12))
def test_fork_and_fit(ops, seed):
    rng = np.random.default_rng(seed)
    page, n, kids = 16, int(rng.integers(1, 9)), int(rng.integers(1, 20))
    past = rng.integers(0, 90, n)
    used = int((-(-past // page)).sum())
    c = Cache(ops, rng, used + int(rng.integers(1, 40)), page, FORMATS[seed % 3], 1)
    table, refs = holdings(rng, past, page, c.pages, 8)
    parent = rng.integers(-1, n, kids)
    got = c.c.fork(parent, past=past, page_table=table, refs=refs, width=9)
    want = P.fork(parent, past, table, refs, 9, page, past.max())
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    past, table, refs, _ = want
    for step in range(3):
        new = rng.integers(0, 30, kids) * (rng.random(kids) < 0.8)
        new = np.minimum(new, 9 * page - past)
        start = np.r_[0, np.cumsum(new)]
        got = c.c.fit(row_start=start, past=past, page_table=table, refs=refs)
        table, refs, granted, moves, refused = P.fit(new, past, table, refs, page)
        for g, w in zip(got, (table, refs, granted)):
            np.testing.assert_array_equal(g, w)
        for x in c.now:
            x = x.reshape((c.pages, page) + x.shape[1:])
            old = x.copy()
            for s, t in moves:
                x[t] = old[s]
        c.check()
        assert c.c.refused() == refused
        held, counts = np.unique(table[table >= 0], return_counts=True)
        np.testing.assert_array_equal(refs[held], counts)
        # Whoever may write does so alone.
        for i in np.nonzero(granted * (new > 0))[0]:
            assert (refs[table[i, past[i] // page:-(-(past[i] + new[i]) // page)]] == 1).all()
        past = np.where(granted > 0, np.maximum(past + rng.integers(-40, 1, kids) + new, 0), past)
        past = np.minimum(past, (table >= 0).sum(1) * page).astype(np.int32)


def test_freeing_sequences(ops):
    rng = np.random.default_rng(20)
    c = Cache(ops, rng, 40, 16)
    past = np.array([100, 3, 64])
    table, refs = holdings(rng, past, 16, 40, 8)
    got = c.c.fit(row_start=[0, 0, 0, 0], past=[0, 3, 0], page_table=table, refs=refs)
    assert (got[0][[0, 2]] == -1).all() and got[1].sum() == 1 and (got[2] == 1).all()
    past, table, refs = c.c.fork([-1, -1], past=past, page_table=table, refs=refs)
    assert (past == 0).all() and (table == -1).all() and (refs == 0).all()


def test_forks_from_and_to_nothing(ops):
    rng = np.random.default_rng(29)
    c = Cache(ops, rng, 20, 16)
    past = np.array([40, 0, 17])
    table, refs = holdings(rng, past, 16, 20, 4)
    got = c.c.fork([-1, -1, 0], past=[], page_table=np.zeros((0, 4)), refs=refs, width=2)
    assert (got[0] == 0).all() and (got[1] == -1).all()
    np.testing.assert_array_equal(got[2], refs)
    assert c.c.refused()  # (the third: there is no such parent)
    got = c.c.fork([], past=past, page_table=table, refs=refs)
    assert got[0].size == 0 and (got[2] == 0).all() and not c.c.refused()


@pytest.mark.parametrize("n", [900, 1500])
def test_many_pages_and_sequences(ops, n):
    # More pages than one run of the search for free ones; sequences of one workgroup and of many.
    rng = np.random.default_rng(21)
    page = 16
    c = Cache(ops, rng, 10000, page, heads=1, d=1)
    past = rng.integers(0, 60, n)
    table, refs = holdings(rng, past, page, c.pages, 6)
    parent = rng.integers(0, n, n)
    past, table, refs, _ = P.fork(parent, past, table, refs, 6, page, 60)
    new = rng.integers(0, 30, n)
    got = c.c.fit(row_start=np.r_[0, np.cumsum(new)], past=past, page_table=table, refs=refs)
    want = P.fit(new, past, table, refs, page)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    assert len(want[3]) > n // 5


def test_tables_that_are_refused(ops):
    rng = np.random.default_rng(22)
    c = Cache(ops, rng, 20, 16)
    past = np.array([40, 40, 40, 40, 40, 16])
    table, refs = holdings(rng, past, 16, 20, 5)
    table[0, 1] = -1             # a page of the past is missing
    table[1, 2] = 20             # no page of this cache
    table[2, 4] = table[2, 0]    # behind a gap
    new = np.array([1, 1, 30, 60, 1, 1])  # (the fourth has too short a table)
    got = c.c.fit(row_start=np.r_[0, np.cumsum(new)], past=past, page_table=table, refs=refs)
    want = P.fit(new, past, table, refs, 16)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    assert want[4] and (want[2] == [0, 0, 0, 0, 1, 1]).all() and c.c.refused()
    # Forks of sequences that are not there, or do not fit.
    past[1] = 100
    parent = [6, 2**31 - 1, 1, 0, 5]
    got = c.c.fork(parent, past=past, page_table=table, refs=refs, width=2)
    want = P.fork(parent, past, table, refs, 2, 16, 100)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    assert c.c.refused()


def test_a_shared_page_waits_for_all_that_share_it(ops):
    # Two share a page that both write into; the first gets no copy, so the second may not write.
    c = Cache(ops, np.random.default_rng(23), 2, 16)
    table = np.array([[0, -1], [0, -1], [1, -1]], np.int32)
    refs = np.array([2, 1], np.int32)
    got = c.c.fit(row_start=[0, 1, 2, 3], past=[5, 5, 5], page_table=table, refs=refs)
    np.testing.assert_array_equal(got[2], [0, 0, 1])
    np.testing.assert_array_equal(got[0], table)
    np.testing.assert_array_equal(got[1], refs)


@pytest.mark.parametrize("width", [101, 2800])  # (one workgroup, many)
def test_the_last_to_share_a_page_waits_in_the_order(ops, width):
    # A and C write into page 0; A gets its copy, so that C could keep page 0, but B between them asks for
    # more than there is: nobody behind B is served who needs a page or keeps a shared one.  D needs
    # and shares none.  The next call finds page 0 C's own.
    c = Cache(ops, np.random.default_rng(30), 4, 16, heads=1)
    table = np.full((4, width), -1, np.int32)
    table[[0, 2, 3], 0] = [0, 0, 3]
    refs, past = np.array([2, 0, 0, 1], np.int32), np.array([5, 0, 5, 7], np.int32)
    new = np.array([1, 1600, 1, 1])
    for granted, held in (([1, 0, 0, 1], [1, -1, 0, 3]), ([1, 0, 1, 1], [1, -1, 0, 3])):
        want = P.fit(new, past, table, refs, 16)
        table, refs, got = c.c.fit(row_start=np.r_[0, np.cumsum(new)], past=past, page_table=table, refs=refs)
        np.testing.assert_array_equal(got, granted)
        np.testing.assert_array_equal(table[:, 0], held)
        np.testing.assert_array_equal(refs, [1, 1, 0, 1])
        assert (table[:, 1:] == -1).all()
        for g, w in zip((table, refs, got), want):
            np.testing.assert_array_equal(g, w)
    for x in c.now:
        x[16:32] = x[:16]
    c.check()
    assert not c.c.refused()


def test_captured_graph(ops):
    # A step that fits its sequences and moves rows: tables, lengths and refs change on the device.
    rng = np.random.default_rng(24)
    with Captured(ops) as g:
        c = Cache(ops, rng, 50, 16, ctx=g.ctx)
        past = np.array([30, 30, 15, 0], np.int32)
        table, refs = holdings(rng, past, 16, 50, 6)
        refs[table[1][:2]] = 0
        table[1], refs[table[0][:2]] = table[0], 2
        new = np.array([2, 2, 3, 9])
        kept = np.array([1, -1, 0, 1, 0, 2, -1, 1, 2, 3, 4, 5, 6, 7, 8, -1], np.int32)
        counts = np.array([1, 2, 2, 8], np.int32)
        d = {k: g.buffer(np.ascontiguousarray(v, np.int32)) for k, v in dict(
            start=np.r_[0, np.cumsum(new)], past=past, table=table, refs=refs, granted=np.zeros(4), kept=kept,
            count=counts).items()}
        s = ops.SeqBatch(batch=4, rows=16, max_new=9, max_len=96, row_start_ptr=d["start"].ptr,
                         past_ptr=d["past"].ptr, page_table_ptr=d["table"].ptr, table_stride=6)

        def step():
            c.c.fit_dev(s, d["refs"].ptr, d["granted"].ptr)
            c.c.compact_dev(s, d["kept"].ptr, d["count"].ptr, past_out_ptr=d["past"].ptr)

        step()
        replay = g.capture(step)
        for _ in range(5):
            g.wait()
            table, refs, granted, moves, refused = P.fit(new, past, table, refs, 16)
            for x in c.now:
                pages = x.reshape((50, 16) + x.shape[1:])
                old = pages.copy()
                for a, t in moves:
                    pages[t] = old[a]
            b = K.Batch(rng, new, past, 16)
            b.page_table = table
            free = moved(c, b, kept, counts)
            past = (past + counts).astype(np.int32)
            for k, w in (("table", table), ("refs", refs), ("granted", granted), ("past", past)):
                np.testing.assert_array_equal(d[k].to_array(w.shape, np.int32), w)
            c.check(free)
            c.now = c.read()
            assert not refused and not c.c.refused()
            replay()
        g.wait()
        c.c.release()
