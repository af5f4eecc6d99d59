"""Low-rank adapters of many requests against 64 bits: few and many rows, ranks, formats, odd
sizes, rows without an adapter, slots that are filled anew, captured graphs."""
import numpy as np
import pytest

from hip_graph import Captured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def adapters(ops, rng, k, ns, slots, max_rank, fmt="f32", ranks=None, ctx=None):
    """A handle, and its slots' values as they are held: [(a, b, scale)], None for empty ones."""
    h = ops.Adapters(k, ns, slots=slots, max_rank=max_rank, fmt=fmt, ctx=ctx)
    held = []
    for s in range(slots):
        r = int(rng.integers(0, max_rank + 1)) if ranks is None else ranks[s % len(ranks)]
        held.append(fill(h, rng, s, r, fmt))
    return h, held


def fill(h, rng, slot, rank, fmt):
    if rank == 0:
        h.set(slot, None, None)
        return None
    a = [(rng.standard_normal((rank, h.k)) / np.sqrt(h.k)).astype(np.float32) for _ in h.ns]
    b = [rng.standard_normal((n, rank)).astype(np.float32) for n in h.ns]
    scale = float(np.float32(rng.uniform(0.1, 2)))
    h.set(slot, a, b, scale=scale)
    if fmt == "f16":
        a, b = ([x.astype(np.float16).astype(np.float32) for x in y] for y in (a, b))
    return a, b, scale


def expected(x, slots, bases, held):
    """In 64 bits, and how far fp32 may be off: a sum of K products runs through chains of at most
    K / 4 of them and 16 joins (each rounding off by 2^-24 of the magnitudes so far), the
    second product adds chains of r and the factor, the base one more."""
    out, off = [], []
    for i, base in enumerate(bases):
        y, e = base.astype(np.float64), np.zeros(base.shape)
        for r, s in enumerate(slots):
            if s >= len(held):
                y[r] = np.nan
            elif s >= 0 and held[s] is not None:
                a, b, f = held[s][0][i].astype(np.float64), held[s][1][i].astype(np.float64), held[s][2]
                v = x[r].astype(np.float64)
                y[r] += f * (b @ (a @ v))
                e[r] = (x.shape[1] / 4 + a.shape[0] + 20) * 2.0**-24 * abs(f) * (np.abs(b) @ (np.abs(a) @ np.abs(v)))
                e[r] += 2.0**-23 * np.abs(y[r])
        out.append(y)
        off.append(e)
    return out, off


def check(got, x, slots, bases, held):
    for g, w, e in zip(got, *expected(x, slots, bases, held)):
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        assert (np.abs(g - w) <= e + 1e-300)[~np.isnan(w)].all(), np.nanmax(np.abs(g - w) / (e + 1e-30))


def inputs(rng, h, rows):
    return (rng.standard_normal((rows, h.k)).astype(np.float32),
            [rng.standard_normal((rows, n)).astype(np.float32) for n in h.ns])


@pytest.mark.parametrize("fmt", ["f32", "f16"])
@pytest.mark.parametrize("k, ns, max_rank", [(1, [1], 1), (7, [5, 9], 3), (64, [64], 8), (130, [33, 100, 7], 16),
                                             (1024, [256, 130], 33), (515, [513], 64), (96, [40], 256)])
@pytest.mark.parametrize("rows", [1, 3, 160, 512, 513, 700])
def test_sizes(ops, fmt, k, ns, max_rank, rows):
    rng = np.random.default_rng(k + rows)
    h, held = adapters(ops, rng, k, ns, 6, max_rank, fmt)
    x, bases = inputs(rng, h, rows)
    slots = rng.integers(-1, 7, rows)  # (6: beyond the handle)
    check(h.apply(x, slots, bases), x, slots, bases, held)


@pytest.mark.parametrize("rows", [40, 65, 513, 575, 576, 577, 640, 1025])
def test_prompts_and_tokens(ops, rows):
    # Runs of one slot, single rows between, all rows of one slot, none.
    rng = np.random.default_rng(rows)
    h, held = adapters(ops, rng, 200, [300, 70], 12, 16)
    x, bases = inputs(rng, h, rows)
    for slots in (np.sort(rng.integers(-1, 12, rows)), rng.integers(0, 12, rows), np.full(rows, 5),
                  np.full(rows, -1), np.where(np.arange(rows) % 64 == 63, 3, 7), np.full(rows, 12)):
        check(h.apply(x, slots, bases), x, slots, bases, held)


@pytest.mark.parametrize("k, ns, rank, rows", [(2048, [2048], 59, 490), (2048, [2048], 61, 490),
                                               (4096, [5000, 5000], 128, 60)])
def test_wide_adapters(ops, k, ns, rank, rows):
    # Few rows of many multiply-adds: on both sides of where they are sorted.
    rng = np.random.default_rng(rank)
    h, held = adapters(ops, rng, k, ns, 3, rank, ranks=[rank, rank - 1, 1])
    x, bases = inputs(rng, h, rows)
    slots = rng.integers(-1, 3, rows)
    check(h.apply(x, slots, bases), x, slots, bases, held)


def test_many_slots(ops):
    rng = np.random.default_rng(1)
    h, held = adapters(ops, rng, 40, [24], 4096, 2)
    for rows in (90, 5000):
        x, bases = inputs(rng, h, rows)
        slots = rng.integers(-1, 4097, rows)
        check(h.apply(x, slots, bases), x, slots, bases, held)
    # Each row a slot of its own: as many tiles as rows.
    x, bases = inputs(rng, h, 4096)
    slots = rng.permutation(4096)
    check(h.apply(x, slots, bases), x, slots, bases, held)


def test_rounds_of_rows(ops):
    rng = np.random.default_rng(2)
    h, held = adapters(ops, rng, 8, [8], 3, 2, ranks=[2, 1, 0])
    rows = 2 * 65536 + 50
    x, bases = inputs(rng, h, rows)
    slots = rng.integers(-1, 4, rows)
    got = h.apply(x, slots, bases)[0]
    at = np.r_[np.arange(300), np.arange(65400, 65700), np.arange(131000, rows)]
    check([got[at]], x[at], slots[at], [bases[0][at]], held)
    none = (slots == -1) | (slots == 2)
    np.testing.assert_array_equal(got[none], bases[0][none])


@pytest.mark.parametrize("rows", [5, 600])
def test_rows_without_an_adapter_are_the_base(ops, rows):
    rng = np.random.default_rng(3)
    h, held = adapters(ops, rng, 64, [100], 2, 4, ranks=[4, 0])
    x, bases = inputs(rng, h, rows)
    bases[0][:, :4] = [-0.0, np.inf, np.nan, 1e-42]
    x[:] = np.nan
    slots = np.where(np.arange(rows) % 3 == 0, 0, np.where(np.arange(rows) % 3 == 1, 1, -5))
    got = h.apply(x, slots, bases)[0]
    none = slots != 0
    np.testing.assert_array_equal(got[none].view(np.int32), bases[0][none].view(np.int32))
    assert np.isnan(got[~none]).all()


@pytest.mark.parametrize("rows", [7, 520])
def test_values_that_are_not_finite_stay_with_their_rows(ops, rows):
    rng = np.random.default_rng(4)
    h, held = adapters(ops, rng, 50, [40], 3, 5, ranks=[5, 3, 4])
    x, bases = inputs(rng, h, rows)
    slots = np.arange(rows) % 3
    want = h.apply(x, slots, bases)[0]
    x[4, 20], x[5, 3] = np.nan, np.inf
    got = h.apply(x, slots, bases)[0]
    rest = np.setdiff1d(np.arange(rows), [4, 5])
    np.testing.assert_array_equal(got[rest], want[rest])
    assert np.isnan(got[4]).all() and not np.isfinite(got[5]).any()
    # A slot that holds Infinity: only its rows.
    a = [np.full((5, 50), np.inf, np.float32)]
    h.set(0, a, [held[0][1][0]])
    got = h.apply(x, slots, bases)[0]
    rest = rest[slots[rest] != 0]
    np.testing.assert_array_equal(got[rest], want[rest])


@pytest.mark.parametrize("fmt", ["f32", "f16"])
@pytest.mark.parametrize("rows", [9, 550])
def test_slots_filled_anew(ops, fmt, rows):
    # Of larger and smaller ranks than before, Infinity among what is left behind.
    rng = np.random.default_rng(5)
    h = ops.Adapters(72, [56, 8], slots=2, max_rank=9, fmt=fmt)
    x, bases = inputs(rng, h, rows)
    slots = np.arange(rows) % 2
    held = [None, None]
    check(h.apply(x, slots, bases), x, slots, bases, held)
    for rank in (9, 3, 0, 1, 8, 2):
        bad = [np.full((9, 72), np.inf, np.float32)] * 2, [np.full((n, 9), np.nan, np.float32) for n in (56, 8)]
        h.set(0, *bad)
        held = [fill(h, rng, 0, rank, fmt), held[1]]
        check(h.apply(x, slots, bases), x, slots, bases, held)
        held[1] = fill(h, rng, 1, 9 - rank, fmt)
        check(h.apply(x, slots, bases), x, slots, bases, held)


def test_rounding_to_fp16(ops):
    # Ties to even, the smallest numbers, and those beyond the range.
    h = ops.Adapters(1, [6], slots=1, max_rank=1, fmt="f16")
    b = np.array([[1 + 2.0**-11], [1 + 3 * 2.0**-11], [65519.0], [65520.0], [2.0**-25], [1.5 * 2.0**-24]], np.float32)
    h.set(0, np.ones((1, 1), np.float32), b)
    got = h.apply(np.ones((1, 1), np.float32), [0], [np.zeros((1, 6), np.float32)])[0]
    np.testing.assert_array_equal(got[0], [1, 1 + 2.0**-9, 65504, np.inf, 0, 2.0**-23])


@pytest.mark.parametrize("rows", [6, 600])
def test_device_calls(ops, rows):
    # In place, apart, from device weights, at odd addresses, rows behind left alone.
    rng = np.random.default_rng(6)
    h, held = adapters(ops, rng, 77, [51, 64], 3, 6, ranks=[6, 2, 5])
    x, bases = inputs(rng, h, rows)
    slots = rng.integers(-1, 3, rows)
    for name, shift in (("a", 0), ("b", 1)):
        dev = [ops.DeviceBuffer.from_array(np.r_[np.zeros(shift, np.float32), v.ravel(), np.full(5, 7, np.float32)])
               for v in [x] + bases]
        outs = [ops.DeviceBuffer.from_array(np.full(shift + v.size + 5, 7, np.float32)) for v in bases]
        s = ops.DeviceBuffer.from_array(slots.astype(np.int32))
        for ys in (outs, dev[1:]):
            h.apply_dev(dev[0].ptr + 4 * shift, rows, s.ptr, [d.ptr + 4 * shift for d in dev[1:]],
                        [y.ptr + 4 * shift for y in ys])
            got = [y.to_array((shift + v.size + 5,), np.float32) for y, v in zip(ys, bases)]
            for g in got:
                assert (g[-5:] == 7).all()
            check([g[shift:-5].reshape(v.shape) for g, v in zip(got, bases)], x, slots, bases, held)
    a, b = ([rng.standard_normal(sh).astype(np.float32) for sh in shs]
            for shs in ([(4, 77)] * 2, [(51, 4), (64, 4)]))
    dev = [[ops.DeviceBuffer.from_array(v) for v in y] for y in (a, b)]
    h.set_dev(1, 4, [d.ptr for d in dev[0]], [d.ptr for d in dev[1]], scale=-0.5)
    h.ctx.synchronize()
    held[1] = a, b, -0.5
    check(h.apply(x, slots, bases), x, slots, bases, held)


@pytest.mark.parametrize("rows", [12, 1560])
def test_captured_graph(ops, rows):
    # Slots, rows' slots and inputs change between replays; another graph shares the workspace.
    rng = np.random.default_rng(7)
    with Captured(ops) as g:
        h, held = adapters(ops, rng, 64, [48], 4, 8, ranks=[8, 1, 0, 5], ctx=g.ctx)
        x, base = (g.buffer(np.zeros((rows, n), np.float32)) for n in (64, 48))
        slot = g.buffer(np.zeros(rows, np.int32))
        ys = [g.buffer(np.zeros((rows, 48), np.float32)) for _ in range(2)]

        def call(n, y):
            h.apply_dev(x.ptr, n, slot.ptr, [base.ptr], [y.ptr])

        n = rows // 3
        call(rows, ys[0])
        graphs = [g.capture(lambda: call(rows, ys[0])), g.capture(lambda: call(n, ys[1]))]
        for step in range(4):
            xs, bases = inputs(rng, h, rows)
            slots = rng.integers(-1, 5, rows)
            held[step] = fill(h, rng, step, int(rng.integers(0, 9)), "f32")
            zeros = np.zeros((rows, 48), np.float32)
            for t, v in ((x, xs), (base, bases[0]), (slot, slots.astype(np.int32)), (ys[1], zeros)):
                g.put(t, v)
            for replay in graphs:
                replay()
            g.wait()
            got = [y.to_array((rows, 48), np.float32) for y in ys]
            check([got[0]], xs, slots, bases, held)
            check([got[1][:n]], xs[:n], slots[:n], [bases[0][:n]], held)
            assert (got[1][n:] == 0).all()
        h.release()


def test_host_weights_are_refused_under_capture(ops):
    from onnx_runtime_dart_amd.errors import UnsupportedError
    rng = np.random.default_rng(9)
    with Captured(ops) as g:
        h, held = adapters(ops, rng, 16, [8], 2, 4, ranks=[4, 2], ctx=g.ctx)
        x, bases = inputs(rng, h, 5)
        slots = np.array([0, 1, -1, 1, 0], np.int32)
        d = [g.buffer(v) for v in (x, slots, bases[0], np.zeros((5, 8), np.float32))]

        def call():
            with pytest.raises(UnsupportedError):
                h.set(0, [np.ones((4, 16), np.float32)], [np.ones((8, 4), np.float32)])
            h.apply_dev(d[0].ptr, 5, d[1].ptr, [d[2].ptr], [d[3].ptr])

        h.apply_dev(d[0].ptr, 5, d[1].ptr, [d[2].ptr], [d[3].ptr])
        g.capture(call)()
        g.wait()
        check([d[3].to_array((5, 8), np.float32)], x, slots, bases, held)
        h.release()


def test_beside_a_shared_projection(ops):
    # int4 q and v projections of all requests, their adapters added in place.
    rng = np.random.default_rng(8)
    k, ns = 256, [128, 64]
    ws = []
    for n in ns:
        q = rng.integers(0, 256, (n, k // 32, 16), dtype=np.uint8)
        ws.append(ops.NBitsWeight(q, rng.uniform(0.002, 0.02, (n, k // 32)).astype(np.float32), k=k, n=n,
                                  block_size=32))
    h, held = adapters(ops, rng, k, ns, 5, 8)
    for rows in (4, 530):
        x = rng.standard_normal((rows, k)).astype(np.float32)
        slots = rng.integers(-1, 5, rows)
        shared = [w(x) for w in ws]
        dx, ds = ops.DeviceBuffer.from_array(x), ops.DeviceBuffer.from_array(slots.astype(np.int32))
        ys = [ops.DeviceBuffer(4 * rows * n) for n in ns]
        ops.matmul_nbits_group_dev(ws, dx.ptr, rows, [y.ptr for y in ys])
        h.apply_dev(dx.ptr, rows, ds.ptr, [y.ptr for y in ys], [y.ptr for y in ys])
        got = [y.to_array((rows, n), np.float32) for y, n in zip(ys, ns)]
        # (The group's results are those of separate calls.)
        check(got, x, slots, shared, held)


@pytest.mark.parametrize("rows", [20, 800])
def test_repeated_calls_are_equal(ops, rows):
    rng = np.random.default_rng(9)
    h, held = adapters(ops, rng, 300, [200], 7, 16)
    x, bases = inputs(rng, h, rows)
    slots = rng.integers(-1, 7, rows)
    first = h.apply(x, slots, bases)[0]
    for _ in range(4):
        np.testing.assert_array_equal(h.apply(x, slots, bases)[0], first)
