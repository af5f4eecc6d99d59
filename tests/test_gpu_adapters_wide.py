"""Low-rank adapters where the second product takes ranks in rounds or many outputs a workgroup, and
where rounds of rows split K each in their own way, against 64 bits."""
import numpy as np
import pytest

from test_gpu_adapters import adapters

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def expected(x, slots, base, held, i):
    """Projection i of some rows in 64 bits, and how far fp32 may be off.  The first product adds K products
    to one accumulator at most (and up to 64 parts of K joined), the second its ranks, at most 256 and two
    rounds of them, each rounding off by 2^-24 of the magnitudes so far; the factor is one
    rounding more, and each round's sum with the base one."""
    y, off = base.astype(np.float64), 2.0**-23 * np.abs(base)
    for s, adapter in enumerate(held):
        at = np.nonzero(slots == s)[0]
        if adapter is None or at.size == 0:
            continue
        a, b, f = adapter[0][i].astype(np.float64), adapter[1][i].astype(np.float64), adapter[2]
        v = x[at].astype(np.float64)
        y[at] += f * (v @ a.T) @ b.T
        size = abs(f) * (np.abs(v) @ np.abs(a).T) @ np.abs(b).T
        off[at] += (x.shape[1] + 64 + a.shape[0] + 3) * 2.0**-24 * size
    return y, off


def check(got, x, slots, bases, held, at=None):
    at = np.arange(len(slots)) if at is None else at
    for i, (g, base) in enumerate(zip(got, bases)):
        want, off = expected(x[at], slots[at], base[at], held, i)
        assert (np.abs(g[at] - want) <= off).all(), np.max(np.abs(g[at] - want) / (off + 1e-30))


def both(ops, h, x, slots, bases):
    """What a call gives in place and apart, which is the same."""
    dx, ds = ops.DeviceBuffer.from_array(x), ops.DeviceBuffer.from_array(slots.astype(np.int32))
    db = [ops.DeviceBuffer.from_array(v) for v in bases]
    ys = [ops.DeviceBuffer.from_array(np.full(v.size + 5, 7, np.float32)) for v in bases]
    h.apply_dev(dx.ptr, len(slots), ds.ptr, [d.ptr for d in db], [y.ptr for y in ys])
    apart = [y.to_array((v.size + 5,), np.float32) for y, v in zip(ys, bases)]
    for d, v in zip(db, bases):
        np.testing.assert_array_equal(d.to_array(v.shape, np.float32), v)
    h.apply_dev(dx.ptr, len(slots), ds.ptr, [d.ptr for d in db], [d.ptr for d in db])
    got = [d.to_array(v.shape, np.float32) for d, v in zip(db, bases)]
    for g, y in zip(got, apart):
        np.testing.assert_array_equal(y[:-5].reshape(g.shape), g)
        assert (y[-5:] == 7).all()
    return got


def inputs(rng, k, ns, rows):
    return (rng.standard_normal((rows, k), np.float32), [rng.standard_normal((rows, n), np.float32) for n in ns])


@pytest.mark.parametrize("fmt", ["f32", "f16"])
@pytest.mark.parametrize("k, ns, ranks", [(96, [700, 333], [129, 256, 128, 200]), (130, [1025], [255, 161, 160, 1]),
                                          (64, [31, 288, 64, 515], [192, 193, 0, 130])])
@pytest.mark.parametrize("rows", [513, 1400])
def test_ranks_in_rounds(ops, fmt, k, ns, ranks, rows):
    rng = np.random.default_rng(k + rows)
    h, held = adapters(ops, rng, k, ns, 4, 256, fmt, ranks)
    x, bases = inputs(rng, k, ns, rows)
    for slots in (rng.integers(-1, 4, rows), np.sort(rng.integers(0, 4, rows))):
        check(both(ops, h, x, slots, bases), x, slots, bases, held)


@pytest.mark.parametrize("fmt", ["f32", "f16"])
@pytest.mark.parametrize("rows, ns, rank", [(2500, [5000, 3001], 8), (4100, [5000, 3001], 40), (8191, [5000, 3001], 16),
                                            (8191, [8100], 65), (8191, [4200, 4100], 130)])
def test_many_outputs_a_workgroup(ops, fmt, rows, ns, rank):
    # (64 rows by 128 outputs are a block: three times as many blocks as 768 workgroups make it 384 outputs,
    # eight times 1024, the most.)
    rng = np.random.default_rng(rows + rank)
    k = 60
    h, held = adapters(ops, rng, k, ns, 5, rank, fmt, [rank, 1, 0, rank - 1])
    x, bases = inputs(rng, k, ns, rows)
    for slots in (np.sort(rng.integers(-1, 5, rows)), rng.integers(-1, 5, rows)):
        at = np.unique(np.r_[:40, rng.integers(0, rows, 200), rows - 40:rows])
        got = both(ops, h, x, slots, bases)
        check(got, x, slots, bases, held, at)
        none = (slots == -1) | (slots == 2)
        for g, base in zip(got, bases):
            np.testing.assert_array_equal(g[none], base[none])


@pytest.mark.parametrize("fmt", ["f32", "f16"])
@pytest.mark.parametrize("k, n, more", [(1500, 40, 700), (1024, 33, 513), (1027, 50, 200)])
def test_rounds_of_rows_that_split_k(ops, fmt, k, n, more):
    # The first 65536 rows take K at once, the rest in parts (or, 200 rows, in the form for few).
    rng = np.random.default_rng(k)
    rows = 65536 + more
    h, held = adapters(ops, rng, k, [n], 3, 16, fmt, [16, 7, 0])
    x, bases = inputs(rng, k, [n], rows)
    slots = rng.integers(-1, 3, rows)
    at = np.unique(np.r_[:60, rng.integers(0, rows, 300), 65536 - 130:rows])
    check(both(ops, h, x, slots, bases), x, slots, bases, held, at)
