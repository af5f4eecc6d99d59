"""Rotary tables and the rotation against 64 bits: every scaling, far positions, both
pairings, part of the head, strided and in-place vectors, positions outside the tables."""
import math

import numpy as np
import pytest

from kv_reference import rotate
from onnx_runtime_dart_amd.errors import UnsupportedError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def frequencies(half, base, kind, f, length, low, high):
    i = np.arange(half, dtype=np.float64)
    if kind == "ntk":
        base = base * f ** (half / (half - 1))
    inv = base ** (-i / half)
    if kind == "linear":
        return inv / f
    if kind == "yarn":
        a, b = (half * math.log(length / (t * 2 * math.pi)) / math.log(base) for t in (high, low))
        a, b = max(math.floor(a), 0), min(math.ceil(b), 2 * half - 1)
        keep = 1 - np.clip((i - a) / max(b - a, 0.001), 0, 1)
        return inv / f * (1 - keep) + inv * keep
    if kind == "bands":
        keep = np.clip((length * inv / (2 * math.pi) - low) / (high - low), 0, 1)
        return inv / f * (1 - keep) + inv * keep
    return inv


@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "yarn", "bands"])
@pytest.mark.parametrize("first, count, half", [(0, 1, 1), (0, 300, 64), (131000, 73, 48),
                                                (2**31 - 70, 69, 128), (5, 1025, 17)])
def test_tables(ops, kind, first, count, half):
    if kind == "ntk" and half < 2:
        half = 2
    f, length, low, high = 8.0, 4096.0, 1.0, 32.0 if kind == "yarn" else 4.0
    cos, sin = ops.rotary_tables(count, half, first=first, base=10000.0,
                                 scaling=ops.RopeScaling(kind, factor=f, original_length=length))
    inv = frequencies(half, 10000.0, kind, f, length, low, high)
    a = 0.1 * math.log(f) + 1 if kind == "yarn" else 1.0
    # The reference's angle from an extended-precision product.
    turns = (np.arange(first, first + count, dtype=np.longdouble)[:, None] *
             inv.astype(np.longdouble) / np.longdouble(2 * np.pi))
    angle = ((turns - np.rint(turns)) * np.longdouble(2 * np.pi)).astype(np.float64)
    # The frequency and its product with a position are off by some 2^-52 (the angle by
    # 2^-50 of itself, in units of its size), the rest of a turn by 2^-25 of half turns, and
    # sine and cosine by 2 units in the last place, 2^-23, the value_factor's product 2^-24.
    tol = a * (np.pi * 2.0**-25 + 2.0**-23 + 2.0**-24 + (first + count) * inv.max() * 2.0**-50)
    assert np.abs(cos - a * np.cos(angle)).max() <= tol
    assert np.abs(sin - a * np.sin(angle)).max() <= tol


def test_no_scaling_is_the_default(ops):
    a = ops.rotary_tables(50, 32, base=500000.0)
    b = ops.rotary_tables(50, 32, base=500000.0, scaling=ops.RopeScaling("linear", factor=1.0))
    np.testing.assert_array_equal(a, b)
    assert (a[0][0] == 1).all() and (a[1][0] == 0).all()


def tables(rng, n, half):
    t = rng.uniform(0, 6, (n, half))
    return np.cos(t).astype(np.float32), np.sin(t).astype(np.float32)


# batch, seq, heads, head size, half, interleaved
CASES = [(1, 1, 1, 2, 1, False), (2, 3, 5, 64, 32, False), (1, 7, 3, 80, 17, True), (3, 1, 40, 128, 64, False),
         (1, 129, 2, 128, 32, True), (2, 5, 1, 256, 128, False), (1, 33, 4, 96, 48, True),
         (4, 2, 3, 130, 30, False), (1, 3, 2, 300, 64, True)]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotation(ops, case):
    b, s, h, d, half, inter = case
    rng = np.random.default_rng(d + s)
    x = rng.standard_normal((b, s, h * d)).astype(np.float32)
    cos, sin = tables(rng, 50, half)
    pos = rng.integers(0, 50, (b, s))
    y = ops.op_rotary_embedding(x, cos, sin, pos, interleaved=inter, num_heads=h)
    want = rotate(x.reshape(b * s, h, d), cos, sin, pos.ravel(), inter)
    np.testing.assert_array_equal(y.reshape(want.shape), want)
    # [batch, heads, seq, head_size]
    y4 = ops.op_rotary_embedding(x.reshape(b, s, h, d).transpose(0, 2, 1, 3), cos, sin, pos,
                                 interleaved=inter)
    np.testing.assert_array_equal(y4.transpose(0, 2, 1, 3).reshape(want.shape), want)


def test_default_positions_and_the_way_back(ops):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 40, 4 * 64)).astype(np.float32)
    cos, sin = tables(rng, 40, 32)
    y = ops.op_rotary_embedding(x, cos, sin, num_heads=4)
    want = rotate(x.reshape(80, 4, 64), cos, sin, np.tile(np.arange(40), 2), False)
    np.testing.assert_array_equal(y.reshape(want.shape), want)
    back = ops.op_rotary_embedding(y, cos, -sin, num_heads=4)
    # Turned twice: c^2 + s^2 is 1 within 2^-23, each turn rounds once.
    assert np.abs(back - x).max() <= 2.0**-21 * np.abs(x).max() * 2


def test_positions_outside_the_tables(ops):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((1, 5, 2 * 24)).astype(np.float32)
    cos, sin = tables(rng, 10, 8)
    pos = np.array([[0, -1, 10, 2**31 - 1, 9]])
    y = ops.op_rotary_embedding(x, cos, sin, pos, num_heads=2).reshape(5, 2, 24)
    assert np.isnan(y[1:4, :, :16]).all()
    np.testing.assert_array_equal(y[:, :, 16:], x.reshape(5, 2, 24)[:, :, 16:])
    assert np.isfinite(y[[0, 4]]).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d, half, offset", [(64, 32, 0), (64, 32, 1), (70, 20, 3), (128, 64, 4)])
def test_strided_and_in_place(ops, inter, d, half, offset):
    # Query heads inside fused rows, turned where they are and into a packed buffer; what
    # lies between stays as it was.  An offset of single elements takes 4-byte accesses.
    rng = np.random.default_rng(5)
    b, s, h = 2, 9, 3
    row = h * d + 37
    mem = rng.standard_normal(offset + b * s * row + 11).astype(np.float32)
    cos, sin = tables(rng, 30, half)
    pos = rng.integers(0, 30, (b, s)).astype(np.int32)
    dev = [ops.DeviceBuffer.from_array(a) for a in (mem, cos, sin, pos)]
    out = ops.DeviceBuffer.from_array(np.full(b * s * h * d + 5, 7, np.float32))
    r = ops.Rope(dev[1].ptr, dev[2].ptr, max_pos=30, half_rot=half, interleaved=inter,
                 positions_ptr=dev[3].ptr)
    strides = (s * row, row, d)
    ops.rotary_embedding_dev(dev[0].ptr + 4 * offset, b, s, h, d, r, out.ptr, x_strides=strides)
    ops.rotary_embedding_dev(dev[0].ptr + 4 * offset, b, s, h, d, r, dev[0].ptr + 4 * offset,
                             x_strides=strides, y_strides=strides)
    x = mem[offset:offset + b * s * row].reshape(b * s, row)[:, :h * d].reshape(b * s, h, d)
    want = rotate(x, cos, sin, pos.ravel(), inter)
    got = out.to_array((b * s * h * d + 5,), np.float32)
    np.testing.assert_array_equal(got[:-5].reshape(want.shape), want)
    assert (got[-5:] == 7).all()
    after = dev[0].to_array(mem.shape, np.float32)
    mem[offset:offset + b * s * row].reshape(b * s, row)[:, :h * d] = want.reshape(b * s, h * d)
    np.testing.assert_array_equal(after, mem)
    for x in dev + [out]:
        x.free()


def test_infinities_stay_in_their_pair(ops):
    x = np.ones((1, 2, 16), np.float32)
    x[0, 0, 3], x[0, 1, 5] = np.inf, np.nan
    cos, sin = np.full((2, 4), 0.6, np.float32), np.full((2, 4), 0.8, np.float32)
    y = ops.op_rotary_embedding(x, cos, sin, num_heads=1)
    bad = ~np.isfinite(y)
    want = np.zeros(x.shape, bool)
    want[0, 0, [3, 7]] = True
    want[0, 1, [1, 5]] = True
    np.testing.assert_array_equal(bad, want)


def test_more_than_a_launch_takes(ops):
    # Refused from the sizes alone: the buffers hold a hundred elements.
    x = ops.DeviceBuffer.from_array(np.zeros(100, np.float32))
    rope = ops.Rope(x.ptr, x.ptr, max_pos=1, half_rot=1)
    with pytest.raises(UnsupportedError):
        ops.rotary_embedding_dev(x.ptr, 1, 2**31 - 1, 8, 3, rope, x.ptr)
    with pytest.raises(UnsupportedError):
        ops.rotary_tables_dev(x.ptr, x.ptr, 0, 2**31 - 1, 127)
    x.free()


def test_positions_beyond_32_bits(ops):
    rng = np.random.default_rng(9)
    cos, sin = tables(rng, 5, 8)
    x = rng.standard_normal((1, 2, 3, 20)).astype(np.float32)  # [batch, heads, seq, head_size]
    y = ops.op_rotary_embedding(x, cos, sin, np.array([[1, 2**32 + 1, -2**32 + 2]]))
    assert np.isfinite(y[0, :, 0]).all()
    assert np.isnan(y[0, :, 1:, :16]).all() and (y[..., 16:] == x[..., 16:]).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("batch, seq, heads, d, half", [(1, 1, 1, 2, 1), (3, 7, 4, 64, 32), (2, 5, 3, 80, 16)])
def test_tables_of_each_row(ops, inter, batch, seq, heads, d, half):
    # The node without position_ids: caches [batch, seq, half], gathered before.
    rng = np.random.default_rng(10)
    x = rng.standard_normal((batch, seq, heads, d)).astype(np.float32)
    cos, sin = tables(rng, batch * seq, half)
    want = rotate(x.reshape(batch * seq, heads, d), cos, sin, np.arange(batch * seq), inter).reshape(x.shape)
    cos, sin = cos.reshape(batch, seq, half), sin.reshape(batch, seq, half)
    y = ops.op_rotary_embedding(x.reshape(batch, seq, -1), cos, sin, num_heads=heads, interleaved=inter)
    np.testing.assert_array_equal(y.reshape(x.shape), want)
    y = ops.op_rotary_embedding(x.transpose(0, 2, 1, 3), cos, sin, interleaved=inter)
    np.testing.assert_array_equal(y, want.transpose(0, 2, 1, 3))


def test_no_rows(ops):
    cos = np.ones((0, 5, 8), np.float32)
    assert ops.op_rotary_embedding(np.zeros((0, 5, 32), np.float32), cos, cos, num_heads=2).shape == (0, 5, 32)
