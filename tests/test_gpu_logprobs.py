"""Log probabilities, entropy and alternatives against 64 bits: vocabulary and row counts
on both sides of the split, ties, masked and non-finite logits, strides."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def expected(x, tokens, top):
    """In 64 bits: (logprobs, entropy, ids, logprobs of ids)."""
    z = x.astype(np.float64)
    with np.errstate(all="ignore"):
        none = ~np.isfinite(z.max(-1)) | np.isnan(z).any(-1)
        m = np.where(none, 0, z.max(-1))[:, None]
        # (Differences to the maximum first: log S would vanish next to a large maximum.)
        lp = z - m - np.log(np.exp(z - m).sum(-1, keepdims=True))
        h = -np.where(np.exp(lp) > 0, np.exp(lp) * lp, 0).sum(-1)
    lp[none], h[none] = np.nan, np.nan
    key = np.where(np.isnan(x), np.inf, x)
    order = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -key, ~np.isnan(x)))[:, :top]
    ok = (tokens >= 0) & (tokens < x.shape[1])
    given = np.where(ok, np.take_along_axis(lp, np.where(ok, tokens, 0)[:, None], 1)[:, 0], np.nan)
    return given, h, order, np.take_along_axis(lp, order, 1)


def check(ops, x, tokens, top):
    lp, ent, ids, tops = ops.op_token_logprobs(x, tokens, top=top)
    a, h, order, b = expected(x, tokens, top)
    np.testing.assert_array_equal(ids, order)
    # A term e^d is off by (|d| + 4) 2^-23 of itself (the product with log2 e, exp2); with
    # p-weighted |d| that is at most (H + log V + 4) 2^-23 of the sum; adding V terms in
    # chains of at most V / 64 and as many roundings again in A; the result rounds once.
    v = x.shape[1]
    rel = (v / 64 + 64) * 2.0**-24 + (3 * np.log(v + 1) + 8) * 2.0**-23
    size = np.abs(x[np.isfinite(x)]).max(initial=0)
    for got, want in ((lp, a), (tops, b)):
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        f = np.isfinite(want)
        np.testing.assert_array_equal(got[~f & ~np.isnan(want)], want[~f & ~np.isnan(want)])
        assert np.abs(got[f] - want[f]).max(initial=0) <= rel + np.abs(want[f]).max(initial=0) * 2.0**-24
    np.testing.assert_array_equal(np.isnan(ent), np.isnan(h))
    f = np.isfinite(h)
    assert np.abs(ent[f] - h[f]).max(initial=0) <= 4 * rel * (np.log(v) + 2), size


@pytest.mark.parametrize("rows, vocab, top", [
    (1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 63, 63), (2, 64, 64), (7, 65, 64), (1, 255, 5), (4, 1000, 20),
    (1, 4099, 64), (8, 50257, 20), (600, 777, 8), (1, 151936, 64), (17, 128256, 1), (700, 2050, 64),
    (2100, 300, 5)])
def test_shapes(ops, rows, vocab, top):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    check(ops, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("rows", [2, 1100])
def test_ties_go_to_the_lowest_token(ops, rows):
    rng = np.random.default_rng(2)
    x = rng.integers(-3, 3, (rows, 3000)).astype(np.float32)
    check(ops, x, rng.integers(0, 3000, rows), 64)
    check(ops, np.zeros((rows, 3000), np.float32), rng.integers(0, 3000, rows), 64)
    x = np.where(rng.random((rows, 3000)) < 0.5, np.float32(-0.0), np.float32(0.0))
    check(ops, x, rng.integers(0, 3000, rows), 64)


@pytest.mark.parametrize("rows", [2, 1030])
@pytest.mark.parametrize("top", [1, 2, 10, 11, 33, 64])
def test_alternatives(ops, rows, top):
    # Few and many of them, of rows of all kinds: ties, rising and falling parts, NaN, nothing.
    rng = np.random.default_rng(top)
    v = 6007
    x = (rng.standard_normal((rows, v)) * 3).astype(np.float32)
    x[::7] = rng.integers(-2, 3, x[::7].shape)
    x[1::7] = np.sort(x[1::7], -1)
    x[2::7, :4000] = np.sort(x[2::7, :4000], -1)[:, ::-1]
    x[3::7, 50:] = -np.inf
    x[4::7][:, rng.permutation(v)[:40]] = np.nan
    x[5::7] = -np.inf
    check(ops, x, rng.integers(0, v, rows), top)


@pytest.mark.parametrize("rows", [3, 1030])
@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(ops, rows, order):
    # Rising logits offer every element to the list, falling ones only the first.
    x = np.linspace(-20, 20, 5000).astype(np.float32)[::order]
    check(ops, np.repeat(x[None], rows, 0), np.arange(rows) % 5000, 64)


@pytest.mark.parametrize("rows", [4, 1030])
def test_masked_logits(ops, rows):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((rows, 4500)) * 2).astype(np.float32)
    x[rng.random(x.shape) < 0.99] = -np.inf
    x[:, 7] = 0.5
    x[0] = -np.inf
    x[0, 4321] = -100.0  # a single token is left
    x[1] = np.finfo(np.float32).min  # masks of the lowest value
    x[1, 5] = 2.0
    tokens = rng.integers(0, 4500, rows)
    tokens[0] = 4321
    check(ops, x, tokens, 64)


@pytest.mark.parametrize("rows", [6, 1030])
def test_non_finite_logits(ops, rows):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((rows, 2600)).astype(np.float32)
    x[0, 2000] = np.nan
    x[1, 17] = np.inf
    x[2] = -np.inf
    x[3, :] = np.nan
    x[4, 9], x[4, 8] = -np.nan, np.inf
    check(ops, x, rng.integers(0, 2600, rows), 8)


def test_large_values(ops):
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((5, 3000)) * 1e4).astype(np.float32)
    x[1] *= np.float32(1e30)
    x[2] = 3e38
    x[3] = rng.uniform(80, 90, 3000)
    check(ops, x, rng.integers(0, 3000, 5), 16)


def test_tokens_outside_the_vocabulary(ops):
    x = np.zeros((4, 10), np.float32)
    lp, _, _, _ = ops.op_token_logprobs(x, np.array([-1, 10, 2**40, 9]))
    assert np.isnan(lp[:3]).all() and abs(lp[3] + np.log(10)) < 1e-6


def test_parts_and_strides(ops):
    # Rows inside a wider buffer, at addresses of 4 bytes; outputs that are not wanted.
    rng = np.random.default_rng(6)
    for rows, vocab, stride, off in ((3, 5001, 5001, 0), (3, 5001, 5003, 1), (4, 8192, 8200, 2),
                                     (900, 1111, 1300, 3)):
        mem = np.full(off + rows * stride, np.nan, np.float32)
        x = rng.standard_normal((rows, vocab)).astype(np.float32)
        mem[off:off + rows * stride].reshape(rows, stride)[:, :vocab] = x
        tokens = rng.integers(0, vocab, rows)
        seven = np.full(rows + 1, 7, np.float32)
        dev = [ops.DeviceBuffer.from_array(a) for a in (mem, tokens.astype(np.int32), seven, seven)]
        want = expected(x, tokens, 1)
        p = dev[0].ptr + 4 * off
        ops.token_logprobs_dev(p, rows, vocab, tokens_ptr=dev[1].ptr, logprob_ptr=dev[2].ptr,
                               row_stride=stride)
        ops.token_logprobs_dev(p, rows, vocab, entropy_ptr=dev[3].ptr, row_stride=stride)
        lp, ent = (d.to_array((rows + 1,), np.float32) for d in dev[2:4])
        assert np.abs(lp[:-1] - want[0]).max() < 1e-4 and np.abs(ent[:-1] - want[1]).max() < 1e-4
        assert lp[-1] == ent[-1] == 7
        for d in dev:
            d.free()


@pytest.mark.parametrize("max_bytes", [0, -1])
def test_without_workspace(ops, max_bytes):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 60000)).astype(np.float32)
    tokens = rng.integers(0, 60000, 2)
    ctx = ops.Context()
    dev = [ops.DeviceBuffer.from_array(t) for t in (x, tokens.astype(np.int32))]
    out = [ops.DeviceBuffer(4 * n) for n in (2, 2, 18, 18)]  # (another context's, within no budget)
    ctx.set_control(max_bytes=max_bytes)
    ops.token_logprobs_dev(dev[0].ptr, 2, 60000, tokens_ptr=dev[1].ptr, logprob_ptr=out[0].ptr,
                           entropy_ptr=out[1].ptr, top=9, top_ids_ptr=out[2].ptr,
                           top_logprobs_ptr=out[3].ptr, ctx=ctx)
    ctx.synchronize()
    a, h, order, tops = expected(x, tokens, 9)
    np.testing.assert_array_equal(out[2].to_array((2, 9), np.int32), order)
    for buf, want in ((out[0], a), (out[1], h), (out[3], tops)):
        assert np.abs(buf.to_array(want.shape, np.float32) - want).max() < 1e-4
    for t in dev + out:
        t.free()
    ctx.close()


def test_repeated_calls_are_equal(ops):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((3, 90000)).astype(np.float32)
    first = ops.op_token_logprobs(x, np.array([1, 2, 3]), top=16)
    for _ in range(3):
        for a, b in zip(first, ops.op_token_logprobs(x, np.array([1, 2, 3]), top=16)):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("max_bytes", [0, -1])
@pytest.mark.parametrize("vocab", [2**20 + 3, 2**26 + 5])
def test_long_rows(ops, vocab, max_bytes):
    # All logits but one are alike, and a lane has up to 2^18 of them: the sums do not feel how many.
    low = np.float32(-0.7)
    x = np.full(vocab, low)
    x[7] = 0
    ctx = ops.Context()
    dev = [ops.DeviceBuffer.from_array(a) for a in (x, np.array([7], np.int32))]
    out = [ops.DeviceBuffer(4) for _ in range(2)]
    ctx.set_control(max_bytes=max_bytes)
    ops.token_logprobs_dev(dev[0].ptr, 1, vocab, tokens_ptr=dev[1].ptr, logprob_ptr=out[0].ptr,
                           entropy_ptr=out[1].ptr, ctx=ctx)
    ctx.synchronize()
    e = np.exp(np.float64(low))
    s = 1 + (vocab - 1) * e
    lp, h = -np.log(s), np.log(s) - (vocab - 1) * e * np.float64(low) / s
    # A term is off by (0.7 + 4) 2^-23 of itself; sums of 128, and those of the lanes, by 200 roundings.
    # The entropy's own sum is 0.7 of the other; both results round once.
    rel = 4.7 * 2.0**-23 + 200 * 2.0**-24
    assert abs(out[0].to_array((1,), np.float32)[0] - lp) <= rel + abs(lp) * 2.0**-24
    assert abs(out[1].to_array((1,), np.float32)[0] - h) <= 3 * rel + abs(h) * 2.0**-24
    for t in dev + out:
        t.free()
    ctx.close()
