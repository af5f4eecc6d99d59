"""Verification of drafted tokens against its definition in 64 bits: chains and trees, with and
without draft distributions, greedy and random, borders of the random numbers, masked and
non-finite logits, strides, loose and broken bounds, captured graphs."""
import numpy as np
import pytest

import drafts_reference as R
from hip_graph import Captured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def batch(rng, new, vocab, tree=False, draft=True, size=2.5):
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(start[-1])
    target = (rng.standard_normal((rows, vocab)) * size).astype(np.float32)
    near = (0.9 * target + 0.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    parent = np.full(rows, -1, np.int32)
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    for b, n in enumerate(new):
        for i in range(1, n):
            up = int(rng.integers(0, i)) if tree else i - 1
            r = start[b] + up
            parent[start[b] + i] = up
            if tree:
                nth = int((parent[start[b] + 1:start[b] + i] == up).sum())
                tokens[start[b] + i] = np.argsort(-near[r], kind="stable")[min(nth, vocab - 1)]
            else:
                tokens[start[b] + i] = R.draw(R.weights(near[r], 1.0), rng.random())
    return dict(target=target, tokens=tokens, uniform=rng.random(rows).astype(np.float32),
                row_start=start, parent=parent if tree else None, draft=near if draft and not tree else None)


def check(ops, **a):
    got = ops.op_verify_drafts(**a)
    want = R.verify(**a)
    for g, w in zip(got[::-1], want[::-1]):
        np.testing.assert_array_equal(g, w)
    return got


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 255, 1000, 2047, 2048, 2049, 4097, 50257])
@pytest.mark.parametrize("draft", [False, True])
def test_chains(ops, vocab, draft):
    rng = np.random.default_rng(vocab)
    new = [1, 5, 0, 2, 9, 1, 17, 3]
    a = batch(rng, new, vocab, draft=draft)
    check(ops, **a, temperature=np.array([1.0, 0.7, 1, 0, 0.3, 2.0, 1.0, 0.9], np.float32))


@pytest.mark.parametrize("vocab", [2, 7, 300, 2048, 33000])
def test_trees(ops, vocab):
    rng = np.random.default_rng(vocab)
    a = batch(rng, [25, 1, 64, 0, 7, 13], vocab, tree=True, size=1.0)
    check(ops, **a, temperature=np.array([1.0, 1, 0.8, 1, 0, 1.5], np.float32))


def test_large_vocabulary(ops):
    rng = np.random.default_rng(1)
    for tree in (False, True):
        a = batch(rng, [6, 3, 4], 151936, tree=tree)
        check(ops, **a, temperature=np.array([1.0, 0.6, 0.0], np.float32))


def test_many_rows(ops):
    rng = np.random.default_rng(2)
    new = [1024, 700, 1]
    a = batch(rng, new, 33, tree=True, size=0.3)
    check(ops, **a)
    # A chain of 1024 that all stay.
    a = batch(rng, [1024], 40, draft=False)
    a["target"][:] = -np.inf
    a["target"][np.arange(1023), a["tokens"][1:]] = 1.0
    a["target"][-1, 7] = 0.0
    out, kept, count = check(ops, **a)
    assert count[0] == 1024 and out[-1] == 7 and (kept == np.arange(1024)).all()


def test_many_sequences(ops):
    rng = np.random.default_rng(3)
    new = rng.integers(0, 4, 3000)
    check(ops, **batch(rng, new, 17), temperature=rng.random(3000).astype(np.float32))


def test_borders_of_the_random_numbers(ops):
    # Equal logits of 4096 tokens: every number is exact, so are comparisons at borders.
    v = 4096
    n = 40
    target = np.zeros((2 * n, v), np.float32)
    tokens = np.zeros(2 * n, np.int32)
    tokens[1::2] = np.arange(n) * 100
    uniform = np.zeros(2 * n, np.float32)
    k = np.arange(n) * 103 % v
    uniform[0::2] = k / v  # of the whole: token k, or among those without the rejected one
    uniform[1::2] = np.where(np.arange(n) % 2, 1 / v, np.nextafter(np.float32(1 / v), np.float32(0)))
    start = np.arange(n + 1, dtype=np.int32) * 2
    out, kept, count = check(ops, target=target, tokens=tokens, uniform=uniform, row_start=start)
    np.testing.assert_array_equal(count, np.where(np.arange(n) % 2, 1, 2))
    assert (out[0::2][::2] == tokens[1::2][::2]).all() and (out[1::2][::2] == k[::2]).all()
    # With a draft of the same distribution all stay; with one that knows better, u q < p at p / q = 1/2.
    draft = np.zeros((2 * n, v), np.float32)
    check(ops, target=target, tokens=tokens, uniform=uniform, row_start=start, draft=draft)
    draft[:, ::2] = -np.inf
    tokens[1::2] = 1
    uniform[1::2] = np.where(np.arange(n) % 2, 0.5, np.nextafter(np.float32(0.5), np.float32(0)))
    _, _, count = check(ops, target=target, tokens=tokens, uniform=uniform, row_start=start, draft=draft)
    np.testing.assert_array_equal(count, np.where(np.arange(n) % 2, 1, 2))


def test_first_and_last_tokens(ops):
    rng = np.random.default_rng(4)
    a = batch(rng, [1] * 6, 5000, draft=False)
    a["uniform"][:] = [0, 0, 0, 1 - 2.0**-24, 1 - 2.0**-24, 1 - 2.0**-24]
    a["target"][1, :4000] = -np.inf
    a["target"][4, 4000:] = -np.inf
    a["target"][2] = -np.inf
    a["target"][2, 3000] = -50
    out = check(ops, **a)[0]
    assert out[0] == 0 and out[1] == 4000 and out[2] == 3000 and out[4] <= 3999


def test_masked_and_non_finite_rows(ops):
    rng = np.random.default_rng(5)
    for draft in (False, True):
        a = batch(rng, [4] * 9, 3000, draft=draft)
        a["uniform"][1::4] = 0.0
        t = a["target"]
        t[0, 17] = np.nan
        t[4, 2999] = np.inf
        t[8] = -np.inf
        t[13, 5] = -np.nan                      # the second row, reached or not
        t[16:20, ::2] = -np.inf                 # half of the vocabulary masked
        t[20:24] = np.where(rng.random((4, 3000)) < 0.99, np.finfo(np.float32).min, t[20:24])
        if draft:
            a["draft"][24, 9] = np.nan          # no draft distribution
            a["draft"][28] = -np.inf
            a["draft"][32:36, 1::2] = -np.inf
        out, _, _ = check(ops, **a)
        assert out[0] == out[4] == out[8] == -1


# Weights of 1 in each run of 2048 logits; the half of them ends with a run, and runs without any follow.
HALVES = [[0, 43, 0, 10, 29, 0, 0, 7, 0, 19, 35, 18, 0, 0, 17, 0],
          [1, 14, 17, 0, 0, 0, 0, 4, 34, 0, 0, 11, 0, 3, 0, 56],
          [0, 41, 0, 0, 30, 20, 0, 0, 0, 7, 17, 0, 38, 29, 0, 0],
          [0, 0, 0, 0, 0, 10, 0, 31, 8, 37, 7, 33, 0, 18, 0, 108],
          [34, 36, 0, 25, 10, 0, 0, 0, 4, 27, 0, 0, 0, 0, 37, 37],
          [0, 7, 38, 0, 7, 0, 0, 23, 0, 6, 18, 15, 0, 0, 36, 0],
          [0, 0, 0, 17, 29, 0, 27, 0, 0, 23, 0, 10, 0, 86, 0, 0],
          [2, 37, 0, 0, 0, 0, 0, 0, 17, 0, 0, 27, 0, 0, 0, 29]]


def test_borders_among_runs_without_weight(ops):
    # The random number 1/2 falls onto the border between two tokens, where sums in 64 bits may decide for
    # either of them; lanes that add the same weights in other orders must not make it a third one.
    target = np.full((len(HALVES), 2048 * 16), -np.inf, np.float32)
    beside = []
    for row, k in zip(target, HALVES):
        for run, n in enumerate(k):
            row[2048 * run:2048 * run + n] = 3.0
        tokens = np.nonzero(row == 3.0)[0]
        assert tokens.size % 2 == 0
        beside.append(tokens[tokens.size // 2 - 1:tokens.size // 2 + 1])
    n = len(HALVES)
    out, _, count = ops.op_verify_drafts(target, np.zeros(n, np.int32), np.full(n, 0.5, np.float32),
                                         np.arange(n + 1))
    assert (count == 1).all()
    assert all(t in two for t, two in zip(out, beside)), (out, beside)


def test_tokens_outside_the_vocabulary_and_parents(ops):
    rng = np.random.default_rng(6)
    a = batch(rng, [8, 8, 8], 50, tree=True, size=0.1)
    a["tokens"] = a["tokens"].astype(np.int64)
    a["tokens"][[1, 2, 10]] = [-1, 50, 2**40]
    # Rows without a parent before them are not reached, nor is what hangs under them.
    a["parent"][[3, 4, 12, 13, 18]] = [3, 7, -5, 2**30, -(2**31)]
    check(ops, **a)


def test_equal_siblings(ops):
    # The same token twice under a node: the second has no weight left.
    rng = np.random.default_rng(7)
    for seed in range(20):
        a = batch(np.random.default_rng(seed), [12] * 8, 5, tree=True, size=0.5)
        a["tokens"] = rng.integers(0, 5, a["tokens"].size).astype(np.int32)
        check(ops, **a)


def test_large_and_small_values(ops):
    rng = np.random.default_rng(8)
    a = batch(rng, [3] * 8, 2500)
    a["target"][:3] = (rng.standard_normal((3, 2500)) * 1e37).astype(np.float32)
    a["target"][3:6] = 3e38
    a["target"][6:9] = -3e38
    a["target"][9] = np.where(np.arange(2500) == 5, 3e38, -3e38)
    temp = np.array([1, 1, 1, 1, 1e-38, 1e38, np.inf, 1e-45], np.float32)
    check(ops, **a, temperature=temp)
    a["target"][18:21, ::3] = -np.inf  # masked under an infinite temperature
    a["draft"][18:21, ::3] = -np.inf
    check(ops, **a, temperature=temp)


@pytest.mark.parametrize("gap", [12.0, 18.0, 23.0])
def test_rejected_tokens_that_hold_most_of_their_runs(ops, gap):
    # A tree's root offers the largest tokens of the first three runs, each but 3400 e^-gap of its run; all
    # are rejected (fp32 has random numbers up to 1 - 2^-24), and the last token is drawn from the rest.
    rng = np.random.default_rng(17)
    seqs, vocab = 48, 7000
    row = rng.standard_normal(vocab).astype(np.float32)
    tops = [40, 2048 + 2047, 2 * 2048]
    row[tops] = [gap, gap - 0.5, gap + 1]
    row[[50, 2 * 2048 + 900]] = -np.inf
    uniform = np.full((seqs, 4), 1 - 2.0**-24, np.float32)
    uniform[:, 0] = rng.random(seqs)
    got = check(ops, target=np.tile(row, (4 * seqs, 1)), tokens=np.tile([7] + tops, seqs).astype(np.int32),
                parent=np.tile([-1, 0, 0, 0], seqs).astype(np.int32), row_start=4 * np.arange(seqs + 1),
                uniform=uniform.ravel(), draft=None)
    assert (got[2] == 1).all() and not np.isin(got[0], tops).any() and len(np.unique(got[0])) > 30


def test_greedy_ties_go_to_the_lowest_token(ops):
    rng = np.random.default_rng(9)
    a = batch(rng, [4] * 20, 7000, draft=False)
    a["target"] = np.rint(a["target"])
    best = a["target"].argmax(1)
    a["tokens"][1::4], a["tokens"][2::4] = best[0::4], best[1::4]
    _, _, count = check(ops, **a, temperature=np.zeros(20, np.float32))
    assert (count >= 3).all()
    check(ops, **a, temperature=np.full(20, np.nan, np.float32))
    a["target"][:] = -0.0
    a["target"][:, ::2] = 0.0
    a["tokens"][:] = 0
    _, _, count = check(ops, **a, temperature=np.full(20, -1, np.float32))
    assert (count == 4).all()


def test_emitted_tokens_have_the_target_distribution(ops):
    # One draft, drawn from another distribution: what is emitted first is the target's.  Shares of
    # n draws are off by 5 deviations of sqrt(p (1 - p) / n) at most (1 in 10^6 a token).
    rng = np.random.default_rng(10)
    n, v = 60000, 6
    t, q = rng.standard_normal((2, v)).astype(np.float32)
    p = R.weights(t, 1.0)
    for draft in (True, False):
        tokens = np.zeros(2 * n, np.int32)
        tokens[1::2] = rng.choice(v, n, p=R.weights(q, 1.0))
        out, _, _ = ops.op_verify_drafts(
            np.tile(t, (2 * n, 1)), tokens, rng.random(2 * n).astype(np.float32),
            np.arange(n + 1) * 2, draft=np.tile(q, (2 * n, 1)) if draft else None)
        share = np.bincount(out[0::2], minlength=v) / n
        assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


def device(ops, a, stride=0, shift=0, **kw):
    """The call on device arrays, rows inside wider buffers; outputs have a row more."""
    rows, vocab = a["target"].shape
    stride = stride or vocab
    dev = []

    def put(x):
        dev.append(ops.DeviceBuffer.from_array(x))
        return dev[-1].ptr

    def wide(x):
        if x is None:
            return 0
        mem = np.full(shift + rows * stride, np.nan, np.float32)
        mem[shift:].reshape(rows, stride)[:, :vocab] = x
        return put(mem) + 4 * shift

    n = np.diff(a["row_start"])
    args = dict(batch=n.size, rows=rows, max_new=int(n.max()), vocab=vocab, target_stride=stride,
                draft_stride=stride, row_start_ptr=put(a["row_start"]), tokens_ptr=put(a["tokens"]),
                target_ptr=wide(a["target"]), draft_ptr=wide(a["draft"]), uniform_ptr=put(a["uniform"]),
                parent_ptr=0 if a["parent"] is None else put(a["parent"]))
    outs = [ops.DeviceBuffer.from_array(np.full(k + 2, 77, np.int32)) for k in (rows, rows, n.size)]
    return ops.Drafts(**{**args, **kw}), outs, dev


@pytest.mark.parametrize("vocab, stride, shift", [(2050, 2051, 1), (3001, 3001, 3), (4096, 5000, 2)])
def test_strides(ops, vocab, stride, shift):
    a = batch(np.random.default_rng(vocab), [3, 6, 1], vocab)
    drafts, outs, dev = device(ops, a, stride, shift)
    ops.verify_drafts_dev(drafts, *[o.ptr for o in outs])
    for o, w in zip(outs, R.verify(**a)):
        got = o.to_array((w.size + 2,), np.int32)
        np.testing.assert_array_equal(got[:-2], w)
        assert (got[-2:] == 77).all()


def test_rows_of_no_sequence_and_loose_bounds(ops):
    a = batch(np.random.default_rng(11), [3, 6, 1], 900)
    want = R.verify(**a)
    # Rows before, behind and between sequences; bounds above what there is.
    pad = dict(a)
    at = np.r_[2:5, 6:12, 13:14]
    for name in ("target", "draft", "tokens", "uniform"):
        pad[name] = np.zeros((17,) + a[name].shape[1:], a[name].dtype)
        pad[name][at] = a[name]
    pad["row_start"] = np.array([2, 5, 6, 12, 13, 14], np.int32)
    ref = R.verify(**pad)
    drafts, outs, dev = device(ops, pad, max_new=1000)
    ops.verify_drafts_dev(drafts, *[o.ptr for o in outs])
    got = [o.to_array((n,), np.int32) for o, n in zip(outs, (19, 19, 7))]
    for g, w, r in zip(got[:2], want[:2], ref[:2]):
        np.testing.assert_array_equal(g[at], w)
        np.testing.assert_array_equal(g[2:14], r[2:14])
        assert (g[:2] == 77).all() and (g[14:] == 77).all()
    np.testing.assert_array_equal(got[2][:5], ref[2])


def test_broken_bounds(ops):
    a = batch(np.random.default_rng(12), [3, 3, 3], 900)
    want = R.verify(**a)
    for start, fine in (([0, 3, 10, 9], [0]), ([-1, 3, 6, 9], [1, 2]), ([0, 3, 6, 5], [0, 1])):
        drafts, outs, dev = device(ops, {**a, "row_start": np.array(start, np.int32)}, max_new=3)
        ops.verify_drafts_dev(drafts, *[o.ptr for o in outs])
        got = [o.to_array((n,), np.int32) for o, n in zip(outs, (11, 11, 5))]
        for b in range(3):
            rows = slice(3 * b, 3 * b + 3)
            if b in fine:
                np.testing.assert_array_equal(got[0][rows], want[0][rows])
                assert got[2][b] == want[2][b]
            else:
                assert got[2][b] == 0
                if start != [0, 3, 6, 5]:
                    assert (got[0][rows] == 77).all() and (got[1][rows] == 77).all()
    drafts, outs, dev = device(ops, a, max_new=0)
    ops.verify_drafts_dev(drafts, *[o.ptr for o in outs])
    assert (outs[2].to_array((5,), np.int32) == [0, 0, 0, 77, 77]).all()


def test_captured_graph(ops):
    # Chains that the replays find changed, lengths among them; a second graph shares the workspace.
    rng = np.random.default_rng(13)
    a = batch(rng, [4, 7], 5000)
    with Captured(ops) as g:
        d = {k: g.buffer(v) for k, v in a.items() if v is not None}
        outs = [[g.buffer(np.zeros(n, np.int32)) for n in (11, 11, 2)] for _ in range(2)]

        def call(which, with_draft):
            drafts = ops.Drafts(batch=2, rows=11, max_new=11, vocab=5000, row_start_ptr=d["row_start"].ptr,
                                tokens_ptr=d["tokens"].ptr, target_ptr=d["target"].ptr,
                                draft_ptr=d["draft"].ptr if with_draft else 0, uniform_ptr=d["uniform"].ptr)
            ops.verify_drafts_dev(drafts, *[o.ptr for o in outs[which]], ctx=g.ctx)

        call(0, True)
        graphs = [g.capture(lambda: call(0, True)), g.capture(lambda: call(1, False))]
        for new in ([4, 7], [9, 2], [1, 10], [11, 0]):
            b = batch(rng, new, 5000)
            for k, buf in d.items():
                g.put(buf, b[k])
            for o in outs[0] + outs[1]:
                g.put(o, np.full(o.nbytes // 4, 77, np.int32))
            for replay in graphs:
                replay()
            g.wait()
            for which, draft in ((0, b["draft"]), (1, None)):
                for o, w in zip(outs[which], R.verify(**{**b, "draft": draft})):
                    np.testing.assert_array_equal(o.to_array(w.shape, np.int32), w)


def test_workspace_and_budget(ops):
    from onnx_runtime_dart_amd.errors import OnnxMemoryLimitException, UnsupportedError
    a = batch(np.random.default_rng(14), [4, 7], 5000)
    drafts, outs, dev = device(ops, a)
    with Captured(ops) as g:
        g.ctx.set_control(max_bytes=10)
        with pytest.raises(OnnxMemoryLimitException):
            ops.verify_drafts_dev(drafts, *[o.ptr for o in outs], ctx=g.ctx)
        g.ctx.set_control(max_bytes=-1)
        # A workspace does not grow while the stream captures: the call is refused, the capture lives.
        x = g.buffer(np.zeros(4, np.float32))

        def call():
            ops.binary_f32_dev("add", x.ptr, (4,), x.ptr, (4,), x.ptr, ctx=g.ctx)
            with pytest.raises(UnsupportedError):
                ops.verify_drafts_dev(drafts, *[o.ptr for o in outs], ctx=g.ctx)

        replay = g.capture(call)
        g.put(x, np.ones(4, np.float32))
        replay()
        g.wait()
        assert (x.to_array((4,), np.float32) == 2).all()
        assert (outs[2].to_array((4,), np.int32) == 77).all()


def test_repeated_calls_are_equal(ops):
    a = batch(np.random.default_rng(15), [8] * 40, 20000)
    first = ops.op_verify_drafts(**a)
    for _ in range(3):
        for x, y in zip(first, ops.op_verify_drafts(**a)):
            np.testing.assert_array_equal(x, y)
