"""Attention over the quantised cache where weights and V scales lie far apart: what a key
contributes is as exact as its weight, whatever the weights and the values of the others are."""
import numpy as np
import pytest

import kv_reference as R

pytestmark = pytest.mark.gpu

FMTS = ["int8", "e4m3", "int4"]
LN2 = np.log(2.0)


@pytest.fixture(scope="module")
def ops():
    from onnx_runtime_dart_amd import ops as _ops
    return _ops


def softmax(s):
    w = np.exp(s - s.max())
    return w / w.sum()


def bound(s, v, tiles):
    """How far a row's output may be off: s [t] its scores, v [t, d] the values as read back,
    tiles of 32 keys that one wave sums at most.

    Queries and keys have one element each, so a score is one product: the query is a power of
    two, its factor scale log2(e) rounds by 2^-24, its product by 2^-24 and to two digits by
    2^-22, the product with the key's scale and the difference to the reference by 2^-24 each
    (INT4: middle and offset, three times the score's size): 8 2^-24 |s|, INT4 three times.
    A weight: that, and 2^-21 (exp2, the scale, its digits of 22 bits).  Digits end at 2^-25
    where the weights times scales of a wave sum to 2^8.5 at least, so each of its keys may lose
    2^-33.5 of its sum.  Twice for the sum of weights; the sums round once a tile and some 32 times
    at the joins.  A value's terms are at most three times its vector's largest element (INT4:
    middle and offset apart)."""
    p, size = softmax(s), np.abs(v).max(-1)
    eps = 24 * np.abs(s) * 2.0**-24 + 2.0**-21
    each = (p * size) @ eps + (p * size).sum() * (p @ eps)
    return 3 * (each + (32 * tiles * 2.0**-33.5 + (tiles + 32) * 2.0**-24) * (p * size).sum())


class Far:
    """One sequence of scores s [t] and values v [t, d]; new rows at its end."""

    def __init__(self, ops, fmt, s, v, new=1, heads=1, kv=1, page=64, **kw):
        t, d = v.shape
        self.ops, self.new, self.heads, self.kv = ops, new, heads, kv
        self.b = R.Batch(np.random.default_rng(1), [new], [t - new], page)
        k = np.zeros((t, kv, d), np.float32)
        k[..., 0] = s[:, None]
        vv = np.repeat(v.astype(np.float32)[:, None], kv, 1)
        self.cache = ops.KvCache(self.b.pages, kv_heads=kv, head_size=d, page_size=page, fmt=fmt, **kw)
        self.cache.append(k, vv, row_start=[0, t], past=[0], page_table=self.b.page_table)
        self.q = np.zeros((new, heads, d), np.float32)
        self.q[..., 0] = 1
        self.s = R.cached(k[:, 0], fmt)[:, 0].astype(np.float64)
        self.v = R.cached(vv[:, 0], fmt).astype(np.float64)

    def check(self, tiles, tree=None, rows=None):
        y = self.cache.attend(self.q, **self.b.args(), scale=1.0, tree=tree)
        see = R.visible(self.new, len(self.s) - self.new, tree)
        for i in range(self.new) if rows is None else rows:
            s, v = self.s[see[i]], self.v[see[i]]
            want, tol = softmax(s) @ v, bound(s, v, tiles)
            err = np.abs(y[i] - want).max()
            assert err <= tol, (i, err, tol)
        self.cache.release()


# One row, whose workgroup shares the keys out; many, in workgroups of 64 and of 128 rows.
SHAPES = [dict(new=1), dict(new=300, heads=256, kv=16), dict(new=500, heads=256, kv=16)]


def sample(new):
    return [r for r in (0, 1, 17, 40, 63, 64, 130, 300, new - 1) if 0 <= r < new]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("larger", [0, 4, 12, 20, 30, 60])
@pytest.mark.parametrize("place", [3, -1])
def test_large_values_of_little_weight(ops, fmt, shape, larger, place):
    # A visible key of weight 2^-40 (2^-80 where it would count) has values 2^larger times the
    # others': they are as exact as without it.
    rng = np.random.default_rng(larger)
    t = 700
    at = place if place >= 0 else t - shape["new"] - 1
    s, v = rng.uniform(-1, 1, t), rng.uniform(0.5, 1.5, (t, 64))
    s[at] = -(40 if larger < 30 else 100) * LN2
    v[at] *= 2.0**larger
    Far(ops, fmt, s, v, **shape).check(t / 32 + 1, rows=sample(shape["new"]))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("low", [12, 20, 24, 28, 34])
@pytest.mark.parametrize("first", [0.0, 1e-6, 1.0])
def test_many_keys_of_little_weight(ops, fmt, low, first):
    # 131071 equal keys `low` bits below an early one, whose values are zero, small or like theirs.
    t = 131072
    rng = np.random.default_rng(low)
    s, v = np.zeros(t), rng.uniform(0.5, 1.5, (t, 64))
    s[5] = low * LN2
    v[5] *= first
    # (The keys are split: no wave sums more than 64 tiles.)
    Far(ops, fmt, s, v).check(64)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("low", [10, 20, 30])
@pytest.mark.parametrize("first", [0.0, 1e-6, 1.0])
@pytest.mark.parametrize("shape", [dict(new=64, heads=256, kv=16), SHAPES[2]], ids=str)
def test_many_rows_over_keys_of_little_weight(ops, fmt, low, first, shape):
    t = 6000
    rng = np.random.default_rng(low)
    s, v = np.zeros(t), rng.uniform(0.5, 1.5, (t, 64))
    s[5] = low * LN2
    v[5] *= first
    Far(ops, fmt, s, v, **shape).check(t / 32 + 1, rows=sample(shape["new"]))


ORDERS = {"rising": np.sort, "falling": lambda x: np.sort(x)[::-1], "any": lambda x: x}


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("scores", ORDERS)
@pytest.mark.parametrize("sizes", ORDERS)
@pytest.mark.parametrize("d", [64, 128, 200])
def test_weights_and_values_of_all_sizes(ops, fmt, shape, scores, sizes, d):
    # Scores over 2^120, values over 2^80, each along the sequence in some order.
    rng = np.random.default_rng(7)
    t = 900
    s = ORDERS[scores](rng.uniform(-60, 60, t)) * LN2
    v = rng.uniform(0.5, 1.5, (t, d)) * np.exp2(ORDERS[sizes](rng.uniform(-40, 40, t)))[:, None]
    Far(ops, fmt, s, v, **shape).check(t / 32 + 1, rows=sample(shape["new"]))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_zero_values_first(ops, fmt, shape):
    # Until late only values of zero; then small ones of small weight; and the largest last.
    rng = np.random.default_rng(8)
    t = 900
    v = rng.uniform(0.5, 1.5, (t, 64))
    v[:200], v[200:250] = 0, v[200:250] * 1e-9
    s = rng.uniform(-2, 2, t)
    s[:100] += 12
    for late in (0.0, 25.0):
        s[300:] += late
        Far(ops, fmt, s, v, **shape).check(t / 32 + 1, rows=sample(shape["new"]))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new, heads", [(30, 1), (64, 512)])
def test_trees_over_values_of_all_sizes(ops, fmt, new, heads):
    # Drafts of values 2^60 apart, of which each row sees a few: as exact as what it sees.
    rng = np.random.default_rng(9)
    past = 40
    t = past + new
    v = rng.uniform(0.5, 1.5, (t, 64)) * np.exp2(rng.choice([-30, 0, 30], t))[:, None]
    s = rng.uniform(-8, 8, t)
    v[:past] *= 1e-18
    tree = np.uint64(1) << rng.integers(0, new, (new, 1)).astype(np.uint64)
    tree[::3] = 0
    Far(ops, fmt, s, v, new=new, heads=heads, kv=min(heads, 16), page=16).check(t / 32 + 1, tree=tree)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new, heads", [(30, 1), (64, 512), (500, 256)])
@pytest.mark.parametrize("drafts", [False, True])
def test_values_of_the_last_size_that_a_row_does_not_see(ops, fmt, d, new, heads, drafts):
    # Some of the new tokens hold values near the largest of all; rows before them, and drafts beside
    # them, are as exact as without.
    rng = np.random.default_rng(10)
    past = 70
    t = past + new
    v = rng.uniform(0.5, 1.5, (t, d)) * np.exp2(rng.choice([-20, 0], t))[:, None]
    s = rng.uniform(-8, 8, t)
    far = past + np.array([new // 3, new // 2, new - 1])
    v[far] = rng.choice([-1, 1], (3, d)) * 1e37
    tree = None
    if drafts:
        words = -(-new // 64)
        j = rng.integers(0, new, new)
        j[np.isin(j + past, far)] = 0
        tree = np.zeros((new, words), np.uint64)
        tree[np.arange(new), j // 64] = np.uint64(1) << (j % 64).astype(np.uint64)
    rows = [r for r in range(new) if drafts or r < new // 3]
    Far(ops, fmt, s, v, new=new, heads=heads, kv=min(heads, 16), page=16).check(
        t / 32 + 1, tree=tree, rows=rows if new < 100 else rows[::7])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("size", [2.0**22, 2.0**24, 2.0**27, 2.0**34, -(2.0**34)])
def test_scores_beyond_what_their_digits_tell_apart(ops, fmt, shape, size):
    # Equal keys share the weight, however large their scores; all others are far below.
    rng = np.random.default_rng(11)
    t = 900
    top = rng.random(t) < 0.3
    top[:2] = [False, True]
    s, v = np.where(top, size, size - 0.5 * abs(size)), rng.uniform(0.5, 1.5, (t, 64))
    far = Far(ops, fmt, s, v, **shape)
    y = far.cache.attend(far.q, **far.b.args(), scale=1.0)
    past = t - far.new
    for i in sample(far.new):
        seen = far.v[:past + i + 1][top[:past + i + 1]]
        tol = bound(np.zeros(len(seen)), seen, t / 32 + 1)
        assert np.abs(y[i] - seen.mean(0)).max() <= tol, i
    far.cache.release()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t, shape", [(9, SHAPES[0]), (300, SHAPES[0]), (40000, SHAPES[0]), (900, SHAPES[1]),
                                      (6000, dict(new=64, heads=256, kv=16))], ids=str)
def test_values_of_the_last_size(ops, fmt, t, shape):
    # Means of values near the largest of all are finite, also where waves and splits are joined.
    rng = np.random.default_rng(12)
    v = rng.uniform(0.9, 1, (t, 64)) * 3.3e38
    new = min(shape["new"], t)
    Far(ops, fmt, rng.uniform(-0.1, 0.1, t), v, **dict(shape, new=new)).check(
        64 if t == 40000 else t / 32 + 1, rows=sample(new))
