"""The quantised KV cache and the attention over it in plain numpy (64 bits), from the
formulas: what each format stores, what it reads back, and which keys a row sees."""
import numpy as np


def rotate(x, cos, sin, pos, inter):
    """Rows [n, heads, d] turned at positions pos [n], in 64 bits, rounded once to fp32."""
    x = np.asarray(x, np.float32)
    half = cos.shape[1]
    y = x.copy()
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = np.where(ok, pos, 0)
    c, s = (t.astype(np.float64)[at][:, None] for t in (cos, sin))
    a = x.astype(np.float64)
    p, q = (a[..., :2 * half:2], a[..., 1:2 * half:2]) if inter else (a[..., :half], a[..., half:2 * half])
    u, w = p * c - q * s, q * c + p * s
    u[~ok], w[~ok] = np.nan, np.nan
    if inter:
        y[..., :2 * half:2], y[..., 1:2 * half:2] = u, w
    else:
        y[..., :half], y[..., half:2 * half] = u, w
    return y


def cached(x, fmt):
    """What the cache gives back for fp32 vectors x [..., d], as fp32."""
    x = np.asarray(x, np.float32)
    ok = np.isfinite(x).all(-1, keepdims=True)
    z = np.where(ok, x, 0).astype(np.float64)
    if fmt == "int4":
        hi, lo = z.max(-1, keepdims=True), z.min(-1, keepdims=True)
        m, h = ((hi + lo) * 0.5).astype(np.float32), ((hi - lo) / 30).astype(np.float32)
        u = np.where(h > 0, (z - m) / np.where(h > 0, h, 1).astype(np.float64), 0.0)
        n = np.clip(np.rint((u + 15) * 0.5), 0, 15)
        # One rounding: the product of 5 and 24 bits and the sum are exact in 64.
        y = m.astype(np.float64) + (2 * n - 15) * h.astype(np.float64)
    else:
        s = (np.abs(z).max(-1, keepdims=True) / (127 if fmt == "int8" else 448)).astype(np.float32)
        u = np.where(s > 0, z / np.where(s > 0, s, 1).astype(np.float64), 0.0)
        if fmt == "int8":
            q = np.clip(np.rint(u), -127, 127)
        else:
            step = np.exp2(np.maximum(np.frexp(u)[1] - 1, -6) - 3.0)
            q = np.clip(np.rint(u / step) * step, -448, 448)
        y = q * s.astype(np.float64)
    return np.where(ok, y, np.nan).astype(np.float32)


def visible(n, past, tree=None):
    """[n, past + n]: which positions each row sees."""
    if tree is None:
        return np.tril(np.ones((n, past + n), bool), past)
    see = np.ones((n, past + n), bool)
    j = np.arange(n)
    bit = (tree[:, j // 64] >> (j % 64).astype(np.uint64)) & np.uint64(1)
    see[:, past:] = bit.astype(bool)
    return see


def attend(q, k, v, see, scale):
    """q [n, heads, d], k / v [t, kv, d], see [n, t] -> [n, heads, d] in 64 bits; a row that
    sees nothing is zero, and nothing of an unseen key or value arrives."""
    n, heads, d = q.shape
    kv = k.shape[1]
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    y = np.zeros((n, heads, d))
    for h in range(heads):
        for i in range(n):
            t = see[i]
            if not t.any():
                continue
            with np.errstate(all="ignore"):
                s = k[t, h * kv // heads] @ q[i, h] * scale
                w = np.exp(s - s.max())
                y[i, h] = (w / w.sum()) @ v[t, h * kv // heads]
    return y


def bound(q, k, v, scale):
    """How far an output may be off.  A row's digits are off by 2^-23 of its largest
    element (two fp16 digits, the first with 11 bits), a sum of d products by (d + 8) 2^-24 of
    its magnitudes, so a score by that much of scale * max|q| * sum|k|; a weight by its
    score's error and 2^-21 (exp2, the scale, its two digits), twice (numerator and sum);
    the sums over t keys by a rounding every 32 keys and some at the joins.  The values'
    terms are at most three times the largest value (INT4: middle and offset apart)."""
    k, v = (np.where(np.isfinite(a), a, 0).astype(np.float64) for a in (k, v))
    d, t = q.shape[-1], max(k.shape[0], 1)
    q = np.where(np.isfinite(q), q, 0)
    size = abs(scale) * np.abs(q).max(initial=0) * np.abs(k).sum(-1).max(initial=0)
    eps = 2 * ((2 + d + 8) * 2.0**-24 * size + 2.0**-21) + (t / 32 + 64) * 2.0**-24
    return 3 * eps * np.abs(v).max(initial=0)


class Batch:
    """A packed batch over shuffled pages: row_start, past, page_table, and its host sizes."""

    def __init__(self, rng, new, past, page, spare=2, extra_rows=0):
        self.new, self.past, self.page = list(new), np.array(past, np.int32), page
        self.row_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.row_start[-1]) + extra_rows
        width = max([-(-(n + p) // page) for n, p in zip(new, past)] + [1])
        self.pages = len(new) * width + spare
        self.page_table = rng.permutation(self.pages)[:len(new) * width].astype(np.int32).reshape(
            len(new), width)

    def args(self):
        return dict(row_start=self.row_start, past=self.past, page_table=self.page_table)
