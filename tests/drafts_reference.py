"""The verification of drafted tokens in plain numpy (64 bits), from its definition."""
import numpy as np


def weights(x, temperature):
    """softmax(x / temperature) in 64 bits; None where the row has no distribution."""
    x = np.asarray(x, np.float32)
    if np.isnan(x).any() or (x == np.inf).any() or not np.isfinite(x).any():
        return None
    z = x.astype(np.float64) - np.float64(x.max())
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(np.isneginf(z), -np.inf, z / np.float64(np.float32(temperature)))
    e = np.exp(z)
    return e / e.sum()


def draw(w, u):
    """The first token whose running sum exceeds u of the whole; -1 if nothing is left."""
    total = np.cumsum(w)
    if not total[-1] > 0:
        return -1
    at = np.nonzero(total > u * total[-1])[0]
    return int(at[0]) if at.size else int(np.nonzero(w > 0)[0][-1])


def verify(target, tokens, uniform, row_start, parent=None, draft=None, temperature=None):
    """(tokens, kept, count) as the library returns them."""
    out, kept = (np.full(len(tokens), -1, np.int32) for _ in range(2))
    count = np.zeros(len(row_start) - 1, np.int32)
    vocab = target.shape[1]
    for b in range(count.size):
        s, n = int(row_start[b]), int(row_start[b + 1] - row_start[b])
        if n == 0:
            continue
        temp = 1.0 if temperature is None else float(np.float32(temperature[b]))
        greedy = not temp > 0
        cur, rows, emitted, left, rest = 0, [0], [], 1.0, None
        p = weights(target[s], 1.0 if greedy else temp)
        gone = []
        for i in range(1, n):
            if (i - 1 if parent is None else int(parent[s + i])) != cur:
                continue
            x, u = int(tokens[s + i]), float(np.float32(uniform[s + i]))
            inside = p is not None and 0 <= x < vocab
            if greedy:
                stays = inside and x == int(np.argmax(target[s + cur]))
            elif draft is not None:
                q = weights(draft[s + cur], temp)
                stays = inside and q is not None and p[x] > 0 and u * q[x] < p[x]
                if not stays and q is not None and p is not None:
                    rest = np.maximum(p - q, 0.0)
            else:
                stays = inside and x not in gone and p[x] > 0 and u * left < p[x]
                if inside and not stays and x not in gone:
                    left -= p[x]
                    gone.append(x)
            if stays:
                emitted.append(x)
                rows.append(i)
                cur, left, rest, gone = i, 1.0, None, []
                p = weights(target[s + cur], 1.0 if greedy else temp)
        if p is None:
            last = -1
        elif greedy:
            last = int(np.argmax(target[s + cur]))
        else:
            w = p.copy()
            if rest is not None and rest.sum() > 2.0**-40:
                w = rest
            w[gone] = 0.0
            last = draw(w, float(np.float32(uniform[s])))
        emitted.append(last)
        count[b] = len(emitted)
        out[s:s + len(emitted)] = emitted
        kept[s:s + len(rows)] = rows
    return out, kept, count
