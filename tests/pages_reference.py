"""Pages of a cache in plain numpy: which pairs are copied, what fork and fit make of tables."""
import numpy as np


def copied(src, dst, pages):
    """[(src, dst)] of the pairs that are copied, and whether one is refused."""
    live = [(int(s), int(d)) for s, d in zip(src, dst) if not (s < 0 and d < 0)]
    moves = [(s, d) for s, d in live if s != d]
    done, refused = [], False
    for s, d in moves:
        bad = not (0 <= s < pages and 0 <= d < pages)
        bad |= sum(e == d for _, e in live) > 1
        bad |= any(t == d or e == s for t, e in moves if (t, e) != (s, d))
        refused |= bad
        if not bad:
            done.append((s, d))
    return done, refused


def fork(parent, past, table, refs, width, page, longest):
    past_out, table_out = np.zeros(len(parent), np.int32), np.full((len(parent), width), -1, np.int32)
    refs, refused = refs.copy(), False
    for row in table:
        for e in row:
            if 0 <= e < refs.size:
                refs[e] -= 1
    for i, p in enumerate(parent):
        if p < 0:
            continue
        if p >= len(past) or not 0 <= past[p] <= longest or -(-past[p] // page) > min(width, table.shape[1]):
            refused = True
            continue
        past_out[i] = past[p]
        for k in range(-(-past[p] // page)):
            e = table[p, k]
            if 0 <= e < refs.size:
                table_out[i, k] = e
                refs[e] += 1
            else:
                refused = True
    return past_out, table_out, refs, refused


def fit(new, past, table, refs, page):
    """(table, refs, granted, [(old, own)] pages copied, refused)."""
    table, refs = table.copy(), refs.copy()
    b = len(past)
    want = [-(-(p + n) // page) for p, n in zip(past, new)]
    held, refused = [-1] * b, False
    for i in range(b):
        row, need = table[i], -(-past[i] // page)
        fine = want[i] <= table.shape[1] and (row[:want[i]] < refs.size).all()
        if fine:
            has = next((k for k in range(want[i]) if row[k] < 0), want[i])
            fine = has >= need and (row[has:want[i]] < 0).all()
        if not fine:
            refused = True
            continue
        held[i] = next((k for k in range(need, has) if refs[row[k]] > 1), has)
    for i in range(b):
        for k in range(held[i], table.shape[1]) if held[i] >= 0 else ():
            if 0 <= table[i, k] < refs.size:
                refs[table[i, k]] -= 1
            table[i, k] = -1
    middle = [int(table[i, past[i] // page]) if held[i] >= 0 and new[i] and past[i] % page else -1
              for i in range(b)]
    copy = [m >= 0 and middle[:i].count(m) + 1 < refs[m] for i, m in enumerate(middle)]
    shared = [m >= 0 and refs[m] > 1 for m in middle]
    free = [k for k in range(refs.size) if refs[k] == 0]
    granted, moves, at = np.zeros(b, np.int32), [], 0
    for i in range(b):
        if held[i] < 0:
            continue
        need = int(copy[i]) + want[i] - held[i]
        fits = at + need <= len(free)
        at += need
        granted[i] = fits or (need == 0 and not shared[i])
        if not granted[i] or not need:
            continue
        mine = free[at - need:at]
        if copy[i]:
            moves.append((middle[i], mine[0]))
            refs[middle[i]] -= 1
            table[i, past[i] // page] = mine[0]
        table[i, held[i]:want[i]] = mine[int(copy[i]):]
        refs[mine] = 1
    return table, refs, granted, moves, refused
